"""Rotary positions (kore_rope_apply_dev) against the formula in 64 bits."""
import math

import numpy as np
import pytest
import torch

from tests.paged_ref import DTYPE, UNIT, rope_bound, rope_freqs, rope_rows, to64

pytestmark = pytest.mark.gpu


def _apply(x, pos, cfg, heads, hd, dtype, in_place=False, transpose=False, pad=0, off=0):
    from kore_amd import rope
    n = x.shape[0]
    wide = torch.full((n, off + heads * hd + pad), 3.0, dtype=DTYPE[dtype])
    wide[:, off:off + heads * hd] = x.reshape(n, -1)
    d = wide.cuda()
    out = d if in_place else torch.full_like(d, 3.0)
    p = torch.as_tensor(pos, dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    with rope.Rope(cfg) as r:
        r.apply_dev(dtype, n, heads, hd, d.data_ptr() + off * d.element_size(), p.data_ptr(),
                    out.data_ptr() + off * d.element_size(), d.shape[1], out.shape[1], transpose)
        r.sync()
    got = out.cpu()
    assert (got[:, :off] == 3.0).all() and (got[:, off + heads * hd:] == 3.0).all(), "written outside the rows"
    if not in_place:
        assert torch.equal(d.cpu().view(torch.uint8), wide.view(torch.uint8)), "the input was written"
    return got[:, off:off + heads * hd].reshape(n, heads, hd)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("n,heads,hd,rot,pad,off", [
    (1, 1, 2, 2, 0, 0), (1, 32, 128, 128, 0, 0), (5, 3, 96, 64, 4, 8), (7, 2, 66, 34, 3, 1), (3, 5, 40, 40, 1, 0),
    (17, 14, 64, 64, 0, 2), (2, 1, 1024, 512, 0, 0), (300, 3, 72, 48, 0, 0),
])
def test_against_the_formula(dtype, layout, n, heads, hd, rot, pad, off):
    from kore_amd import rope
    rng = np.random.default_rng(hd + rot)
    x = torch.from_numpy(rng.standard_normal((n, heads, hd))).to(DTYPE[dtype])
    pos = rng.integers(0, 200000, n)
    pos[0] = 0
    got = _apply(x, pos, rope.Config(rot, layout), heads, hd, dtype, pad=pad, off=off)
    f, m = rope_freqs(rot)
    want, size = rope_rows(to64(x), pos, f, m, layout)
    assert (np.abs(to64(got) - want) <= rope_bound(want, size, dtype)).all()
    assert torch.equal(got[..., rot:], x[..., rot:]), "dims behind the rotated ones are copied"
    assert torch.equal(_apply(x, pos, rope.Config(rot, layout), heads, hd, dtype, in_place=True, pad=pad, off=off), got)


@pytest.mark.parametrize("cfg", [
    dict(scaling="linear", factor=2.5), dict(scaling="yarn", factor=4.0, orig_ctx=32768),
    dict(scaling="yarn", factor=16.0, orig_ctx=4096, beta_fast=16.0, beta_slow=2.0), dict(base=10000.0),
    dict(scaling="yarn", factor=1.0, orig_ctx=100), dict(magnitude=0.5),
])
def test_scalings_and_far_positions(cfg):
    """Angles up to 2^31 - 1: the reduction is exact where fp32 would have lost the angle."""
    from kore_amd import rope
    rng = np.random.default_rng(5)
    pos = np.concatenate([[0, 1, 2 ** 31 - 1, 2 ** 30, 1000003], rng.integers(0, 2 ** 31 - 1, 200)])
    x = torch.from_numpy(rng.standard_normal((len(pos), 2, 128))).float()
    got = _apply(x, pos, rope.Config(128, **cfg), 2, 128, "f32")
    ref = {k: v for k, v in cfg.items() if k in ("scaling", "factor", "orig_ctx", "base")}
    f, m = rope_freqs(128, fast=cfg.get("beta_fast", 32.0), slow=cfg.get("beta_slow", 1.0), **ref)
    with rope.Rope(rope.Config(128, **cfg)) as r:
        gf, gm = r.freqs()
    m = cfg.get("magnitude", m)
    assert np.array_equal(gf, f) and gm == np.float32(m)
    want, size = rope_rows(to64(x), pos, f, m, "half")
    # the angle in double is off by up to 2^31 2^-53 at the farthest position, in the oracle and in the kernel
    assert (np.abs(to64(got) - want) <= rope_bound(want, size, "f32") + 4 * 2.0 ** -22 * 2.0 ** -1 * np.abs(to64(x)).max() *
            (np.asarray(pos) / 2.0 ** 31)[:, None, None]).all()


def test_pair_factors():
    from kore_amd import rope
    rng = np.random.default_rng(8)
    fac = rng.uniform(0.5, 8.0, 32)
    x = torch.from_numpy(rng.standard_normal((9, 3, 80))).float()
    pos = rng.integers(0, 5000, 9)
    got = _apply(x, pos, rope.Config(64, "interleaved", freq_factors=fac), 3, 80, "f32")
    f, m = rope_freqs(64, factors=fac)
    want, size = rope_rows(to64(x), pos, f, m, "interleaved")
    assert (np.abs(to64(got) - want) <= rope_bound(want, size, "f32")).all()


def test_rows_equal_the_contiguous_caches():
    """The half layout over the whole head gives the cache rows of KoreAttn (kore's own) bit for bit."""
    import kore_amd
    from kore_amd import rope
    rng = np.random.default_rng(2)
    n, nkv, hd = 300, 4, 128
    k, v = (rng.standard_normal((n, nkv * hd)).astype(np.float32) for _ in range(2))
    with kore_amd.KoreAttn(1, n, 28, nkv, hd, 1e6) as a:
        dk, dv = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
        torch.cuda.synchronize()
        a.append_dev(0, 0, n, dk.data_ptr(), dv.data_ptr())
        a.sync()
        want, _ = a.read_kv(0, 0, n)
    got = _apply(torch.from_numpy(k).view(n, nkv, hd), np.arange(n), rope.Config(hd), nkv, hd, "f32")
    assert np.array_equal(got.reshape(n, -1).numpy().view(np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_transpose_is_the_gradient(layout):
    """<apply(x), g> against <x, transpose(g)> from the formula, and the derivative of <apply(x), g> by differences (the
    call is linear, so a step of 1 is exact but for rounding)."""
    from kore_amd import rope
    rng = np.random.default_rng(4)
    n, heads, hd, rot = 6, 3, 48, 32
    cfg = rope.Config(rot, layout, scaling="yarn", factor=4.0, orig_ctx=64)
    f, m = rope_freqs(rot, scaling="yarn", factor=4.0, orig_ctx=64)
    x, g = (torch.from_numpy(rng.standard_normal((n, heads, hd))).float() for _ in range(2))
    pos = rng.integers(0, 9999, n)
    dx = _apply(g, pos, cfg, heads, hd, "f32", transpose=True)
    want, size = rope_rows(to64(g), pos, f, m, layout, transpose=True)
    assert (np.abs(to64(dx) - want) <= rope_bound(want, size, "f32")).all()
    y0 = to64(_apply(x, pos, cfg, heads, hd, "f32"))
    for d in (0, 1, rot // 2, rot - 1, rot, hd - 1):
        x1 = x.clone()
        x1[..., d] += 1.0
        diff = ((to64(_apply(x1, pos, cfg, heads, hd, "f32")) - y0) * to64(g)).sum(-1)
        step = to64(x1)[..., d] - to64(x)[..., d]
        # two outputs of a pair, each off by 4 half steps of (|x| + 1) m twice over, weighted by |g|
        tol = 2 * 2 * 4 * UNIT["f32"] * 1.5 * (np.abs(to64(x)).max() + 1) * 2 * np.abs(to64(g)).max()
        assert np.abs(diff - step * to64(dx)[..., d]).max() <= tol + 1e-6 * np.abs(step - 1).max() + 2 ** -22
    back = to64(_apply(torch.from_numpy(y0).float(), pos, cfg, heads, hd, "f32", transpose=True))
    back[..., :rot] /= m * m
    assert np.abs(back - to64(x)).max() <= 32 * UNIT["f32"] * np.abs(to64(x)).max()


@pytest.mark.skipif(np.finfo(np.longdouble).nmant < 63, reason="the oracle's long double holds no more than a double")
@pytest.mark.parametrize("factor", [1.0, 0.37, 2.0 ** -20])
def test_angles_past_a_doubles_53_bits(factor):
    """Positions and frequencies whose product takes up to 55 bits: within the bound of near ones."""
    from kore_amd import rope
    rng = np.random.default_rng(6)
    pos = np.concatenate([[2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30 + 1, 2 ** 29 + 3], rng.integers(2 ** 29, 2 ** 31 - 1, 400)])
    x = torch.from_numpy(rng.standard_normal((len(pos), 1, 96))).float()
    cfg = dict(scaling="linear", factor=factor)
    got = to64(_apply(x, pos, rope.Config(96, **cfg), 1, 96, "f32"))[:, 0]
    f, _ = rope_freqs(96, **cfg)
    ang = pos.astype(np.longdouble)[:, None] * f.astype(np.longdouble)   # exact: 31 + 24 bits
    c, s, x = np.cos(ang), np.sin(ang), to64(x)[:, 0]
    a, b = x[:, :48], x[:, 48:]
    want = np.concatenate([a * c - b * s, a * s + b * c], 1)
    size = np.concatenate([np.abs(a * c) + np.abs(b * s), np.abs(a * s) + np.abs(b * c)], 1)
    assert (np.abs(got - want) <= rope_bound(want, size, "f32")).all()


def test_nothing_and_infinities():
    from kore_amd import rope
    with rope.Rope(rope.Config(8)) as r:
        r.apply_dev("f32", 0, 2, 8, None, None, None)
        r.sync()
    x = torch.zeros(1, 2, 8)
    x[0, 0, 1], x[0, 1, 2] = math.inf, math.nan
    got = _apply(x, [3], rope.Config(8), 2, 8, "f32")
    bad = ~torch.isfinite(got)
    assert bad[0, 0].tolist() == [False, True, False, False, False, True, False, False]
    assert bad[0, 1].tolist() == [False, False, True, False, False, False, True, False]
