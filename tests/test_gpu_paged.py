"""The paged cache: append and attention against plain implementations in 64 bits."""
import math

import numpy as np
import pytest
import torch

from tests.paged_ref import DTYPE, PAIRS, UNIT, Case, check_rows, rope_bound, rope_freqs, rope_rows, to64

pytestmark = pytest.mark.gpu

GEO = [(14, 2, 64), (28, 4, 128), (33, 3, 96)]


def _append(c, kv, q_out="out", layer=0, with_q=True, stream=None):
    kv.append_dev(layer, c.batch(), c.dtype, c.ptr("k"), c.ptr("v"), q=c.ptr("q") if with_q else None,
                  q_out=c.ptr(q_out) if with_q else None, k_stride=c.step("k"), v_stride=c.step("v"),
                  q_stride=c.step("q"), q_out_stride=c.step(q_out), stream=stream)
    if stream is None:
        kv.sync()


# ---- append --------------------------------------------------------------------

@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("nh,nkv,hd,rot,layout,ps,pad,off", [
    (14, 2, 64, 64, "half", 16, 0, 0), (28, 4, 128, 128, "half", 64, 8, 8), (6, 3, 96, 32, "interleaved", 32, 4, 4),
    (5, 5, 40, 18, "interleaved", 256, 3, 1), (2, 1, 256, 256, "half", 128, 1, 1), (4, 2, 72, 0, "half", 16, 0, 0),
])
def test_append(dtype, cache, nh, nkv, hd, rot, layout, ps, pad, off):
    """Rows of several sequences, one without rows, one that starts in the middle of a page, one longer than the table's
    pages for it, one with an unmapped page; rows behind the last sequence; every other slot keeps its bits."""
    from kore_amd import rope
    lens = [(1, 1), (0, 5), (3, ps + 1), (2 * ps + 3, 2 * ps + 3), (1, 4 * ps), (4, 2)]
    c = Case(lens, nh, nkv, hd, ps, dtype, cache, seed=hd, extra_rows=2, row_pad=pad, row_off=off, n_layer=2)
    c.pages[3, 1] = -1
    c.pages[4, 3] = c.n_pages          # not a page
    c.up()
    cfg = rope.Config(rot, layout, scaling="yarn", factor=4.0, orig_ctx=64) if rot else None
    before = {k: c.d[k].clone() for k in ("k_pool", "v_pool")}
    with c.handle(cfg) as kv:
        _append(c, kv, layer=1)
    f, m = rope_freqs(rot, scaling="yarn", factor=4.0, orig_ctx=64) if rot else (np.zeros(0, np.float32), 1.0)
    q, clean = c.rows("out", nh)
    assert clean and (q[c.used:] == 77.0).all(), "rows behind the last sequence are left"
    got_k, got_v = to64(c.d["k_pool"]), to64(c.d["v_pool"])
    mark = torch.zeros(c.d["k_pool"].shape, dtype=torch.bool)
    for s, (n, _) in enumerate(lens):
        for i in range(n):
            row, pos = int(c.starts[s]) + i, int(c.kv_len[s]) - n + i
            want, size = rope_rows(to64(c.q[row:row + 1]), [pos], f, m, layout)
            assert (np.abs(to64(q[row:row + 1]) - want) <= rope_bound(want, size, dtype)).all()
            page = int(c.pages[s, pos // ps]) if 0 <= pos < c.stride * ps else -1
            if not 0 <= page < c.n_pages:
                continue
            mark[1, page, :, pos % ps] = True
            want, size = rope_rows(to64(c.k[row:row + 1]), [pos], f, m, layout)
            assert (np.abs(got_k[1, page, :, pos % ps] - want[0]) <= rope_bound(want, size, cache)[0]).all()
            assert torch.equal(c.d["v_pool"][1, page, :, pos % ps].cpu(), c.v[row].to(DTYPE[cache]))
    for k in ("k_pool", "v_pool"):
        a, b = (t.cpu().view(torch.int32 if cache == "f32" else torch.int16)[~mark] for t in (before[k], c.d[k]))
        assert torch.equal(a, b), "a slot of no row was written"


def test_append_in_place_and_without_q():
    from kore_amd import rope
    c = Case([(3, 9), (1, 17)], 6, 2, 64, 16, "f32", "f16", seed=3).up()
    d = Case([(3, 9), (1, 17)], 6, 2, 64, 16, "f32", "f16", seed=3).up()
    with c.handle(rope.Config(64)) as kv, d.handle(rope.Config(64)) as kv2:
        _append(c, kv)
        _append(d, kv2, q_out="q")
        assert torch.equal(c.rows("out", 6)[0], d.rows("q", 6)[0])
        d.d["k_pool"].zero_()
        torch.cuda.synchronize()
        _append(d, kv2, with_q=False)
    a, b = c.d["k_pool"].cpu(), d.d["k_pool"].cpu()
    assert torch.equal(a[b != 0], b[b != 0]) and int((b != 0).sum()) >= 4 * 2 * 64 - 8
    assert torch.equal(c.rows("out", 6)[0], d.rows("q", 6)[0])


# ---- attention -------------------------------------------------------------------

LENS = {
    "one_token": [(1, 1)],
    "decode": [(1, 5), (1, 64), (1, 17), (0, 0), (1, 300), (1, 16), (1, 129)],
    "chunks": [(3, 3), (40, 75), (0, 9), (1, 130), (17, 200), (64, 64)],
    "past_the_rows": [(5, 3), (1, 0), (2, 2)],      # rows before position 0 see nothing
    "verify": [(4, 70), (2, 33), (5, 5)],
}


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("nh,nkv,hd", GEO + [(4, 4, 40), (8, 1, 256), (40, 2, 72), (2, 2, 8)])
@pytest.mark.parametrize("lens", sorted(LENS))
def test_attend(dtype, cache, nh, nkv, hd, lens):
    c = Case(LENS[lens], nh, nkv, hd, 16, dtype, cache, seed=nh + hd, extra_rows=3).up()
    with c.handle() as kv:
        c.attend(kv)
    got, clean = c.rows("out", nh)
    assert clean and (got[c.used:] == 77.0).all()
    check_rows(c, got, *c.exact())


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
def test_page_sizes(dtype, cache, ps):
    c = Case([(1, 2 * ps + 5), (70, 3 * ps - 1 + 70), (1, ps)], 12, 2, 128, ps, dtype, cache, seed=ps).up()
    with c.handle() as kv:
        for max_q in (None, 0, 1, 1000):    # a wrong hint changes the kernel, not the result
            c.d["out"].fill_(55.0)
            torch.cuda.synchronize()
            c.attend(kv, max_q=max_q)
            check_rows(c, c.rows("out", 12)[0], *c.exact(), "max_q %s" % max_q)


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 100, 1000])
def test_windows(dtype, cache, window):
    c = Case([(1, 150), (50, 260), (130, 130), (3, 2)], 6, 2, 64, 32, dtype, cache, seed=window).up()
    with c.handle() as kv:
        c.attend(kv, window=window)
    check_rows(c, c.rows("out", 6)[0], *c.exact(window=window))


@pytest.mark.parametrize("dtype,cache", PAIRS)
def test_long_contexts_are_split(dtype, cache):
    """Few rows over many keys: the work of a row is split over workgroups and joined, ragged and in one piece."""
    c = Case([(1, 4001), (1, 70), (9, 3333)], 8, 2, 128, 64, dtype, cache, seed=1).up()
    with c.handle() as kv:
        c.attend(kv)
        check_rows(c, c.rows("out", 8)[0], *c.exact())
        first = c.d["out"].clone()
        c.d["out"].fill_(0)
        torch.cuda.synchronize()
        c.attend(kv)
    assert torch.equal(first[:, :1024], c.d["out"][:, :1024]), "the same call gives the same bits"


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("nh,nkv,hd", [(14, 2, 64), (28, 4, 128), (33, 3, 96)])
@pytest.mark.parametrize("window", [0, 50])
def test_short_tables(dtype, cache, nh, nkv, hd, window):
    """A few tokens over a table of few pages: tiles in one piece on either side of where splitting begins, some without a key."""
    for keys in (65, 112, 240, 448, 500, 1000):
        c = Case([(1, keys), (1, 1), (2, keys // 2), (1, 0), (1, 7)], nh, nkv, hd, 16, dtype, cache, seed=keys, extra_rows=1)
        c.kv_len[1] = 10 ** 6 if keys == 240 else 1     # past the table: its last positions are all there are
        c.up()
        with c.handle() as kv:
            c.attend(kv, window=window)
        got = c.rows("out", nh)[0]
        assert (got[c.used:] == 77.0).all()
        check_rows(c, got, *c.exact(window=window), "%d keys" % keys)


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("new,n_seq,kv", [(1, 75, (1, 120)), (80, 6, (80, 200))])
def test_a_long_sequence_among_many_tiles(dtype, cache, new, n_seq, kv):
    """Tiles enough to fill the card, those of two sequences longer than the rest by far: theirs alone are split."""
    rng = np.random.default_rng(n_seq)
    lens = [(new, int(rng.integers(*kv))) for _ in range(n_seq)]
    lens.insert(2, (1, 3001))
    lens.append((2, 2750))
    c = Case(lens, 28, 4, 64, 64, dtype, cache, seed=n_seq, extra_rows=1).up()
    with c.handle() as kv_:
        ws = torch.full((kv_.workspace_bytes() + 4096,), 9, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        c.attend(kv_, workspace=ws.data_ptr())
    got = c.rows("out", 28)[0]
    assert (got[c.used:] == 77.0).all() and (ws[-4096:] == 9).all()
    check_rows(c, got, *c.exact())


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("nh,nkv,hd,ps,n_seq", [(28, 4, 128, 16, 70), (6, 1, 64, 32, 200)])
def test_many_sequences(dtype, cache, nh, nkv, hd, ps, n_seq):
    rng = np.random.default_rng(n_seq)
    lens = [(int(rng.integers(0, 3)), int(rng.integers(1, 90))) for _ in range(n_seq)]
    c = Case(lens, nh, nkv, hd, ps, dtype, cache, seed=n_seq, extra_rows=1).up()
    with c.handle() as kv:
        c.attend(kv)
    got = c.rows("out", nh)[0]
    assert (got[c.used:] == 77.0).all()
    check_rows(c, got, *c.exact())


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("pad,off", [(8, 8), (3, 1), (0, 4), (2, 2)])
def test_strides_and_alignment(dtype, cache, pad, off):
    c = Case([(1, 40), (20, 50)], 4, 2, 64, 16, dtype, cache, seed=off, row_pad=pad, row_off=off, extra_rows=1).up()
    with c.handle() as kv:
        c.attend(kv)
    got, clean = c.rows("out", 4)
    assert clean and (got[c.used:] == 77.0).all()
    check_rows(c, got, *c.exact())


@pytest.mark.parametrize("dtype,cache", PAIRS)
def test_pages_that_are_none(dtype, cache):
    """Holes (-1), numbers past the pool, the largest and smallest int: their positions are not attended; a sequence longer
    than its row of the table ends there; all pages gone: zeros."""
    c = Case([(1, 100), (20, 90), (1, 64), (1, 48)], 6, 2, 64, 16, dtype, cache, seed=6)
    c.pages[0, 2], c.pages[0, 4] = -1, c.n_pages
    c.pages[1, 0], c.pages[1, 5] = 2 ** 31 - 1, -2 ** 31
    c.pages[2, :] = -1
    c.kv_len[3] = 5000
    c.up()
    with c.handle() as kv:
        for max_q in (1, 20):
            c.attend(kv, max_q=max_q)
            got = c.rows("out", 6)[0]
            # sequence 3: 5000 positions, of which the table holds the first 7 pages, of which 3 are pages
            check_rows(c, got, *c.exact())
            assert (got[21] == 0).all()


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("max_q", [1, 64])
def test_values_that_a_row_does_not_attend(dtype, cache, bad, max_q):
    """K and V of later positions, and of those before the window, are infinite or NaN: the other rows do not notice."""
    for window in (0, 40):
        c = Case([(30, 70), (5, 5), (1, 33)], 6, 2, 64, 16, dtype, cache, seed=9)
        for s, p in ((0, 69), (0, 55), (1, 4), (1, 2)) + (((0, 1), (0, 7)) if window else ()):
            c.k_pool[0, c.pages[s, p // 16], 0, p % 16, 3] = bad
            c.v_pool[0, c.pages[s, p // 16], 1, p % 16, 5] = bad
        c.up()
        with c.handle() as kv:
            c.attend(kv, window=window, max_q=max_q)
        got = c.rows("out", 6)[0]
        want, bound = c.exact(window=window)
        fine = np.isfinite(want).all(-1)
        # rows of kv-head 1 that attend no bad V: positions 40..54 (with the window 47..54, the first ones see 1 and 7), 0..1, 32
        assert fine[:, 3:].any(-1).sum() == (11 if window else 18)
        g = to64(got)
        assert (np.abs(g - want)[fine] <= bound[fine]).all()
        # a V that a row attends reaches it, in its own dim alone
        v_rows = ~np.isfinite(want[:, 3:]).all(-1)
        assert np.array_equal(np.isfinite(g[:, 3:]), np.isfinite(want[:, 3:])) and v_rows.any()
        # a K of NaN or +-inf that a row attends: what softmax makes of its score
        assert np.array_equal(np.isnan(g[:, :3]), np.isnan(want[:, :3]))


@pytest.mark.parametrize("dtype,cache", PAIRS)
def test_large_and_small_scores(dtype, cache):
    """Scores of hundreds (one key takes all) and of nothing; a large sink with a tiny V beside many small weights."""
    for size in (6.0, 1e-3):
        c = Case([(1, 500), (40, 300)], 6, 2, 128, 32, dtype, cache, seed=12, size=size).up()
        with c.handle() as kv:
            c.attend(kv)
        check_rows(c, c.rows("out", 6)[0], *c.exact())
    c = Case([(1, 500), (40, 300)], 6, 2, 128, 32, dtype, cache, seed=13, size=0.5)
    for s in (0, 1):
        c.k_pool[0, c.pages[s, 0], :, 0] = 0
        c.k_pool[0, c.pages[s, 0], :, 0, 0] = 40.0
        c.v_pool[0, c.pages[s, 0], :, 0] *= 1e-3
    c.q[:, :, 0] = 3.0
    c.up()
    with c.handle() as kv:
        c.attend(kv)
    check_rows(c, c.rows("out", 6)[0], *c.exact())


@pytest.mark.parametrize("dtype,cache", PAIRS)
def test_out_in_the_place_of_q(dtype, cache):
    for lens in ([(1, 900), (1, 40)], [(40, 300), (2, 9)]):
        c = Case(lens, 6, 2, 64, 16, dtype, cache, seed=8, extra_rows=1).up()
        with c.handle() as kv:
            c.attend(kv)
            kv.attend_dev(0, c.batch(), dtype, c.ptr("q"), c.ptr("q"))
            kv.sync()
        assert torch.equal(c.d["q"][:c.used], c.d["out"][:c.used]) and torch.equal(c.rows("q", 6)[0][c.used:], c.q[c.used:])


@pytest.mark.parametrize("dtype,cache", [p for p in PAIRS if p[1] != "f16"])
def test_values_near_the_largest(dtype, cache):
    """V near fp32's largest value: a weighted mean of them is finite, and so is what is summed on the way (V up to 2^120,
    300 keys of weights up to 1)."""
    c = Case([(1, 300), (40, 280)], 6, 2, 64, 16, dtype, cache, seed=10)
    c.v_pool = (c.v_pool.double().clamp(-4, 4) * 2.0 ** 117).to(c.v_pool.dtype)
    c.up()
    with c.handle() as kv:
        for max_q in (1, 100):
            c.attend(kv, max_q=max_q)
            got, want, bound = to64(c.rows("out", 6)[0]), *c.exact()
            assert np.isfinite(got).all() and (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("dtype,cache", [p for p in PAIRS if p[0] == "f32"])
def test_tiny_and_huge_q(dtype, cache):
    """Rows of q of 1e-38 (scores of nothing: the mean of V) and of 1e30 against K of 1e-30 beside ordinary ones, with masked
    keys in the same tiles."""
    c = Case([(1, 70), (30, 90)], 6, 2, 64, 16, dtype, cache, seed=14)
    c.q[::3] *= 1e-38
    c.q[1::3, 2:] *= 1e30
    if cache != "f16":
        c.k_pool[0, :, 1] *= 1e-30
    c.up()
    with c.handle() as kv:
        for max_q in (1, 100):
            c.attend(kv, max_q=max_q)
            got, want, bound = to64(c.rows("out", 6)[0]), *c.exact()
            # an fp16 K cannot be that small: those rows' scores of 1e30 leave one key, wherever its score is the largest by far
            fine = np.isfinite(bound) & (bound < 1)
            assert np.isfinite(got).all() and (np.abs(got - want)[fine] <= bound[fine]).all() and fine.mean() > 0.5


def test_scale():
    c = Case([(1, 50), (30, 60)], 4, 2, 64, 16, "f32", "f32", seed=2).up()
    with c.handle() as kv:
        for scale in (0.03, 1.0):
            c.attend(kv, scale=scale)
            check_rows(c, c.rows("out", 4)[0], *c.exact(scale=scale))


def test_shared_pages_and_layers():
    """Two sequences that share their first pages, in the second of two layers."""
    c = Case([(1, 70), (20, 90)], 6, 2, 64, 16, "f32", "bf16", seed=5, n_layer=2)
    c.pages[1, :3] = c.pages[0, :3]
    c.up()
    with c.handle() as kv:
        for layer in (0, 1):
            c.attend(kv, layer=layer)
            check_rows(c, c.rows("out", 6)[0], *c.exact(layer=layer))


# ---- both together -----------------------------------------------------------------

@pytest.mark.parametrize("cache", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd", [(14, 2, 64), (28, 4, 128)])
def test_steps_against_the_contiguous_cache(cache, nh, nkv, hd):
    """Two sequences grown together, a prompt's chunks and then tokens, each step an append and an attention: against
    KoreAttn over each sequence alone.  A 16-bit cache rounds K and V: a score moves by up to u sum|q k|, and with it the
    weights and V."""
    import kore_amd
    from kore_amd import paged, rope
    rng = np.random.default_rng(hd)
    total, ps, E, kvd = [90, 61], 16, nh * hd, nkv * hd
    data = [{n: rng.standard_normal((t, w)).astype(np.float32) for n, w in (("q", E), ("k", kvd), ("v", kvd))} for t in total]
    want = []
    for t, x in zip(total, data):
        with kore_amd.KoreAttn(1, t, nh, nkv, hd, 1e6) as a:
            want.append(a.prefill(0, 0, x["q"], x["k"], x["v"]))
    table = rng.permutation(12).astype(np.int32).reshape(2, 6)
    pages = torch.from_numpy(table).cuda()
    tol = {"f32": 1e-4, "f16": 2.0 ** -7, "bf16": 2.0 ** -4}[cache]
    with paged.PagedKV(1, 12, ps, nh, nkv, hd, cache, rope.Config(hd)) as kv:
        done = [0, 0]
        for step in [(33, 7), (17, 1), (1, 0), (0, 13), (1, 1), (38, 39)]:
            new = [min(n, t - d) for n, t, d in zip(step, total, done)]
            rows = {n: torch.from_numpy(np.concatenate([x[n][d:d + m] for x, d, m in zip(data, done, new)])).cuda() for n in "qkv"}
            done = [d + m for d, m in zip(done, new)]
            starts = torch.tensor([0, new[0], sum(new)], dtype=torch.int32).cuda()
            lens = torch.tensor(done, dtype=torch.int32).cuda()
            out = torch.empty_like(rows["q"])
            torch.cuda.synchronize()
            b = paged.Batch(2, sum(new), starts.data_ptr(), lens.data_ptr(), pages.data_ptr(), 6, max(new))
            kv.append_dev(0, b, "f32", rows["k"].data_ptr(), rows["v"].data_ptr(), rows["q"].data_ptr(), rows["q"].data_ptr())
            kv.attend_dev(0, b, "f32", rows["q"].data_ptr(), out.data_ptr())
            kv.sync()
            w = np.concatenate([x[d - m:d] for x, d, m in zip(want, done, new)])
            assert np.abs(out.cpu().numpy() - w).max() <= tol * np.abs(w).max()
        assert done == total


@pytest.mark.parametrize("dtype,cache", [("f32", "f32"), ("f32", "bf16"), ("f16", "f16")])
def test_graph_replays(dtype, cache):
    """A step captured once and replayed with other rows, lengths and pages, the program's own work between the replays: each
    equals the eager call's bits.  The captured calls have a workspace of their own."""
    from kore_amd import rope
    lens = [(1, 1500), (12, 300), (1, 2)]
    cases = [Case(lens, 12, 2, 128, 32, dtype, cache, seed=i, extra_rows=1).up() for i in range(4)]
    for i, c in enumerate(cases[1:]):
        c.kv_len = c.kv_len - np.asarray([97 * i, 3 * i, 0], np.int32)
        c.d["kv_len"].copy_(torch.from_numpy(c.kv_len))
    c = cases[0]
    with c.handle(rope.Config(128)) as kv:
        ws = torch.empty(kv.workspace_bytes(), dtype=torch.uint8, device="cuda")
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()

        def step(st, w):
            _append(c, kv, q_out="q", stream=st)
            c.attend(kv, workspace=w, stream=st)

        step(stream.cuda_stream, ws.data_ptr())
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            step(torch.cuda.current_stream().cuda_stream, ws.data_ptr())
        for other in cases[1:] + cases[1:2]:
            names = ("k_pool", "v_pool", "pages", "kv_len", "starts", "q", "k", "v")

            def fill():
                for n in names:
                    c.d[n].copy_(other.d[n])
                c.d["out"].fill_(77.0)
                torch.cuda.synchronize()

            fill()
            step(stream.cuda_stream, None)
            stream.synchronize()
            eager = {n: c.d[n].clone() for n in ("out", "k_pool", "v_pool", "q")}
            fill()
            g.replay()
            torch.cuda.synchronize()
            for n, t in eager.items():
                assert torch.equal(t.view(torch.uint8), c.d[n].view(torch.uint8)), n
        del g


def test_two_streams_with_their_own_workspaces():
    cs = [Case([(1, 3000), (5, 700)], 16, 2, 128, 64, "f32", "f16", seed=i).up() for i in range(2)]
    with cs[0].handle() as a, cs[1].handle() as b:
        want = []
        for c, kv in zip(cs, (a, b)):
            c.attend(kv)
            want.append(c.d["out"].clone())
        streams = [torch.cuda.Stream() for _ in cs]
        spaces = [torch.empty(a.workspace_bytes(), dtype=torch.uint8, device="cuda") for _ in cs]
        for c in cs:
            c.d["out"].fill_(0)
        torch.cuda.synchronize()
        for _ in range(3):
            for c, kv, s, w in zip(cs, (a, b), streams, spaces):
                c.attend(kv, workspace=w.data_ptr(), stream=s.cuda_stream)
        torch.cuda.synchronize()
        for c, w in zip(cs, want):
            assert torch.equal(c.d["out"], w)


def test_a_cache_past_32_bits():
    """Slots whose offset in the pool passes 2^32 bytes and 2^31 elements."""
    from kore_amd import paged
    nkv, hd, ps = 8, 128, 256
    n_pages = (2 ** 31 + 2 ** 28) // (nkv * hd * ps)
    c = Case([(1, 300), (40, 280)], 16, nkv, hd, ps, "f16", "f16", seed=4)
    with paged.PagedKV(1, n_pages, ps, 16, nkv, hd, "f16") as kv:
        assert kv.info().pool_bytes > 2 ** 32
        c.n_pages = n_pages
        far = {int(p): n_pages - 1 - i for i, p in enumerate(sorted(set(c.pages[c.pages >= 0].tolist())))}
        # rows in through append (which stores them as given), a sequence at a time: the whole of it is new
        full = [(kv_, kv_) for _, kv_ in c.lens]
        w = Case(full, 16, nkv, hd, ps, "f16", "f16", seed=5)
        for s, (n, _) in enumerate(full):
            p = np.arange(n)
            at = int(w.starts[s])
            w.k[at:at + n] = c.k_pool[0, c.pages[s, p // ps], :, p % ps]
            w.v[at:at + n] = c.v_pool[0, c.pages[s, p // ps], :, p % ps]
        c.up()
        w.up()
        table = np.vectorize(lambda x: far.get(int(x), -1))(c.pages).astype(np.int32)
        d_table = torch.from_numpy(table).cuda()
        torch.cuda.synchronize()
        wb = paged.Batch(2, w.n_tok, w.d["starts"].data_ptr(), w.d["kv_len"].data_ptr(), d_table.data_ptr(), c.stride, 300)
        kv.append_dev(0, wb, "f16", w.ptr("k"), w.ptr("v"))
        cb = paged.Batch(2, c.n_tok, c.d["starts"].data_ptr(), c.d["kv_len"].data_ptr(), d_table.data_ptr(), c.stride, 40)
        kv.attend_dev(0, cb, "f16", c.ptr("q"), c.ptr("out"))
        kv.sync()
    check_rows(c, c.rows("out", 16)[0], *c.exact())


@pytest.mark.parametrize("dtype,cache", [("f32", "f32"), ("f32", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("lens", [[(1, 90), (1, 1), (1, 400)], [(40, 90), (70, 70)]])
def test_rows_of_one_wide_buffer(dtype, cache, lens):
    """q, k, v and out side by side in one buffer's rows, as a fused projection writes them: q rotated in place, out beside it."""
    from kore_amd import rope
    c = Case(lens, 6, 2, 64, 16, dtype, cache, seed=12, extra_rows=1).up()
    E, D = 6 * 64, 2 * 64
    wide = torch.full((c.n_tok, 2 * E + 2 * D + 8), 33.0, dtype=DTYPE[dtype])
    wide[:, :E], wide[:, E:E + D], wide[:, E + D:E + 2 * D] = (t.reshape(c.n_tok, -1) for t in (c.q, c.k, c.v))
    w = wide.cuda()
    size, step = w.element_size(), w.shape[1]
    p = [w.data_ptr() + size * at for at in (0, E, E + D, E + 2 * D)]
    torch.cuda.synchronize()
    with c.handle(rope.Config(64)) as kv:
        kv.append_dev(0, c.batch(), dtype, p[1], p[2], p[0], p[0], step, step, step, step)
        kv.attend_dev(0, c.batch(), dtype, p[0], p[3], step, step)
        kv.sync()
    got = w.cpu()
    assert torch.equal(got[:, E:E + 2 * D], wide[:, E:E + 2 * D]) and (got[:, -8:] == 33.0).all() and torch.equal(got[c.used:], wide[c.used:])
    c.q = got[:, :E].reshape(c.n_tok, 6, 64)   # rotated
    c.k_pool, c.v_pool = c.d["k_pool"].cpu(), c.d["v_pool"].cpu()
    f, m = rope_freqs(64)
    pos = np.concatenate([np.arange(kv - n, kv) for n, kv in lens])
    want, bound = rope_rows(wide[:c.used, :E].reshape(-1, 6, 64).double().numpy(), pos, f, m, "half")
    assert (np.abs(to64(c.q[:c.used]) - want) <= rope_bound(want, bound, dtype)).all()
    check_rows(c, got[:, E + 2 * D:2 * E + 2 * D].reshape(c.n_tok, 6, 64), *c.exact())


# ---- odd batches -----------------------------------------------------------------------

@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("max_q", [1, 64])
def test_scores_of_minus_infinity(dtype, cache, max_q):
    """Rows whose every attended score is -inf get zeros; one finite score is all of a row that has it."""
    c = Case([(3, 40), (20, 300), (1, 900)], 6, 2, 64, 16, dtype, cache, seed=3)
    c.q[..., 7] = c.q[..., 7].abs() + 0.5
    c.k_pool[..., 7] = -math.inf
    page = int(c.pages[1, 2])
    c.k_pool[0, page, 1, 5, 7] = 0.25   # sequence 1, position 37, kv-head 1
    c.up()
    with c.handle() as kv:
        c.attend(kv, max_q=max_q)
    got = to64(c.rows("out", 6)[0])
    v = to64(c.v_pool[0, page, 1, 5])
    assert (got[:3] == 0).all() and (got[23:] == 0).all() and (got[3:23, :3] == 0).all()
    # one weight, which divides out but for its parts' rounding, and the result's own
    assert (np.abs(got[3:23, 3:] - v) <= (UNIT[dtype] + 2.0 ** -20) * np.abs(v)).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("max_q", [1, 64])
def test_keys_of_every_size(hd, max_q):
    """An fp32 cache whose keys reach from the smallest subnormal to 2^40, some 0, and a channel 2^12 times the others that q
    hardly has."""
    c = Case([(20, 150), (1, 70)], 4, 2, hd, 16, "f32", "f32", seed=hd)
    rng = np.random.default_rng(hd)
    for s, (_, kv) in enumerate(c.lens):
        for p in range(kv):
            e = [-149, -140, -126, -100, -30, -3, 0, 0, 0][int(rng.integers(0, 9))] if p else 40
            c.k_pool[0, c.pages[s, p // 16], :, p % 16] *= 2.0 ** e
    c.k_pool[0, c.pages[0, 3], 0, 4] = 0.0
    c.k_pool[..., 5] *= 2.0 ** 12
    c.q[..., 5] *= 2.0 ** -12
    c.q[3] *= 2.0 ** -40     # a row that the largest key is nothing special to
    c.q[7] *= 2.0 ** -130
    c.up()
    with c.handle() as kv:
        c.attend(kv, max_q=max_q)
    check_rows(c, c.rows("out", 4)[0], *c.exact())


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("max_q", [1, 64])
def test_a_page_twice_in_a_sequence(dtype, cache, max_q):
    c = Case([(5, 200), (1, 130)], 6, 2, 64, 16, dtype, cache, seed=4)
    c.pages[0, 3] = c.pages[0, 9] = c.pages[0, 0]
    c.pages[1, :4] = c.pages[1, 5]
    c.up()
    with c.handle() as kv:
        c.attend(kv, max_q=max_q)
    check_rows(c, c.rows("out", 6)[0], *c.exact())


@pytest.mark.parametrize("dtype,cache", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("starts", [[0, 40] * 8 + [0], [40, 0] * 8 + [40], [-5, 100, -2 ** 31, 2 ** 31 - 1, 7] * 3 + [40, 40]])
@pytest.mark.parametrize("max_q", [1, 64])
def test_q_start_that_is_not_ascending(dtype, cache, starts, max_q):
    """Nothing of use comes out, and nothing but out, q_out, the slots of the table and the workspace is written."""
    c = Case([(40, 700)], 6, 2, 64, 16, dtype, cache, seed=5, extra_rows=2, row_pad=8, row_off=8)
    n_seq = len(starts) - 1
    c.lens = [(40, 700)] * n_seq
    c.pages = np.repeat(c.pages, n_seq, 0)
    c.kv_len = np.repeat(c.kv_len, n_seq, 0)
    c.starts = np.asarray(starts, np.int32)
    c.up()
    spare = [p for p in range(c.n_pages) if p not in set(c.pages[0])]
    with c.handle() as kv:
        ws = torch.full((kv.workspace_bytes() + 4096,), 9, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        c.attend(kv, max_q=max_q, workspace=ws.data_ptr())
        _append(c, kv)
    assert (ws[-4096:] == 9).all()
    assert c.rows("out", 6)[1] and torch.equal(c.d["q"], c.wide(c.q))
    for pool in ("k_pool", "v_pool"):
        assert torch.isnan(c.d[pool][0, spare]).all()


# ---- refusals ------------------------------------------------------------------------

def test_calls_refuse():
    """Every refusal leaves the buffers alone and says what it is."""
    from kore_amd import paged, rope
    c = Case([(2, 5)], 4, 2, 64, 16, "f32", "f16", seed=1).up()
    before = {n: t.clone() for n, t in c.d.items()}
    with c.handle(rope.Config(64)) as kv, rope.Rope(rope.Config(64)) as r:
        good = dict(layer=0, batch=c.batch(), dtype="f32", q=c.ptr("q"), out=c.ptr("out"))

        def batch(**kw):
            b = c.batch()
            for k, v in kw.items():
                setattr(b.struct, k, v)
            return b

        for kw, text in [
                (dict(layer=1), "layer 1"), (dict(layer=-1), "layer"), (dict(dtype="bf16"), "type"), (dict(q_stride=255), "stride"),
                (dict(out_stride=-256), "stride"), (dict(q_stride=1 << 60), "too large"), (dict(window=-1), "window"),
                (dict(scale=-1.0), "scale"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"),
                (dict(scale=1e-40), "scale"), (dict(scale=1e31), "scale"), (dict(out=c.ptr("q") + 4), "overlap"),
                (dict(workspace=8), "workspace"), (dict(q=None), "null"), (dict(out=None), "null"),
                (dict(q=c.ptr("q") + 2), "aligned"), (dict(batch=batch(n_seq=-1)), "negative"), (dict(batch=batch(n_tok=-1)), "negative"),
                (dict(batch=batch(max_q=-1)), "negative"), (dict(batch=batch(q_start=None)), "null"), (dict(batch=batch(kv_len=None)), "null"),
                (dict(batch=batch(pages=None)), "null"), (dict(batch=batch(pages_stride=0)), "pages_stride"),
                (dict(batch=batch(pages_stride=1 << 28)), "pages_stride"), (dict(batch=batch(n_tok=1 << 27)), "too large"),
                (dict(batch=batch(n_tok=(1 << 23) + 1)), "too large"), (dict(batch=batch(n_seq=(1 << 21) + 1)), "too large")]:
            with pytest.raises(paged.PagedError) as e:
                kv.attend_dev(**{**good, **kw})
            assert text in e.value.message, (kw, e.value.message)
        put = dict(layer=0, batch=c.batch(), dtype="f32", k=c.ptr("k"), v=c.ptr("v"), q=c.ptr("q"), q_out=c.ptr("out"))
        for kw, text in [
                (dict(k=None), "null"), (dict(v=None), "null"), (dict(q=None), "q_out without q"), (dict(q_out=None), "q without"),
                (dict(k_stride=127), "stride"), (dict(v_stride=0), "stride"), (dict(q_stride=1), "stride"), (dict(q_out_stride=1), "stride"),
                (dict(q_out=c.ptr("q") + 4), "overlap"), (dict(q_out=c.ptr("q"), q_out_stride=300), "overlap"), (dict(v=c.ptr("v") + 1), "aligned"),
                (dict(dtype="bf16"), "type"), (dict(layer=7), "layer")]:
            with pytest.raises(paged.PagedError) as e:
                kv.append_dev(**{**put, **kw})
            assert text in e.value.message, (kw, e.value.message)
        rot = dict(dtype="f32", n_tok=2, n_head=4, head_dim=64, x=c.ptr("q"), pos=c.d["kv_len"].data_ptr(), out=c.ptr("out"))
        for kw, text in [
                (dict(n_tok=-1), "n_tok"), (dict(n_head=0), "n_head"), (dict(head_dim=62), "head_dim"), (dict(head_dim=65), "head_dim"),
                (dict(head_dim=1026), "head_dim"), (dict(x_stride=10), "stride"), (dict(out_stride=10), "stride"), (dict(x=None), "null"),
                (dict(pos=None), "null"), (dict(out=c.ptr("q") + 4), "overlap"), (dict(out=c.ptr("out") + 3), "aligned"),
                (dict(n_tok=(1 << 23) + 1), "n_tok")]:
            with pytest.raises(rope.PagedError) as e:
                r.apply_dev(**{**rot, **kw})
            assert text in e.value.message, (kw, e.value.message)
        # nothing to do is no error
        kv.attend_dev(**{**good, "batch": batch(n_tok=0), "q": None, "out": None})
        kv.append_dev(**{**put, "batch": batch(n_seq=0), "k": None, "v": None})
        kv.sync()
        r.sync()
    torch.cuda.synchronize()
    for n, t in before.items():
        assert torch.equal(t.view(torch.uint8), c.d[n].view(torch.uint8)), n
