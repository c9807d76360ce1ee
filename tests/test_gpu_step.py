"""Steps of drafted tokens: their tables (plan), normalised heads, the store by slots, attention of trees, and what is kept,
each against a plain implementation; and all of them together."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from tests import step_ref
from tests.paged_ref import DTYPE, PAIRS, Case, check_rows, rope_freqs, to64

pytestmark = pytest.mark.gpu


def _dev(x, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x), dtype=dtype).cuda()


def _bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# ---- the plan --------------------------------------------------------------------

class Tables:
    """The arrays of a plan, each between guards."""

    def __init__(self, n_new, held, ps, n_tok=None, words=0, parent=None, n_free=None, stride=None, extra=3, seed=0, alias=False,
                 n_pages=None):
        rng = np.random.default_rng(seed)
        self.n_new, self.held, self.ps, self.words = list(n_new), list(held), ps, words
        had = [-(-max(h, 0) // ps) for h in held]
        has = [-(-max(h + n, 0) // ps) for n, h in zip(n_new, held)]
        self.stride = stride or max(has + had + [1])
        self.n_tok = sum(max(n, 0) for n in n_new) + 2 if n_tok is None else n_tok
        self.n_pages = sum(max(a, b) for a, b in zip(has, had)) + extra if n_pages is None else n_pages
        order = rng.permutation(self.n_pages)
        self.pages = np.full((len(held), self.stride), -1, np.int64)
        at = 0
        for s, h in enumerate(had):
            self.pages[s, :min(h, self.stride)] = order[at:at + min(h, self.stride)]
            at += h
        self.free = np.full(self.n_pages, -7, np.int64)
        self.free[:max(0, self.n_pages - at)] = order[at:]
        self.n_free = self.n_pages - at if n_free is None else n_free
        self.parent = parent
        self.alias = alias

    def up(self):
        def guarded(values, dtype=torch.int32):
            v = torch.as_tensor(np.asarray(values), dtype=dtype).reshape(-1)
            return torch.cat([torch.full((8,), 123, dtype=dtype), v, torch.full((8,), 123, dtype=dtype)]).cuda()

        n, t = len(self.held), self.n_tok
        d = {"n_new": guarded(self.n_new), "held": guarded(self.held), "pages": guarded(self.pages), "free": guarded(self.free),
             "n_free": guarded([self.n_free]), "q_start": guarded([99] * (n + 1)), "pos": guarded([99] * t),
             "slot": guarded([99] * t, torch.int64), "status": guarded([99]), "mask": guarded([99] * (t * self.words), torch.int64)}
        d["kv_len"] = d["held"] if self.alias else guarded([99] * n)
        d["n_free_out"] = d["n_free"] if self.alias else guarded([99])
        if self.words:
            d["parent"] = guarded(list(self.parent) + [55] * (t - len(self.parent)))
        self.d = d
        torch.cuda.synchronize()
        return self

    def ptr(self, name):
        t = self.d[name]
        return t.data_ptr() + 8 * t.element_size()

    def plan(self):
        from kore_amd import paged
        p = self.ptr
        return paged.Plan(len(self.held), self.n_tok, p("n_new"), p("held"), p("kv_len"), p("pages"), self.stride, p("free"), p("n_free"),
                          p("n_free_out"), p("q_start"), p("pos"), p("slot"), p("status"),
                          *((p("parent"), p("mask"), self.words) if self.words else ()))

    def handle(self):
        from kore_amd import paged
        return paged.PagedKV(1, self.n_pages, self.ps, 1, 1, 8, "f16")

    def get(self, name):
        t = self.d[name].cpu()
        assert (t[:8] == 123).all() and (t[-8:] == 123).all(), name + ": written outside"
        return t[8:-8].numpy()

    def check(self):
        want = step_ref.plan(self.n_new, self.held, self.pages.tolist(), self.free, self.n_free, self.n_tok, self.ps, self.n_pages,
                             self.parent, self.words)
        for name, out in (("status", "status"), ("kv_len", "kv_len"), ("n_free", "n_free_out"), ("q_start", "q_start"), ("pos", "pos"),
                          ("slot", "slot")):
            assert np.array_equal(self.get(out), want[name]), name
        assert np.array_equal(self.get("pages").reshape(len(self.held), -1) if self.held else want["pages"], want["pages"])
        if self.words:
            assert np.array_equal(self.get("mask").view(np.uint64).reshape(self.n_tok, self.words), want["mask"])
        assert np.array_equal(self.get("free"), self.free) and np.array_equal(self.get("n_new"), self.n_new)
        return int(want["status"][0])

    def run(self):
        self.up()
        with self.handle() as kv:
            kv.plan_dev(self.plan())
            kv.sync()
        return self.check()


def _lens(rng, n_seq, new, held):
    return [int(x) for x in rng.integers(0, new + 1, n_seq)], [int(x) for x in rng.integers(0, held + 1, n_seq)]


@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("ps", [16, 64, 256])
@pytest.mark.parametrize("n_seq,new,held", [(0, 0, 0), (1, 1, 0), (1, 1, 500), (3, 40, 40), (64, 32, 300), (65, 1, 70), (200, 30, 9),
                                            (1000, 8, 50), (1024, 4, 20), (1025, 2, 20), (2500, 5, 33), (3, 4000, 100), (9, 700, 1)])
def test_plan(n_seq, new, held, ps, alias):
    n_new, h = _lens(np.random.default_rng(n_seq + new), n_seq, new, held)
    assert Tables(n_new, h, ps, seed=ps, alias=alias).run() == 0


@pytest.mark.parametrize("words", [1, 2, 5, 16])
@pytest.mark.parametrize("n_seq,width", [(1, 0), (1, 3), (17, 5), (130, 2)])
def test_plan_of_trees(words, n_seq, width):
    """Trees of up to all the bits of a mask, chains (width 0) among them; parents that are none are roots."""
    rng = np.random.default_rng(words * 100 + n_seq)
    n_new = [int(x) for x in rng.integers(0, 64 * words + 1, n_seq)]
    n_new[0] = 64 * words
    parent = []
    for n in n_new:
        p = step_ref.tree(rng, n, width) if width else list(range(-1, n - 1))
        for i in rng.integers(0, max(n, 1), 2 if n > 8 and width else 0):
            p[i] = int(rng.choice([i, i + 3, -5, 2 ** 31 - 1, -2 ** 31]))
        parent += p
    assert Tables(n_new, [int(x) for x in rng.integers(0, 90, n_seq)], 16, words=words, parent=parent, seed=n_seq).run() == 0


@pytest.mark.parametrize("words,n_seq,most", [(1, 1500, 9), (2, 40, 128), (16, 9, 1024)])
def test_plan_of_trees_in_place(words, n_seq, most):
    """More sequences than one workgroup's threads, or many rows whose outputs take the inputs' place: two launches."""
    rng = np.random.default_rng(words)
    n_new = [int(x) for x in rng.integers(most // 2, most + 1, n_seq)]
    n_new[-1] = min(most, 64 * words)
    parent = [q for n in n_new for q in step_ref.tree(rng, n, max(1, n // 7))]
    held = [int(x) for x in rng.integers(0, 70, n_seq)]
    assert Tables(n_new, held, 16, words=words, parent=parent, seed=n_seq, alias=True).run() == 0


def test_plan_without_slack():
    """The last page and the last row of the buffers; a table's row that is full; a page of the table that is none."""
    assert Tables([16, 0, 5], [16, 33, 11], 16, n_tok=21, extra=0).run() == 0
    t = Tables([5, 3], [20, 30], 16, stride=3)
    t.pages[0, 1], t.pages[1, 1] = -1, t.n_pages + 4
    assert t.run() == 0


@pytest.mark.parametrize("big", [False, True])
@pytest.mark.parametrize("kw,status", [
    (dict(n_free=1), 1), (dict(n_free=0), 2), (dict(n_new=[-1, 5, 18]), -1), (dict(held=[4, -2, 15]), -1), (dict(stride=2), -1),
    (dict(n_tok=22), -1), (dict(n_free=-1), -1), (dict(n_free=100), -1), (dict(n_new=[2 ** 31 - 1, 2 ** 31 - 1, 2], n_tok=23, stride=8), -1),
    (dict(words=1, n_new=[65, 0, 0], n_tok=70, parent=list(range(-1, 64))), -1),
])
def test_plan_refused_on_the_device(kw, status, big):
    """Nothing is taken, and the tables are those of a step without rows: in one launch and in two."""
    kw = {"n_new": [4, 1, 18], "held": [4, 2, 15], "extra": 0, "n_pages": 8, **kw}
    if big and "n_tok" not in kw:
        kw["n_tok"] = 5000
    t = Tables(kw.pop("n_new"), kw.pop("held"), 16, **kw)
    assert t.run() == status


@pytest.mark.parametrize("n_tok", [0, 3])
@pytest.mark.parametrize("words", [0, 1])
@pytest.mark.parametrize("alias", [False, True])
def test_steps_without_sequences(n_tok, words, alias):
    """Arrays that hold nothing may be NULL, with free pages beside them."""
    from kore_amd import paged
    t = Tables([], [], 16, n_tok=n_tok, words=words, parent=[], alias=alias).up()
    p = t.ptr
    with t.handle() as kv:
        kv.plan_dev(paged.Plan(0, n_tok, None, None, None, None, 1, None, p("n_free"), p("n_free_out"), p("q_start"),
                               p("pos") if n_tok else None, p("slot") if n_tok else None, p("status"),
                               *((p("parent"), p("mask"), words) if words else ())))
        kv.sync()
        assert t.check() == 0
        assert t.get("n_free_out")[0] == t.n_free > 0
        kv.keep_dev(paged.Keep(0, n_tok, None, None, None, None, None, 1, free_pages=p("free"), n_free=p("n_free"),
                               n_free_out=p("n_free_out")))
        kv.keep_dev(paged.Keep(0, n_tok, None, None, None, None, None, 1))
        kv.sync()
    assert t.check() == 0


def test_plan_missing_is_whole():
    """What is missing of a step of many pages is their number."""
    t = Tables([4000, 4000], [0, 0], 16, n_free=100)
    assert t.run() == 400


# ---- heads that are normalised -------------------------------------------------------

def _wide(x, pad, off):
    n = x.shape[0]
    w = torch.full((n, off + x[0].numel() + pad), 3.0, dtype=x.dtype)
    w[:, off:off + x[0].numel()] = x.reshape(n, -1)
    return w.cuda()


def _inner(w, heads, hd, off):
    w = w.cpu()
    assert (w[:, :off] == 3.0).all() and (w[:, off + heads * hd:] == 3.0).all(), "written outside the rows"
    return w[:, off:off + heads * hd].reshape(-1, heads, hd)


def _norm(dtype, xs, pos, ws, cfg, pad=0, off=0, eps=1e-6, in_place=False):
    """kore_rope_norm_dev over one or two sets of rows [n][heads][hd]."""
    from kore_amd import rope
    hd = xs[0].shape[2]
    d = [_wide(x, pad, off) for x in xs]
    out = d if in_place else [torch.full_like(x, 3.0) for x in d]
    w = [None if x is None else torch.as_tensor(x, dtype=torch.float32).cuda() for x in ws]
    p = _dev(pos)
    torch.cuda.synchronize()
    with rope.Rope(cfg) as r:
        at = off * d[0].element_size()
        r.norm_dev(dtype, len(pos), hd, [rope.Heads(x.data_ptr() + at, y.data_ptr() + at, z.shape[1], hd,
                                                    norm=None if v is None else v.data_ptr(), x_stride=x.shape[1], out_stride=y.shape[1])
                                         for x, y, z, v in zip(d, out, xs, w)], p.data_ptr(), eps)
        r.sync()
    return [_inner(y, x.shape[1], hd, off) for x, y in zip(xs, out)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("n,nh,nkv,hd,rot,pad,off", [
    (1, 28, 4, 128, 128, 0, 0), (5, 6, 3, 96, 64, 4, 8), (7, 2, 1, 66, 34, 3, 1), (3, 5, 5, 40, 40, 1, 0), (2, 1, 1, 2, 2, 0, 0),
    (17, 14, 2, 64, 64, 0, 2), (2, 1, 1, 1024, 512, 0, 0), (300, 3, 1, 72, 48, 0, 0), (2, 2, 1, 1022, 512, 0, 0), (33, 33, 3, 96, 96, 0, 0),
    (2, 3, 1, 640, 512, 0, 0), (4, 9, 2, 8, 8, 0, 0), (1500, 4, 1, 64, 64, 0, 0), (1, 300, 7, 24, 16, 0, 0),
])
def test_norm_against_the_formula(dtype, layout, n, nh, nkv, hd, rot, pad, off):
    from kore_amd import rope
    rng = np.random.default_rng(hd + rot)
    xs = [torch.from_numpy(rng.standard_normal((n, h, hd)) * rng.choice([0.02, 1, 30], (n, h, 1))).to(DTYPE[dtype]) for h in (nh, nkv)]
    ws = [1 + 0.3 * rng.standard_normal(hd).astype(np.float32) for _ in range(2)]
    pos = rng.integers(0, 200000, n)
    pos[0] = 0
    got = _norm(dtype, xs, pos, ws, rope.Config(rot, layout), pad, off)
    f, m = rope_freqs(rot)
    for x, w, g in zip(xs, ws, got):
        want, size = step_ref.heads(to64(x), pos, f, m, layout, w, 1e-6)
        assert (np.abs(to64(g) - want) <= step_ref.heads_bound(want, size, dtype, True)).all()
    for a, b in zip(got, _norm(dtype, xs, pos, ws, rope.Config(rot, layout), pad, off, in_place=True)):
        assert _bits(a, b)
    one = _norm(dtype, xs[1:], pos, ws[1:], rope.Config(rot, layout), pad, off)
    assert _bits(one[0], got[1]), "a set alone"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,rot", [(128, 128), (66, 34)])
def test_norm_without_weights_is_the_rotation(dtype, hd, rot):
    """A set without weights has the bits of kore_rope_apply_dev; scaled frequencies and magnitude are the plan's."""
    from kore_amd import rope
    rng = np.random.default_rng(hd)
    cfg = rope.Config(rot, scaling="yarn", factor=4.0, orig_ctx=4096)
    xs = [torch.from_numpy(rng.standard_normal((9, h, hd))).to(DTYPE[dtype]) for h in (5, 2)]
    pos, w = rng.integers(0, 100000, 9), np.full(hd, 0.5, np.float32)
    got = _norm(dtype, xs, pos, [None, w], cfg)
    x, p = xs[0].cuda(), _dev(pos)
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    with rope.Rope(cfg) as r:
        r.apply_dev(dtype, 9, 5, hd, x.data_ptr(), p.data_ptr(), y.data_ptr())
        r.sync()
        f, m = r.freqs()
    assert _bits(got[0], y.cpu())
    want, size = step_ref.heads(to64(xs[1]), pos, f, float(m), "half", w, 1e-6)
    # (m is a double there, a float here: half a step of it more)
    assert (np.abs(to64(got[1]) - want) <= step_ref.heads_bound(want, size, dtype, True) + 2.0 ** -24 * size).all()


def test_norm_of_extremes():
    """Heads of values whose squares pass fp32's range either way, heads of zeros, a head with a NaN, rows without a position."""
    from kore_amd import rope
    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, 4, 64)).astype(np.float32)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2, 1] = 0
    x[3, 2, 5] = np.nan
    x[4, 0, 7] = np.inf
    x = torch.from_numpy(x)
    pos = [3, 0, 70000, 5, 9, -1]
    got, = _norm("f32", [x], pos, [np.ones(64, np.float32)], rope.Config(64), eps=1e-6)
    assert (got[5] == 3.0).all(), "a row without a position was written"
    f, m = rope_freqs(64)
    good = np.ones((6, 4), bool)
    good[3, 2] = good[4, 0] = good[5] = False
    want, size = step_ref.heads(to64(x), np.maximum(pos, 0), f, m, "half", np.ones(64), 1e-6)
    # (values of 1e-30 times 1 / sqrt(1e-6): far above the smallest float)
    assert (np.abs(to64(got) - want) <= step_ref.heads_bound(want, size, "f32", True))[good].all()
    assert (got[2, 1] == 0).all()


def test_norm_refuses():
    from kore_amd import rope
    x, y = torch.ones(4, 6 * 64, device="cuda"), torch.full((4, 6 * 64), 7.0, device="cuda")
    pos = _dev([0, 1, 2, 3])
    torch.cuda.synchronize()
    X, Y, P = x.data_ptr(), y.data_ptr(), pos.data_ptr()
    H = rope.Heads
    good = [H(X, Y, 4, 64, x_stride=384, out_stride=384), H(X + 1024, Y + 1024, 2, 64, x_stride=384, out_stride=384)]
    with rope.Rope(rope.Config(64)) as r:
        for kw, code, text in [
                (dict(sets=[]), -1, "null set"), (dict(eps=0.0), -1, "eps"), (dict(eps=math.nan), -1, "eps"),
                (dict(eps=math.inf), -1, "eps"), (dict(pos=None), -1, "pos"), (dict(pos=P + 2), -1, "pos"), (dict(hd=62), -1, "head_dim"),
                (dict(hd=65), -1, "head_dim"), (dict(hd=1026), -3, "head_dim"), (dict(n=-1), -1, "n_tok"), (dict(n=2 ** 23 + 1), -3, "n_tok"),
                (dict(sets=[H(X, Y, 0, 64)]), -1, "n_head"), (dict(sets=[H(X, Y, 4, 64, x_stride=255)]), -1, "stride"),
                (dict(sets=[H(X, Y, 4, 64, out_stride=255)]), -1, "stride"), (dict(sets=[H(0, Y, 4, 64)]), -1, "null"),
                (dict(sets=[H(X, 0, 4, 64)]), -1, "null"), (dict(sets=[H(X + 2, Y, 4, 64)]), -1, "aligned"),
                (dict(sets=[H(X, Y, 4, 64, norm=P + 1)]), -1, "norm"), (dict(sets=[H(X, X + 4, 4, 64)]), -1, "overlap"),
                (dict(sets=[good[0], H(X, Y + 1020, 2, 64, x_stride=384, out_stride=384)]), -1, "overlap"),
                (dict(sets=[good[0], H(X, X, 2, 64, x_stride=384, out_stride=384)]), -1, "overlap"),
                (dict(sets=[H(X, X, 4, 64, x_stride=384, out_stride=384), H(X + 512, Y, 2, 64, x_stride=384, out_stride=384)]), -1, "overlap")]:
            with pytest.raises(rope.PagedError, match=text) as e:
                r.norm_dev("f32", kw.get("n", 4), kw.get("hd", 64), kw.get("sets", good), kw.get("pos", P), kw.get("eps", 1e-6))
            assert e.value.code == code
        with pytest.raises(ValueError, match="sets"):
            r.norm_dev("f32", 4, 64, good * 2, P)
        r.norm_dev("f32", 0, 64, good, None)
        r.sync()
        assert (y == 7.0).all()
        r.norm_dev("f32", 4, 64, good, P)
        r.sync()
        assert (y != 7.0).all()


# ---- the store by slots ---------------------------------------------------------------

def _slots(c):
    """(positions, slots) of a Case's rows as its batch has them; rows behind the last sequence have none."""
    pos, slot = np.full(c.n_tok, -1, np.int32), np.full(c.n_tok, -1, np.int64)
    for s, (n, _) in enumerate(c.lens):
        for i in range(n):
            p, row = int(c.kv_len[s]) - n + i, int(c.starts[s]) + i
            page = int(c.pages[s, p // c.ps]) if 0 <= p < c.stride * c.ps else -1
            pos[row], slot[row] = p, page * c.ps + p % c.ps if 0 <= page < c.n_pages else -1
    return pos, slot


def _store(c, kv, pos, slot, ws=(None, None), q_out="out", layer=0, with_q=True, stream=None, eps=1e-6):
    from kore_amd import paged
    w = [None if x is None else torch.as_tensor(x, dtype=torch.float32).cuda() for x in ws]
    p, t = _dev(pos), _dev(slot, torch.int64)
    torch.cuda.synchronize()
    rows = paged.Rows(c.n_tok, p.data_ptr(), t.data_ptr(), *[None if x is None else x.data_ptr() for x in w], norm_eps=eps)
    kv.append_rows_dev(layer, rows, c.dtype, c.ptr("k"), c.ptr("v"), q=c.ptr("q") if with_q else None,
                       q_out=c.ptr(q_out) if with_q else None, k_stride=c.step("k"), v_stride=c.step("v"), q_stride=c.step("q"),
                       q_out_stride=c.step(q_out), stream=stream)
    kv.sync()


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("nh,nkv,hd,rot,layout,ps,pad,off", [
    (14, 2, 64, 64, "half", 16, 0, 0), (28, 4, 128, 128, "half", 64, 8, 8), (6, 3, 96, 32, "interleaved", 32, 4, 4),
    (5, 5, 40, 18, "interleaved", 256, 3, 1), (2, 1, 256, 256, "half", 128, 1, 1), (4, 2, 72, 0, "half", 16, 0, 0),
])
def test_store(dtype, cache, nh, nkv, hd, rot, layout, ps, pad, off):
    """Without norms, the bits of kore_paged_append_dev; with them, the formula; slots that are none, rows without a position,
    a position that is not the slot's; every other slot keeps its bits."""
    from kore_amd import rope
    lens = [(1, 1), (0, 5), (3, ps + 1), (2 * ps + 3, 2 * ps + 3), (1, 4 * ps)]
    make = lambda: Case(lens, nh, nkv, hd, ps, dtype, cache, seed=hd, extra_rows=2, row_pad=pad, row_off=off, n_layer=2).up()  # noqa: E731
    c, d = make(), make()
    cfg = rope.Config(rot, layout, scaling="yarn", factor=4.0, orig_ctx=64) if rot else None
    pos, slot = _slots(c)
    with c.handle(cfg) as kv, d.handle(cfg) as kv2:
        kv.append_dev(1, c.batch(), dtype, c.ptr("k"), c.ptr("v"), c.ptr("q"), c.ptr("out"), c.step("k"), c.step("v"), c.step("q"),
                      c.step("out"))
        kv.sync()
        _store(d, kv2, pos, slot, layer=1)
    for n in ("k_pool", "v_pool", "out"):
        assert _bits(c.d[n], d.d[n]), n
    rng = np.random.default_rng(7)
    ws = [1 + 0.3 * rng.standard_normal(hd).astype(np.float32) for _ in range(2)]
    c = make()
    pos[1:] += rng.integers(0, 50, len(pos) - 1) * (pos[1:] >= 0)
    slot[2], slot[4] = -5, c.n_pages * ps
    pos[3] = -1
    before = {k: c.d[k].clone() for k in ("k_pool", "v_pool")}
    with c.handle(cfg) as kv:
        _store(c, kv, pos, slot, ws, layer=1)
    f, m = rope_freqs(rot, scaling="yarn", factor=4.0, orig_ctx=64) if rot else (np.zeros(0, np.float32), 1.0)
    q, clean = c.rows("out", nh)
    assert clean and (q[pos < 0] == 77.0).all()
    got_k = to64(c.d["k_pool"])
    mark = torch.zeros(c.d["k_pool"].shape, dtype=torch.bool)
    for row in np.flatnonzero(pos >= 0):
        want, size = step_ref.heads(to64(c.q[row:row + 1]), [pos[row]], f, m, layout, ws[0], 1e-6)
        assert (np.abs(to64(q[row:row + 1]) - want) <= step_ref.heads_bound(want, size, dtype, True)).all()
        if not 0 <= slot[row] < c.n_pages * ps:
            continue
        page, at = int(slot[row]) // ps, int(slot[row]) % ps
        mark[1, page, :, at] = True
        want, size = step_ref.heads(to64(c.k[row:row + 1]), [pos[row]], f, m, layout, ws[1], 1e-6)
        assert (np.abs(got_k[1, page, :, at] - want[0]) <= step_ref.heads_bound(want, size, cache, True)[0]).all()
        assert torch.equal(c.d["v_pool"][1, page, :, at].cpu(), c.v[row].to(DTYPE[cache]))
    for k in ("k_pool", "v_pool"):
        a, b = (t.cpu().view(torch.int32 if cache == "f32" else torch.int16)[~mark] for t in (before[k], c.d[k]))
        assert torch.equal(a, b), "a slot of no row was written"


def test_store_in_place_and_without_q():
    from kore_amd import rope
    w = [np.linspace(0.5, 2, 64, dtype=np.float32)] * 2
    c, d, e = (Case([(3, 9), (1, 17)], 6, 2, 64, 16, "f32", "f16", seed=3).up() for _ in range(3))
    with c.handle(rope.Config(64)) as a, d.handle(rope.Config(64)) as b, e.handle(rope.Config(64)) as f:
        _store(c, a, *_slots(c), w)
        _store(d, b, *_slots(d), w, q_out="q")
        _store(e, f, *_slots(e), w, with_q=False)
    assert _bits(c.d["out"], d.d["q"]) and (e.d["out"] == 77.0).all()
    for n in ("k_pool", "v_pool"):
        assert _bits(c.d[n], d.d[n]) and _bits(c.d[n], e.d[n])


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("nh,nkv,hd", [(6, 2, 64), (5, 1, 72), (3, 3, 40)])
def test_rows_of_q_k_and_v_side_by_side(dtype, cache, nh, nkv, hd):
    """One wide row holds all three, as one product leaves them: normalised and stored in place, the bits of rows of their own."""
    from kore_amd import paged, rope
    w = [np.linspace(0.5, 2, hd, dtype=np.float32)] * 2
    c, d = (Case([(3, 9), (20, 37), (1, 64)], nh, nkv, hd, 16, dtype, cache, seed=hd).up() for _ in range(2))
    pos, slot = _slots(c)
    E, kvd, n = nh * hd, nkv * hd, c.n_tok
    wide = torch.cat([x.reshape(n, -1) for x in (c.q, c.k, c.v)], 1).cuda()
    two = wide.clone()
    step, size = wide.shape[1], wide.element_size()
    at = lambda t, i: t.data_ptr() + i * size  # noqa: E731
    g, p, t = torch.from_numpy(w[0]).cuda(), _dev(pos), _dev(slot, torch.int64)
    torch.cuda.synchronize()
    with c.handle(rope.Config(hd)) as a, d.handle(rope.Config(hd)) as b, rope.Rope(rope.Config(hd)) as r:
        _store(c, a, pos, slot, w)
        rows = paged.Rows(n, p.data_ptr(), t.data_ptr(), g.data_ptr(), g.data_ptr(), norm_eps=1e-6)
        b.append_rows_dev(0, rows, dtype, at(wide, E), at(wide, E + kvd), q=at(wide, 0), q_out=at(wide, 0), k_stride=step, v_stride=step,
                          q_stride=step, q_out_stride=step)
        b.sync()
        r.norm_dev(dtype, n, hd, [rope.Heads(at(two, 0), at(two, 0), nh, hd, g.data_ptr(), step, step),
                                  rope.Heads(at(two, E), at(two, E), nkv, hd, g.data_ptr(), step, step)], p.data_ptr(), 1e-6)
        r.sync()
    for k in ("k_pool", "v_pool"):
        assert _bits(c.d[k], d.d[k])
    k_v = torch.cat([c.k.reshape(n, -1), c.v.reshape(n, -1)], 1)
    assert _bits(wide[:, :E].cpu(), c.rows("out", nh)[0].reshape(n, E)) and _bits(wide[:, E:].cpu(), k_v)
    assert _bits(two[:, :E], wide[:, :E]) and _bits(two[:, E + kvd:].cpu(), c.v.reshape(n, -1))
    got = two[:, E:E + kvd].cpu().reshape(n, nkv, hd)
    want, most = step_ref.heads(to64(c.k), pos, *rope_freqs(hd), "half", w[1], 1e-6)
    assert (np.abs(to64(got) - want) <= step_ref.heads_bound(want, most, dtype, True)).all()


# ---- attention of trees -------------------------------------------------------------

def _masks(c, rng, kind, words):
    """(masks [n_tok][words], positions).  tree: ancestors and the row itself; any: any new rows, or none."""
    mask, pos = np.zeros((c.n_tok, words), np.uint64), np.zeros(c.n_tok, np.int32)
    for s, (n, _) in enumerate(c.lens):
        at, h = int(c.starts[s]), int(c.kv_len[s]) - n
        parent = step_ref.tree(rng, n, max(1, n // 6)) if kind == "tree" else list(range(-1, n - 1))
        seen, depth = [], []
        for i in range(n):
            up = parent[i]
            depth.append(depth[up] + 1 if up >= 0 else 0)
            seen.append((seen[up] if up >= 0 else 0) | 1 << i)
            if kind == "any":
                seen[i] = int.from_bytes(rng.bytes(8 * words), "little") if rng.random() < 0.7 else 0
            pos[at + i] = h + depth[i]
            for w in range(words):
                mask[at + i, w] = seen[i] >> (64 * w) & (1 << 64) - 1
    return mask, pos


def _attend_tree(c, kv, mask, pos=None, layer=0, window=0, scale=0.0, max_q=None, workspace=None, stream=None):
    from kore_amd import paged
    m = _dev(mask.view(np.int64), torch.int64)
    p = None if pos is None else _dev(pos)
    torch.cuda.synchronize()
    t = paged.Tree(m.data_ptr(), mask.shape[1], None if p is None else p.data_ptr())
    kv.attend_tree_dev(layer, c.batch(max_q), t, c.dtype, c.ptr("q"), c.ptr("out"), q_stride=c.step("q"), out_stride=c.step("out"),
                       scale=scale, window=window, workspace=workspace, stream=stream)
    torch.cuda.synchronize()


TREES = {
    "token": [(1, 1)],
    "few": [(3, 5), (1, 64), (2, 17), (0, 0), (6, 300), (4, 4), (5, 129)],
    "trees": [(31, 31), (40, 75), (0, 9), (16, 130), (33, 200), (64, 64), (17, 1000)],
    "before_the_first": [(5, 3), (1, 0), (2, 2)],      # new rows before position 0 are not there
}


@pytest.mark.parametrize("kind", ["tree", "any"])
@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("nh,nkv,hd", [(14, 2, 64), (28, 4, 128), (33, 3, 96), (4, 4, 40), (8, 1, 256), (2, 2, 8)])
@pytest.mark.parametrize("lens", sorted(TREES))
def test_tree(dtype, cache, nh, nkv, hd, lens, kind):
    c = Case(TREES[lens], nh, nkv, hd, 16, dtype, cache, seed=nh + hd, extra_rows=3).up()
    mask, _ = _masks(c, np.random.default_rng(hd), kind, 1)
    with c.handle() as kv:
        _attend_tree(c, kv, mask)
    got, clean = c.rows("out", nh)
    assert clean and (got[c.used:] == 77.0).all()
    check_rows(c, got, *step_ref.tree_exact(c, mask))


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("ps,words", [(16, 2), (32, 3), (64, 4), (128, 16), (256, 4)])
def test_wide_trees(dtype, cache, ps, words):
    """Masks of several words, also more and fewer than the rows; any hint of the rows; pages that end inside a tile."""
    c = Case([(150, 2 * ps + 155), (70, 3 * ps - 1 + 70), (1, ps), (130, 130)], 6, 2, 128, ps, dtype, cache, seed=ps, extra_rows=1).up()
    mask, _ = _masks(c, np.random.default_rng(ps), "tree", words)
    want = step_ref.tree_exact(c, mask)
    with c.handle() as kv:
        for max_q in (None, 0, 1):
            c.d["out"].fill_(55.0)
            _attend_tree(c, kv, mask, max_q=max_q)
            check_rows(c, c.rows("out", 6)[0], *want, name=str(max_q))


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("window", [1, 5, 64, 200, 100000])
def test_trees_in_a_window(dtype, cache, window):
    """The window cuts what is cached, by each row's own position, and none of the new rows; positions outside the step's are
    taken to its ends."""
    c = Case([(20, 420), (3, 90), (64, 100), (1, 333), (9, 9)], 12, 2, 64, 32, dtype, cache, seed=window).up()
    mask, pos = _masks(c, np.random.default_rng(window), "tree", 1)
    pos[2], pos[25] = -4, 2 ** 31 - 1
    with c.handle() as kv:
        for max_q in (None, 1):
            _attend_tree(c, kv, mask, pos, window=window, max_q=max_q)
            check_rows(c, c.rows("out", 12)[0], *step_ref.tree_exact(c, mask, pos, window=window))


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("new", [2, 30])
def test_trees_over_long_contexts(dtype, cache, new):
    """Long sequences, whose keys are split over workgroups, and others too short for it; with a window as well."""
    c = Case([(new, 6000), (1, 20), (new, 2500)], 8, 2, 128, 64, dtype, cache, seed=new).up()
    mask, pos = _masks(c, np.random.default_rng(new), "tree", 1)
    with c.handle() as kv:
        _attend_tree(c, kv, mask)
        check_rows(c, c.rows("out", 8)[0], *step_ref.tree_exact(c, mask))
        _attend_tree(c, kv, mask, pos, window=3000)
        check_rows(c, c.rows("out", 8)[0], *step_ref.tree_exact(c, mask, pos, window=3000))


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("max_q", [1, 64])
def test_a_chain_is_causal(dtype, cache, max_q):
    """Masks of all rows up to each: kore_paged_attend_dev's rows."""
    c = Case([(12, 300), (5, 5), (1, 77)], 12, 2, 96, 16, dtype, cache, seed=1).up()
    mask, _ = _masks(c, np.random.default_rng(0), "chain", 1)
    with c.handle() as kv:
        _attend_tree(c, kv, mask, max_q=max_q)
    check_rows(c, c.rows("out", 12)[0], *c.exact())


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("max_q", [1, 64])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_new_rows_that_are_not_attended(dtype, cache, max_q, bad):
    """Infinities and NaN in K and V of new rows reach the rows whose masks name them, and no other; pages that are none."""
    c = Case([(9, 60), (20, 20), (3, 100)], 6, 2, 64, 16, dtype, cache, seed=5)
    rng = np.random.default_rng(5)
    mask, _ = _masks(c, rng, "tree", 1)
    out = [(0, 51 + 3), (1, 7), (2, 99)]     # (sequence, position): a new row each
    for s, p in out:
        page = int(c.pages[s, p // 16])
        c.v_pool[0, page, :, p % 16, 3] = bad
        i = p - (int(c.kv_len[s]) - c.lens[s][0])
        for row in range(int(c.starts[s]), int(c.starts[s + 1])):
            if row != int(c.starts[s]) + i:
                mask[row, 0] &= ~np.uint64(1 << i)
    c.pages[2, 1] = -1
    c.up()
    k2 = c.k_pool.clone()
    with c.handle() as kv:
        _attend_tree(c, kv, mask, max_q=max_q)
        got = c.rows("out", 6)[0]
        check_rows(c, got, *step_ref.tree_exact(c, mask))
        # the same in K: rows that do not attend the position are as they were
        for s, p in out:
            k2[0, int(c.pages[s, p // 16]), :, p % 16, 3] = bad
        c.d["k_pool"].copy_(k2)
        _attend_tree(c, kv, mask, max_q=max_q)
    other = c.rows("out", 6)[0]
    hit = np.zeros(c.n_tok, bool)
    for s, p in out:
        hit[int(c.starts[s]) + p - (int(c.kv_len[s]) - c.lens[s][0])] = True
    assert _bits(got[~hit], other[~hit])


def _tall(c, keys=131072):
    """The case with a table of so many keys, more than any sequence has: a step that may be as long as that takes tiles of
    128 rows, where a few of 16 would do for what it is (16 heads share a kv-head)."""
    c.pages = np.ascontiguousarray(np.pad(c.pages, ((0, 0), (0, keys // c.ps - c.stride)), constant_values=-1))
    c.stride = keys // c.ps
    return c


@pytest.mark.parametrize("kind", ["tree", "any"])
@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("nh,nkv,hd,ps", [(32, 2, 64, 16), (16, 1, 64, 32), (16, 1, 40, 128), (16, 1, 128, 16), (32, 2, 96, 64), (16, 1, 256, 16)])
@pytest.mark.parametrize("lens", ["few", "trees", "before_the_first"])
def test_trees_in_tall_tiles(dtype, cache, nh, nkv, hd, ps, lens, kind):
    c = _tall(Case(TREES[lens], nh, nkv, hd, ps, dtype, cache, seed=hd + ps, extra_rows=3)).up()
    mask, pos = _masks(c, np.random.default_rng(hd), kind, 1)
    with c.handle() as kv:
        _attend_tree(c, kv, mask)
        got, clean = c.rows("out", nh)
        assert clean and (got[c.used:] == 77.0).all()
        check_rows(c, got, *step_ref.tree_exact(c, mask))
        if lens != "before_the_first" and kind == "tree":
            for window in (1, 100):
                _attend_tree(c, kv, mask, pos, window=window)
                check_rows(c, c.rows("out", nh)[0], *step_ref.tree_exact(c, mask, pos, window=window), name=str(window))


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("hd", [48, 64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_bad_values_in_tall_tiles(dtype, cache, hd, bad):
    """Infinities and NaN in V of what is held, which all rows attend, and of new rows that some masks name; pages that are
    none; then in K of a new row that no other attends."""
    c = _tall(Case([(40, 700), (33, 33), (5, 100)], 16, 1, hd, 16, dtype, cache, seed=hd))
    mask, _ = _masks(c, np.random.default_rng(6), "tree", 1)
    for s, p, dim in ((0, 300, 3), (0, 680, hd - 1), (1, 9, 5), (2, 96, 8)):
        c.v_pool[0, int(c.pages[s, p // 16]), :, p % 16, dim] = bad
    c.pages[0, 4], c.pages[0, 30] = -1, c.n_pages
    mask[40 + 32, 0] |= np.uint64(1 << 32)
    for i in range(40, 40 + 32):
        mask[i, 0] &= ~np.uint64(1 << 32)      # (row 32 of the second sequence is attended by itself alone)
    c.up()
    with c.handle() as kv:
        _attend_tree(c, kv, mask)
        got = c.rows("out", 16)[0]
        check_rows(c, got, *step_ref.tree_exact(c, mask))
        page = int(c.pages[1, 2])
        c.k_pool[0, page, :, 0, 3] = bad       # position 32
        c.d["k_pool"].copy_(c.k_pool)
        _attend_tree(c, kv, mask)
    other = c.rows("out", 16)[0]
    keep = np.arange(c.n_tok) != 72
    assert _bits(got[keep], other[keep])


@pytest.mark.parametrize("dtype,cache", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("pad,off", [(0, 0), (8, 8), (3, 1)])
def test_tree_strides_and_places(dtype, cache, pad, off):
    c = Case([(12, 80), (3, 40)], 5, 1, 72, 32, dtype, cache, seed=2, row_pad=pad, row_off=off).up()
    mask, _ = _masks(c, np.random.default_rng(1), "tree", 1)
    with c.handle() as kv:
        ws = torch.empty(kv.workspace_bytes(), dtype=torch.uint8, device="cuda")
        _attend_tree(c, kv, mask, workspace=ws.data_ptr(), stream=torch.cuda.Stream().cuda_stream, scale=0.2)
    got, clean = c.rows("out", 5)
    assert clean
    check_rows(c, got, *step_ref.tree_exact(c, mask, scale=float(np.float32(0.2))))


@pytest.mark.parametrize("starts,max_q", [([0, 9, 4, 12], 1), ([5, 2, 20, 3], 64), ([-3, 40, 2, 9], 0)])
def test_tree_of_a_q_start_that_is_not_ascending(starts, max_q):
    """Nothing outside the buffers is touched."""
    c = Case([(4, 40), (4, 90), (4, 17)], 4, 2, 64, 16, "f32", "f16", seed=2, row_pad=4, row_off=4).up()
    mask = np.full((c.n_tok, 1), 2 ** 64 - 1, np.uint64)
    c.d["starts"].copy_(torch.tensor(starts, dtype=torch.int32))
    with c.handle() as kv:
        _attend_tree(c, kv, mask, np.zeros(c.n_tok, np.int32), window=20, max_q=max_q)
    assert c.rows("out", 4)[1]


# ---- what is kept -----------------------------------------------------------------------

class Kept:
    """A step over a pool of pages, of which some rows are kept."""

    def __init__(self, lens, n_keep, nkv, hd, ps, cache, n_layer=1, rows="path", seed=0, extra=3, free=True, alias=False, n_free=None):
        rng = np.random.default_rng(seed)
        self.lens, self.n_keep, self.ps = lens, list(n_keep), ps
        held = [-(-kv // ps) for _, kv in lens]
        self.n_pages = sum(held) + extra
        self.stride = max(held + [1]) + 1
        order = rng.permutation(self.n_pages)
        self.pages = np.full((len(lens), self.stride), -1, np.int32)
        at = 0
        for s, h in enumerate(held):
            self.pages[s, :h] = order[at:at + h]
            at += h
        self.free = np.full(self.n_pages, -9, np.int32)
        self.free[:extra] = order[at:]
        self.n_free = extra if n_free is None else n_free
        self.starts = np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32)
        self.kv_len = [kv for _, kv in lens]
        self.rows = None
        if rows == "path":
            self.rows = np.full(int(self.starts[-1]) + 2, -1, np.int32)
            for s, (n, _) in enumerate(lens):
                k = min(max(self.n_keep[s], 0), n)
                self.rows[self.starts[s]:self.starts[s] + k] = np.sort(rng.choice(n, k, replace=False)) if k else []
        gen = torch.Generator().manual_seed(seed)
        self.pools = [torch.randn(n_layer, self.n_pages, nkv, ps, hd, generator=gen).to(DTYPE[cache]) for _ in range(2)]
        self.use_free, self.alias = free, alias
        self.geo = (n_layer, self.n_pages, ps, 2 * nkv, nkv, hd, cache)

    def run(self):
        from kore_amd import paged
        d = [p.cuda() for p in self.pools]
        n_tok = int(self.starts[-1]) + 2
        guard = lambda x: torch.cat([torch.full((4,), 77, dtype=torch.int32), torch.as_tensor(np.asarray(x, np.int32)).reshape(-1),  # noqa: E731
                                     torch.full((4,), 77, dtype=torch.int32)]).cuda()
        t = {n: guard(v) for n, v in (("starts", self.starts), ("n_keep", self.n_keep), ("kv_len", self.kv_len), ("pages", self.pages),
                                      ("free", self.free), ("n_free", [self.n_free]), ("kv_out", [55] * len(self.lens)), ("n_out", [55]))}
        rows = None if self.rows is None else _dev(self.rows)
        if self.alias:
            t["kv_out"], t["n_out"] = t["kv_len"], t["n_free"]
        torch.cuda.synchronize()
        p = {n: x.data_ptr() + 16 for n, x in t.items()}
        with paged.PagedKV(*self.geo, k_pool=d[0].data_ptr(), v_pool=d[1].data_ptr()) as kv:
            free = dict(free_pages=p["free"], n_free=p["n_free"], n_free_out=p["n_out"]) if self.use_free else {}
            kv.keep_dev(paged.Keep(len(self.lens), n_tok, p["starts"], p["n_keep"], p["kv_len"], p["kv_out"], p["pages"], self.stride,
                                   rows=None if rows is None else rows.data_ptr(), **free))
            kv.sync()
        free, pools = self.free.copy(), [x.clone() for x in self.pools]
        if not self.use_free:
            free = np.zeros(self.n_pages, np.int32)
        ends, n_free = step_ref.keep(pools, self.starts.tolist(), self.n_keep, None if self.rows is None else self.rows.tolist(), self.kv_len,
                                     self.pages.tolist(), free, self.n_free, self.ps)
        got = {n: x.cpu().numpy() for n, x in t.items()}
        for n, x in got.items():
            assert (x[:4] == 77).all() and (x[-4:] == 77).all(), n
        inner = {n: x[4:-4] for n, x in got.items()}
        assert np.array_equal(inner["kv_out"], ends)
        assert np.array_equal(inner["pages"], self.pages.reshape(-1))
        if self.use_free:
            assert inner["n_out"][0] == n_free and np.array_equal(inner["free"], free)
        else:
            assert np.array_equal(inner["free"], self.free)
        for a, b in zip(d, pools):
            assert _bits(a.cpu(), b)


@pytest.mark.parametrize("cache", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nkv,hd,ps,n_layer", [(2, 64, 16, 3), (4, 128, 64, 2), (3, 96, 32, 1), (1, 8, 16, 5), (5, 40, 256, 2), (1, 256, 128, 1)])
@pytest.mark.parametrize("rows", ["path", None])
@pytest.mark.parametrize("free", [True, False])
def test_keep(cache, nkv, hd, ps, n_layer, rows, free):
    lens = [(9, 40), (0, 33), (1, 1), (40, 200), (64, 64), (5, ps + 2), (30, 3 * ps), (2, 77), (20, 20)]
    n_keep = [3, 0, 1, 7, 64, 2, -1, 90, 0]
    Kept(lens, n_keep, nkv, hd, ps, cache, n_layer, rows, seed=hd, free=free, alias=ps > 32).run()


def test_keep_of_many_rows_and_sequences():
    Kept([(700, 1000), (300, 300)], [650, 257], 1, 64, 32, "f16", seed=1).run()
    rng = np.random.default_rng(2)
    for n_seq in (16, 17, 64, 65, 300, 1030, 3000):
        lens = [(int(n), int(n + h)) for n, h in zip(rng.integers(0, 20, n_seq), rng.integers(0, 200, n_seq))]
        Kept(lens, [int(x) for x in rng.integers(-1, 9, n_seq)], 1, 8, 16, "f32", seed=n_seq).run()
    Kept([(3, 20000), (1, 9000), (0, 5)], [-1, -1, -1], 1, 8, 16, "f16", seed=4).run()
    Kept([], [], 1, 8, 16, "f16").run()


def test_keep_of_what_is_not_there():
    """Entries of `rows` and pages that are none, a sequence of fewer positions than rows, more free pages than there are."""
    k = Kept([(9, 40), (6, 60), (4, 2)], [5, 4, 3], 2, 64, 16, "f16", n_layer=2, seed=3)
    k.rows[:5] = [0, 2, 9, 100, 8]
    k.rows[9:13] = [-1, -2 ** 31, 2 ** 31 - 1, 5]
    k.pages[0, 1], k.pages[1, 2] = -1, k.n_pages
    k.run()
    k = Kept([(9, 40), (6, 60)], [-1, -1], 2, 64, 16, "f16", seed=3)
    k.pages[0, 1], k.pages[1, 2] = -1, k.n_pages + 7
    k.run()
    Kept([(9, 40), (6, 60)], [-1, -1], 2, 64, 16, "f16", seed=3, n_free=8).run()


# ---- places and streams ---------------------------------------------------------------------

def test_store_into_pools_at_16_bytes():
    """Pools, rows and weights that start at 16 bytes, at an element, or at any: the same bits."""
    from kore_amd import paged, rope
    w = [np.linspace(0.5, 2, 128, dtype=np.float32), np.linspace(2, 0.5, 128, dtype=np.float32)]
    for dtype, cache in (("f32", "f32"), ("bf16", "bf16"), ("f32", "f16")):
        got = []
        for off, row_off in ((0, 0), (16, 0), (16, 4), (0, 1)):
            c = Case([(3, 9), (1, 17), (40, 40)], 6, 2, 128, 16, dtype, cache, seed=3, row_off=row_off, row_pad=8 - row_off).up()
            n = c.d["k_pool"].numel() * c.d["k_pool"].element_size()
            raw = [torch.zeros(n + 64, dtype=torch.uint8, device="cuda") for _ in range(2)]
            torch.cuda.synchronize()
            with paged.PagedKV(1, c.n_pages, 16, 6, 2, 128, cache, rope.Config(128), *[r.data_ptr() + off for r in raw]) as kv:
                _store(c, kv, *_slots(c), w)
            got.append([r[off:off + n].cpu() for r in raw] + [c.rows("out", 6)[0]])
        for other in got[1:]:
            for a, b in zip(got[0], other):
                assert _bits(a, b)


def test_steps_past_32_bits():
    """Slots whose offset in the pool passes 2^32 bytes and 2^31 elements: rows stored there, a tree attended, a path kept."""
    from kore_amd import paged
    nkv, hd, ps = 8, 128, 256
    n_pages = (2 ** 31 + 2 ** 28) // (nkv * hd * ps)
    c = Case([(9, 300), (40, 280)], 16, nkv, hd, ps, "f16", "f16", seed=4)
    mask, _ = _masks(c, np.random.default_rng(4), "tree", 1)
    far = {int(p): n_pages - 1 - i for i, p in enumerate(sorted(set(c.pages[c.pages >= 0].tolist())))}
    table = np.vectorize(lambda x: far.get(int(x), -1))(c.pages).astype(np.int32)
    with paged.PagedKV(1, n_pages, ps, 16, nkv, hd, "f16") as kv:
        assert kv.info().pool_bytes > 2 ** 32
        # the whole of either sequence through the store, which keeps rows as they are
        w = Case([(k, k) for _, k in c.lens], 16, nkv, hd, ps, "f16", "f16", seed=5)
        slot = []
        for s, (n, _) in enumerate(w.lens):
            p, at = np.arange(n), int(w.starts[s])
            w.k[at:at + n] = c.k_pool[0, c.pages[s, p // ps], :, p % ps]
            w.v[at:at + n] = c.v_pool[0, c.pages[s, p // ps], :, p % ps]
            slot += (table[s, p // ps].astype(np.int64) * ps + p % ps).tolist()
        assert max(slot) * nkv * hd > 2 ** 31
        c.up()
        w.up()
        _store(w, kv, np.zeros(w.n_tok, np.int32), np.asarray(slot))
        t = _dev(table)
        m = _dev(mask.view(np.int64), torch.int64)
        torch.cuda.synchronize()
        b = paged.Batch(2, c.n_tok, c.d["starts"].data_ptr(), c.d["kv_len"].data_ptr(), t.data_ptr(), c.stride, 40)
        kv.attend_tree_dev(0, b, paged.Tree(m.data_ptr()), "f16", c.ptr("q"), c.ptr("out"))
        kv.sync()
        check_rows(c, c.rows("out", 16)[0], *step_ref.tree_exact(c, mask))
        # the second sequence keeps rows 3, 20 and 39 of its 40
        keep, rows, ends = _dev([0, 3]), _dev([0] * 9 + [3, 20, 39] + [0] * 37), torch.zeros(2, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        kv.keep_dev(paged.Keep(2, c.n_tok, c.d["starts"].data_ptr(), keep.data_ptr(), c.d["kv_len"].data_ptr(), ends.data_ptr(), t.data_ptr(),
                               c.stride, rows=rows.data_ptr()))
        kv.sync()
        assert ends.tolist() == [291, 243]
        # what lies there now, by a token that attends one position at a time
        one = Case([(1, 1)], 16, nkv, hd, ps, "f16", "f16", seed=6).up()
        for i, row in enumerate((3, 20, 39)):
            n = torch.tensor([241 + i], dtype=torch.int32, device="cuda")
            t2 = t[1:].contiguous()
            torch.cuda.synchronize()
            kv.attend_dev(0, paged.Batch(1, 1, one.d["starts"].data_ptr(), n.data_ptr(), t2.data_ptr(), c.stride, 1), "f16", one.ptr("q"),
                          one.ptr("out"), window=1)
            kv.sync()
            p = 240 + row
            want = c.v_pool[0, c.pages[1, p // ps], :, p % ps]
            got = one.rows("out", 16)[0][0].view(nkv, 2, hd)
            assert torch.equal(got[:, 0], want) and torch.equal(got[:, 1], want)


def test_two_streams_at_once():
    """Trees of two caches, each call with a workspace of its own, on two streams at once: the bits of one after the other."""
    cs = [Case([(20, 3000), (5, 700)], 16, 2, 128, 64, "f32", "f16", seed=i).up() for i in range(2)]
    masks = [_masks(c, np.random.default_rng(i), "tree", 1)[0] for i, c in enumerate(cs)]
    from kore_amd import paged
    with cs[0].handle() as kv:
        dev = [(_dev(m.view(np.int64), torch.int64), torch.empty(kv.workspace_bytes(), dtype=torch.uint8, device="cuda"), torch.cuda.Stream())
               for m in masks]

        def attend(c, m, ws, st, handle):
            handle.attend_tree_dev(0, c.batch(), paged.Tree(m.data_ptr()), "f32", c.ptr("q"), c.ptr("out"), workspace=ws.data_ptr(),
                                   stream=st.cuda_stream)

        with cs[1].handle() as kv2:
            want = []
            for c, (m, ws, st), h in zip(cs, dev, (kv, kv2)):
                torch.cuda.synchronize()
                attend(c, m, ws, st, h)
                torch.cuda.synchronize()
                want.append(c.d["out"].clone())
            for _ in range(10):
                for c in cs:
                    c.d["out"].fill_(77.0)
                torch.cuda.synchronize()
                for c, (m, ws, st), h in zip(cs, dev, (kv, kv2)):
                    attend(c, m, ws, st, h)
                torch.cuda.synchronize()
                for c, w in zip(cs, want):
                    assert _bits(c.d["out"], w)


# ---- refusals ----------------------------------------------------------------------------

def test_steps_refuse():
    """Each refusal says what it is and leaves everything as it was."""
    from kore_amd import paged
    c = Case([(2, 20), (1, 5)], 4, 2, 64, 16, "f32", "f16", seed=1).up()
    z = torch.full((64,), 5, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    Z = z.data_ptr()
    before = {n: t.clone() for n, t in c.d.items()}

    def plan(**kw):
        base = dict(n_seq=1, n_tok=4, n_new=Z, kv_held=Z, kv_len=Z, pages=Z, pages_stride=2, free_pages=Z, n_free=Z, n_free_out=Z, q_start=Z,
                    pos=Z, slot=Z, status=Z)
        return paged.Plan(**{**base, **kw})

    def rows(**kw):
        return paged.Rows(**{**dict(n_tok=3, pos=Z, slot=Z), **kw})

    def keep(**kw):
        return paged.Keep(**{**dict(n_seq=1, n_tok=4, q_start=Z, n_keep=Z, kv_len=Z, kv_out=Z, pages=Z, pages_stride=2), **kw})

    with c.handle() as kv:
        def store(r, k=c.ptr("k"), v=c.ptr("v"), layer=0, dtype="f32", **kw):
            kv.append_rows_dev(layer, r, dtype, k, v, **kw)

        def tree(t, layer=0, dtype="f32", q=c.ptr("q"), batch=None, **kw):
            kv.attend_tree_dev(layer, batch or c.batch(), t, dtype, q, c.ptr("out"), **kw)

        T = paged.Tree
        for call, code, text in [
                *[(lambda kw=kw: kv.plan_dev(plan(**kw)), code, text) for kw, code, text in [
                    (dict(n_seq=-1), -1, "n_seq"), (dict(n_tok=-1), -1, "n_tok"), (dict(pages_stride=0), -1, "pages_stride"),
                    (dict(pages_stride=2 ** 27), -1, "pages_stride"), (dict(n_seq=2 ** 16 + 1), -3, "n_seq"), (dict(n_tok=2 ** 23 + 1), -3, "n_tok"),
                    *[({n: None}, -1, "null " + n) for n in ("n_new", "kv_held", "kv_len", "pages", "free_pages", "n_free", "n_free_out", "q_start",
                                                             "pos", "slot", "status")],
                    *[({n: Z + 2}, -1, n + " is not aligned") for n in ("n_new", "kv_held", "kv_len", "pages", "n_free", "q_start", "pos", "status")],
                    (dict(slot=Z + 4), -1, "slot is not aligned"), (dict(parent=Z), -1, "mask_words"), (dict(parent=Z, mask=Z, mask_words=17), -1, "mask_words"),
                    (dict(parent=Z, mask_words=1), -1, "null mask"), (dict(mask=Z, mask_words=1), -1, "null parent"),
                    (dict(mask_words=1), -1, "mask_words"), (dict(parent=Z, mask=Z + 4, mask_words=1), -1, "mask is not aligned")]],
                *[(lambda kw=kw: store(rows(**kw)), code, text) for kw, code, text in [
                    (dict(n_tok=-1), -1, "n_tok"), (dict(n_tok=2 ** 23 + 1), -3, "n_tok"), (dict(pos=None), -1, "pos"), (dict(slot=None), -1, "slot"),
                    (dict(slot=Z + 4), -1, "slot"), (dict(q_norm=Z, norm_eps=0.0), -1, "norm_eps"), (dict(k_norm=Z, norm_eps=math.nan), -1, "norm_eps"),
                    (dict(q_norm=Z + 2), -1, "q_norm"), (dict(k_norm=Z + 1), -1, "k_norm")]],
                (lambda: store(rows(), layer=1), -1, "layer"), (lambda: store(rows(), dtype="bf16"), -1, "type"),
                (lambda: store(rows(), k=None), -1, "null"), (lambda: store(rows(), v=None), -1, "null"),
                (lambda: store(rows(), q=c.ptr("q")), -1, "q without"), (lambda: store(rows(), k_stride=127), -1, "k stride"),
                (lambda: store(rows(), q=c.ptr("q"), q_out=c.ptr("k")), -1, "rows overlap"),
                (lambda: tree(T(None)), -1, "mask"), (lambda: tree(T(Z + 4)), -1, "mask"), (lambda: tree(T(Z, 0)), -1, "mask_words"),
                (lambda: tree(T(Z, 17)), -1, "mask_words"), (lambda: tree(T(Z), window=5), -1, "pos"), (lambda: tree(T(Z, 1, Z + 2)), -1, "pos"),
                (lambda: tree(T(Z), window=-1), -1, "window"), (lambda: tree(T(Z), layer=2), -1, "layer"), (lambda: tree(T(Z), q=None), -1, "null"),
                (lambda: tree(T(Z), scale=-1.0), -1, "scale"), (lambda: tree(T(Z), workspace=8), -1, "workspace"),
                *[(lambda kw=kw: kv.keep_dev(keep(**kw)), code, text) for kw, code, text in [
                    (dict(n_seq=-1), -1, "n_seq"), (dict(n_tok=-1), -1, "n_tok"), (dict(pages_stride=0), -1, "pages_stride"),
                    (dict(n_seq=2 ** 16 + 1), -3, "n_seq"), *[({n: None}, -1, "null " + n) for n in ("q_start", "n_keep", "kv_len", "kv_out", "pages")],
                    (dict(rows=Z + 2), -1, "rows"), (dict(free_pages=Z), -1, "n_free"), (dict(n_free=Z, n_free_out=Z), -1, "free_pages"),
                    (dict(free_pages=Z, n_free=Z), -1, "n_free_out")]]]:
            with pytest.raises(paged.PagedError, match=text) as e:
                call()
            assert e.value.code == code, text
        L, h = paged.lib(), kv.handle
        assert L.kore_paged_plan_dev(h, None, None) == -1 and L.kore_paged_keep_dev(h, None, None) == -1
        assert L.kore_paged_append_rows_dev(h, 0, None, 0, None, 0, None, 0, None, 0, None, 0, None) == -1
        assert L.kore_paged_attend_tree_dev(h, 0, C.byref(c.batch().struct), None, 0, None, 256, None, 256, 0.0, 0, None, None) == -1
        store(rows(n_tok=0, pos=None, slot=None), k=None, v=None)
        kv.sync()
    assert (z == 5).all()
    for n, t in before.items():
        assert _bits(t, c.d[n]), n


def test_an_error_of_another_call_is_not_theirs():
    """An error that another HIP call of the thread has left is neither reported by a call of these nor taken away."""
    from kore_amd import hip, paged, rope
    t = Tables([4, 9], [20, 0], 16, seed=1).up()
    c = Case([(2, 40), (20, 90)], 4, 2, 64, 16, "f32", "f16", seed=1).up()
    L = hip.lib()
    L.hipPeekAtLastError.restype = L.hipGetLastError.restype = C.c_int
    pos, slot = (_dev(x, d) for x, d in zip(_slots(c), (torch.int32, torch.int64)))
    mask = torch.full((22, 1), -1, dtype=torch.int64, device="cuda")
    keep = torch.ones(2, dtype=torch.int32, device="cuda")
    with t.handle() as plans, c.handle(rope.Config(64)) as kv, rope.Rope(rope.Config(64)) as r:
        torch.cuda.synchronize()
        for call in [lambda: plans.plan_dev(t.plan()),
                     lambda: kv.append_rows_dev(0, paged.Rows(22, pos.data_ptr(), slot.data_ptr()), "f32", c.ptr("k"), c.ptr("v")),
                     lambda: kv.attend_tree_dev(0, c.batch(), paged.Tree(mask.data_ptr()), "f32", c.ptr("q"), c.ptr("out")),
                     lambda: kv.keep_dev(paged.Keep(2, 22, *[c.d[n].data_ptr() if n else keep.data_ptr() for n in ("starts", "", "kv_len", "kv_len", "pages")], c.stride)),
                     lambda: r.norm_dev("f32", 22, 64, [rope.Heads(c.ptr("q"), c.ptr("out"), 4, 64)], pos.data_ptr())]:
            assert L.hipSetDevice(1 << 20) != 0      # no such device
            left = L.hipPeekAtLastError()
            try:
                call()
                assert L.hipPeekAtLastError() == left
            finally:
                L.hipGetLastError()
        for h in (plans, kv, r):
            h.sync()
