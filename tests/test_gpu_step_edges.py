"""Steps of drafted tokens where they could go wrong and tests/test_gpu_step.py does not look: windows that a path is as deep as,
heads next to the largest float, masks of many words in tiles of 128 rows, many sequences."""
import numpy as np
import pytest
import torch

from tests import step_ref
from tests.paged_ref import PAIRS, Case, check_rows, to64
from tests.test_gpu_step import Tables, _attend_tree, _bits, _masks, _norm, _tall

pytestmark = pytest.mark.gpu


# ---- windows of masks ------------------------------------------------------------------

def _windowed(parents, window, words):
    """Masks of trees, [sum of rows][words]: each row and those above it in its tree that are fewer than `window` rows up."""
    mask = []
    for parent in parents:
        for i in range(len(parent)):
            bits, at, up = 0, i, 0
            while at >= 0 and up < (window or 1 << 30):
                bits |= 1 << at
                at, up = parent[at], up + 1
            mask.append([bits >> (64 * w) & (1 << 64) - 1 for w in range(words)])
    return np.asarray(mask, np.uint64).reshape(-1, words)


class Windowed(Tables):
    """Tables of a plan with a window, which its masks alone are to show."""

    def __init__(self, n_new, held, ps, parents, words, window, **kw):
        super().__init__(n_new, held, ps, words=words, parent=[q for p in parents for q in p], **kw)
        self.parents, self.window = parents, window

    def plan(self):
        p = super().plan()
        p.struct.window = self.window
        return p

    def get(self, name):
        got = super().get(name)
        if name != "mask":
            return got
        n = sum(self.n_new)
        mask = got.view(np.uint64).reshape(self.n_tok, self.words)
        assert np.array_equal(mask[:n], _windowed(self.parents, self.window, self.words))
        return np.concatenate([_windowed(self.parents, 0, self.words), mask[n:]]).view(np.int64)


@pytest.mark.parametrize("window", [1, 2, 7, 63, 64, 65, 130, 2 ** 31 - 1])
@pytest.mark.parametrize("words,n_seq,alias", [(1, 9, False), (2, 9, False), (5, 9, False), (16, 9, False), (1, 9, True), (16, 9, True),
                                               (1, 1100, False), (2, 1100, True)])
def test_masks_in_a_window(words, window, n_seq, alias):
    """A mask is the window's last of a row's path, positions and slots are as without one: in one launch and in two."""
    rng = np.random.default_rng(words * 1000 + window % 1000)
    n_new = [int(x) for x in rng.integers(0, 64 * words + 1 if n_seq < 10 else 20, n_seq)]
    n_new[0] = 64 * words
    parents = [list(range(-1, n - 1)) if i % 3 == 0 else step_ref.tree(rng, n, 1 + i % 3) for i, n in enumerate(n_new)]
    assert Windowed(n_new, [int(x) for x in rng.integers(0, 90, n_seq)], 16, parents, words, window, alias=alias).run() == 0


def _plan_masks(c, parents, words, window):
    """(masks, positions) that a plan makes of a Case's new rows."""
    held = [int(kv) - n for n, kv in c.lens]
    t = Windowed([n for n, _ in c.lens], held, c.ps, parents, words, window, n_tok=c.n_tok)
    assert t.run() == 0
    mask = Tables.get(t, "mask").view(np.uint64).reshape(c.n_tok, words)
    return mask, t.get("pos").astype(np.int32)


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("window", [1, 5, 12, 64, 100])
@pytest.mark.parametrize("max_q", [1, None])
def test_a_planned_chain_in_a_window_is_causal(dtype, cache, window, max_q):
    """Plan and attention with the window of a model: kore_paged_attend_dev's rows, paths deeper than the window among them."""
    c = Case([(12, 300), (5, 5), (1, 77), (90, 100), (64, 64)], 12, 2, 96, 16, dtype, cache, seed=window).up()
    mask, pos = _plan_masks(c, [list(range(-1, n - 1)) for n, _ in c.lens], 2, window)
    with c.handle() as kv:
        _attend_tree(c, kv, mask, pos, window=window, max_q=max_q)
    check_rows(c, c.rows("out", 12)[0], *c.exact(window=window))


@pytest.mark.parametrize("window", [2, 4])
def test_a_planned_tree_in_a_window_is_its_paths(window):
    """Each row of a tree is the last of its path, decoded as a chain of its own in the same window."""
    rng = np.random.default_rng(window)
    n, held = 24, 30
    parent = step_ref.tree(rng, n, 1)
    c = Case([(n, held + n)], 4, 2, 64, 16, "f32", "f32", seed=window).up()
    mask, pos = _plan_masks(c, [parent], 1, window)
    with c.handle() as kv:
        _attend_tree(c, kv, mask, pos, window=window)
    got = c.rows("out", 4)[0].double().numpy()
    deepest = 0
    for i in range(n):
        path = [i]
        while parent[path[0]] >= 0:
            path.insert(0, parent[path[0]])
        deepest = max(deepest, len(path))
        one = Case([(len(path), held + len(path))], 4, 2, 64, 16, "f32", "f32")
        at = lambda p: (c.pages[0, p // 16], slice(None), p % 16)  # noqa: E731
        for p, src in enumerate(list(range(held)) + [held + r for r in path]):
            for a, b in ((one.k_pool, c.k_pool), (one.v_pool, c.v_pool)):
                a[0, one.pages[0, p // 16], :, p % 16] = b[0][at(src)]
        one.q[:] = c.q[path]
        want, bound = one.exact(window=window)
        assert (np.abs(got[i] - want[-1]) <= bound[-1]).all(), i
    assert deepest > window


def test_a_window_below_zero_is_refused():
    from kore_amd import paged
    t = Tables([2], [3], 16, words=1, parent=[-1, 0]).up()
    p = t.ptr
    with t.handle() as kv:
        with pytest.raises(paged.PagedError, match="window") as e:
            kv.plan_dev(paged.Plan(1, t.n_tok, p("n_new"), p("held"), p("kv_len"), p("pages"), t.stride, p("free"), p("n_free"),
                                   p("n_free_out"), p("q_start"), p("pos"), p("slot"), p("status"), p("parent"), p("mask"), 1, window=-1))
        assert e.value.code == -1
        kv.sync()
    assert (t.get("status") == 99).all() and (t.get("pos") == 99).all() and (t.get("mask") == 99).all()


# ---- heads next to the largest float --------------------------------------------------------

@pytest.mark.parametrize("hd", [2, 64, 66, 128, 640, 1022])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_next_to_the_largest_float(hd, dtype):
    """Heads whose root mean square passes 2^126, beside ordinary ones and one without weights.  Position 0 turns by 1 and 0,
    exactly, so that 1 / root, its product and the weights' (powers of two, exact) leave two half steps of fp32 and the rounding
    to the type."""
    from kore_amd import rope
    rng = np.random.default_rng(hd)
    x = np.sign(rng.standard_normal((12, 5, hd))) * (0.5 + 0.5 * rng.random((12, 5, hd)))
    x[:, :3] *= np.float64(2.0) ** rng.uniform(126.5, 127.9, (12, 3, 1))
    x[:, 3] *= 1e-3
    x[3, 1, 1:] *= 2.0 ** -200
    x = torch.from_numpy(x).to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    assert torch.isfinite(x).all()
    w = 2.0 ** rng.integers(-2, 3, hd)
    cfg = rope.Config(min(hd, 512))
    got, bare = _norm(dtype, [x, x], np.zeros(12, int), [w, None], cfg)
    v = to64(x)
    want = v / np.sqrt(np.mean(v * v, -1, keepdims=True) + float(np.float32(1e-6))) * w
    bound = 2 * 2.0 ** -24 * (1 + 2.0 ** -20) * np.abs(want) + 2.0 ** -149
    if dtype == "bf16":
        bound += 2.0 ** -8 * (np.abs(want) + bound)
    assert (np.abs(to64(got) - want) <= bound).all()
    assert _bits(bare, x)


# ---- trees of many rows, and of many sequences -------------------------------------------------
#
# A table of many keys lets a step take tiles of 128 rows (_tall); in a window it is the hint of the most rows, which may be any.
TALL_Q = 1 << 17


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("hd,ps,words", [(64, 16, 2), (128, 64, 5), (128, 16, 16), (48, 32, 3), (256, 128, 2)])
def test_wide_trees_in_tall_tiles(dtype, cache, hd, ps, words):
    """Masks of several words in tiles of 128 rows: fewer bits than rows and more, what is held no multiple of a word, windows."""
    c = _tall(Case([(150, 150 + 61), (65, 65), (333, 333 + 100), (1, 40), (129, 129 + 7)], 8, 1, hd, ps, dtype, cache, seed=hd + words,
                   extra_rows=2)).up()
    with c.handle() as kv:
        for kind, window in (("tree", 0), ("tree", 70), ("any", 0)):
            mask, pos = _masks(c, np.random.default_rng(words), kind, words)
            c.d["out"].fill_(55.0)
            _attend_tree(c, kv, mask, pos, window=window, max_q=TALL_Q)
            got, clean = c.rows("out", 8)
            assert clean and (got[c.used:] == 55.0).all()
            check_rows(c, got, *step_ref.tree_exact(c, mask, pos, window=window), name="%s, window %d" % (kind, window))


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("hd", [64, 128])
def test_planned_chains_in_tall_tiles_are_causal(dtype, cache, hd):
    """Chains of up to some hundred rows in tiles of 128 rows, with a window and without: kore_paged_attend_dev's rows."""
    c = _tall(Case([(12, 300), (5, 5), (1, 77), (200, 230), (128, 128), (64, 131)], 8, 1, hd, 16, dtype, cache, seed=hd)).up()
    with c.handle() as kv:
        for window in (0, 5, 64, 100):
            mask, pos = _plan_masks(c, [list(range(-1, n - 1)) for n, _ in c.lens], 4, window)
            _attend_tree(c, kv, mask, pos, window=window, max_q=TALL_Q)
            check_rows(c, c.rows("out", 8)[0], *c.exact(window=window), name=str(window))


@pytest.mark.parametrize("dtype,cache", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("n_seq", [64, 65, 130])
@pytest.mark.parametrize("tall", [False, True])
def test_trees_of_many_sequences(dtype, cache, n_seq, tall):
    """As many sequences as a wave has lanes, and more: some without rows, a few long enough to be split, with a window and without."""
    rng = np.random.default_rng(n_seq)
    lens = [(int(n), int(n + h)) for n, h in zip(rng.integers(0, 40 if tall else 9, n_seq), rng.integers(0, 120, n_seq))]
    for s in (0, 40, 63, n_seq - 1):
        lens[s] = (int(rng.integers(2, 20)), int(rng.integers(2500, 4000)))
    c = Case(lens, 8, 1, 64, 64, dtype, cache, seed=n_seq, extra_rows=1)
    c = (_tall(c) if tall else c).up()
    mask, pos = _masks(c, np.random.default_rng(1), "tree", 1)
    with c.handle() as kv:
        for window in (0, 700):
            _attend_tree(c, kv, mask, pos, window=window, max_q=TALL_Q if tall else 1)
            check_rows(c, c.rows("out", 8)[0], *step_ref.tree_exact(c, mask, pos, window=window), name=str(window))


@pytest.mark.parametrize("dtype,cache", [("f32", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("n,max_q", [(30, 1), (100, TALL_Q)])
def test_more_tiles_than_the_card_holds_at_once(dtype, cache, n, max_q):
    """Forty trees whose tiles are over twice the CUs (16 rows) or over them (128 rows), beside a long sequence that is split."""
    rng = np.random.default_rng(n)
    lens = [(n, n + int(h)) for h in rng.integers(0, 60, 40)]
    lens[7] = (n, 3000)
    c = Case(lens, 8, 1, 64, 16, dtype, cache, seed=n)
    c = (c if max_q == 1 else _tall(c)).up()
    mask, pos = _masks(c, np.random.default_rng(1), "tree", 2)
    with c.handle() as kv:
        for window in (0, 1500):
            _attend_tree(c, kv, mask, pos, window=window, max_q=max_q)
            check_rows(c, c.rows("out", 8)[0], *step_ref.tree_exact(c, mask, pos, window=window), name=str(window))


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("lens,tall", [([(8, 60), (3, 40), (1, 1)], False), ([(20, 3000), (5, 700)], False), ([(64, 3000), (40, 90)], True)])
def test_trees_in_place(dtype, cache, lens, tall):
    """The result in q's own rows, in one launch and with splits joined: the bits of rows of its own."""
    from kore_amd import paged
    c = Case(lens, 8, 2, 64, 64, dtype, cache, seed=3, extra_rows=2)
    c = (_tall(c) if tall else c).up()
    mask, _ = _masks(c, np.random.default_rng(3), "tree", 1)
    m = torch.from_numpy(mask.view(np.int64)).cuda()
    with c.handle() as kv:
        _attend_tree(c, kv, mask)
        want, behind = c.d["out"][:c.used].clone(), c.d["q"][c.used:].clone()
        kv.attend_tree_dev(0, c.batch(), paged.Tree(m.data_ptr()), dtype, c.ptr("q"), c.ptr("q"), q_stride=c.step("q"), out_stride=c.step("q"))
        kv.sync()
    assert _bits(c.d["q"][:c.used], want) and _bits(c.d["q"][c.used:], behind)
