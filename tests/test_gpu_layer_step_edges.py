"""A layer's step of drafted tokens at its edges: batches that its attention would refuse, windows."""
import numpy as np
import pytest
import torch

from tests.test_gpu_layer_paged import E, _weights
from tests.test_gpu_layer_step import N_TOK, PS, STRIDE, Server

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("with_tree", [False, True])
def test_a_refused_batch_stores_nothing(with_tree):
    """A batch that the attention refuses is refused before the rows' K and V are stored: x and the pools keep their bits."""
    from kore_amd import paged
    from kore_amd.layer import LayerError
    ws = _weights(1)
    s = Server()
    try:
        p = s.p
        for n in ("x", "k_pool", "v_pool"):
            s.t[n].fill_(1.0)
        s.t["slot"].copy_(torch.arange(N_TOK, dtype=torch.int64))
        torch.cuda.synchronize()
        good = dict(n_seq=3, n_tok=N_TOK, pages_stride=STRIDE, max_q=16)
        for bad in (dict(max_q=-1), dict(max_q=-2 ** 31), dict(pages_stride=0), dict(pages_stride=-STRIDE), dict(pages_stride=2 ** 30 // 16 + 1),
                    dict(pages_stride=2 ** 31 - 1), dict(n_seq=2 ** 16 + 1), dict(n_seq=2 ** 31 - 1)):
            kw = {**good, **bad}
            batch = paged.Batch(kw["n_seq"], kw["n_tok"], p["q_start"], p["kv_len"], p["pages"], kw["pages_stride"], kw["max_q"])
            with pytest.raises(LayerError, match="max_q|pages_stride|n_seq"):
                s.L.paged_ex_dev(ws[0], s.kv, 0, batch, p["x"], p["pos"], p["slot"], p["q_norm"], p["k_norm"], s.tree if with_tree else None)
            s.L.sync()
            for n in ("x", "k_pool", "v_pool"):
                assert (s.t[n] == 1).all(), (bad, n)
    finally:
        s.close()
        for w in ws:
            w.close()


def _held(s, w, lens, rng):
    """Sequences of so many positions, appended by causal steps of the layer."""
    stream = torch.cuda.Stream()
    while s.t["held"].tolist() != lens:
        n = [min(8, a - b) for a, b in zip(lens, s.t["held"].tolist())]
        s.fill(n, [list(range(-1, k - 1)) for k in n], rng.standard_normal((sum(n), E)).astype(np.float32), [list(range(k)) for k in n])
        s.step([w], stream)
        torch.cuda.synchronize()
    return stream


def _layer_step(s, w, stream, **kw):
    """One layer over a plan; the rows' outputs, and the state before the plan put back."""
    p, st, x = s.p, stream.cuda_stream, s.t["x"].clone()
    keep = {n: s.t[n].clone() for n in ("pages", "k_pool", "v_pool")}
    torch.cuda.synchronize()
    s.kv.plan_dev(s.plan, stream=st)
    torch.cuda.synchronize()
    if "none" in kw:                       # (sequence, entries): pages that are taken out of the table
        for seq, n in kw.pop("none"):
            s.t["pages"][seq, :n] = -1
        torch.cuda.synchronize()
    s.L.paged_ex_dev(w, s.kv, 0, s.batch, p["x"], p["pos"], p["slot"], p["q_norm"], p["k_norm"], stream=st, **kw)
    torch.cuda.synchronize()
    assert int(s.t["status"]) == 0
    out = s.t["x"][:int(s.t["q_start"][s.n_seq])].cpu().numpy()
    s.t["x"].copy_(x)
    for n, t in keep.items():
        s.t[n].copy_(t)
    torch.cuda.synchronize()
    return out


def _close(a, b, what):
    """Outputs of two layers whose attention is off by 1e-4 of the largest at most, either."""
    assert np.isfinite(a).all() and np.isfinite(b).all()
    assert np.abs(a - b).max() <= 2e-4 * np.abs(b).max(), what


@pytest.mark.parametrize("with_tree", [False, True])
def test_a_window_is_pages_that_are_not_there(with_tree):
    """Rows that follow 32, 48 and 16 positions, in a window of 17: as without one, the pages before it taken out of the table.
    A tree's rows are all roots, at one position."""
    from kore_amd import paged
    rng = np.random.default_rng(8)
    ws = _weights(1)
    s = Server(seed=8)
    try:
        stream = _held(s, ws[0], [2 * PS, 3 * PS, PS], rng)
        n = [6, 3, 5] if with_tree else [1, 1, 1]
        s.fill(n, [[-1] * k for k in n], rng.standard_normal((sum(n), E)).astype(np.float32), [[]] * 3)
        tree = paged.Tree(s.p["mask"], 1, s.p["pos"]) if with_tree else None
        got = _layer_step(s, ws[0], stream, tree=tree, window=PS + 1)
        want = _layer_step(s, ws[0], stream, tree=tree, none=[(0, 1), (1, 2)])
        whole = _layer_step(s, ws[0], stream, tree=tree)
        _close(got, want, "window")
        first = n[0] + n[1]
        assert np.abs(got[:first] - whole[:first]).max() > 1e-2 * np.abs(whole).max(), "the window does something"
        _close(got[first:], whole[first:], "nothing lies before the third sequence's window")
    finally:
        s.close()
        for w in ws:
            w.close()


@pytest.mark.parametrize("window", [1, 3, 7, 20, 200])
def test_a_chain_of_drafts_in_a_window_is_a_chunk(window):
    """The window of a model in plan and layer: a chain given as a tree has the rows of the same tokens without one."""
    from kore_amd import paged
    rng = np.random.default_rng(window)
    ws = _weights(1)
    s = Server(seed=window)
    try:
        stream = _held(s, ws[0], [5, 40, 0], rng)
        n = [8, 3, 12]
        s.fill(n, [list(range(-1, k - 1)) for k in n], rng.standard_normal((sum(n), E)).astype(np.float32), [[]] * 3)
        s.plan.struct.window = window
        got = _layer_step(s, ws[0], stream, tree=paged.Tree(s.p["mask"], 1, s.p["pos"]), window=window)
        _close(got, _layer_step(s, ws[0], stream, window=window), "tree")
        if window < 8:
            whole = _layer_step(s, ws[0], stream)
            assert np.abs(got - whole).max() > 1e-2 * np.abs(whole).max(), "the window does something"
    finally:
        s.close()
        for w in ws:
            w.close()
