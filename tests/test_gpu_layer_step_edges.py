"""A layer's step of drafted tokens at its edges: batches that its attention would refuse."""
import pytest
import torch

from tests.test_gpu_layer_paged import _weights
from tests.test_gpu_layer_step import N_TOK, STRIDE, Server

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
