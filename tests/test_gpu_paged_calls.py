"""Calls of the rotary and paged entry points beside what else a program does."""
import ctypes as C

import pytest
import torch

from tests.paged_ref import Case, check_rows

pytestmark = pytest.mark.gpu


def test_an_error_of_another_call_is_not_theirs():
    """An error that another HIP call of the thread has left is neither reported by a call of this library nor taken away."""
    from kore_amd import hip, rope
    c = Case([(2, 40), (20, 90)], 4, 2, 64, 16, "f32", "f16", seed=1).up()
    L = hip.lib()
    L.hipPeekAtLastError.restype = L.hipGetLastError.restype = C.c_int
    with c.handle(rope.Config(64)) as kv, rope.Rope(rope.Config(64)) as r:
        pos = torch.arange(22, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        calls = [lambda: kv.append_dev(0, c.batch(), "f32", c.ptr("k"), c.ptr("v")),
                 lambda: kv.attend_dev(0, c.batch(), "f32", c.ptr("q"), c.ptr("out")),
                 lambda: kv.attend_dev(0, c.batch(1), "f32", c.ptr("q"), c.ptr("out")),
                 lambda: r.apply_dev("f32", 22, 4, 64, c.ptr("q"), pos.data_ptr(), c.ptr("out"))]
        for call in calls:
            assert L.hipSetDevice(1 << 20) != 0      # no such device
            left = L.hipPeekAtLastError()
            try:
                call()
                assert L.hipPeekAtLastError() == left
            finally:
                L.hipGetLastError()
        kv.sync()
        r.sync()


@pytest.mark.parametrize("max_q", [1, 64])
def test_the_most_sequences(max_q):
    """2^16 sequences, three of which have rows, the last among them; one more is refused, by either call, with nothing written."""
    from kore_amd import paged
    c = Case([(1, 40), (20, 90), (2, 17)], 4, 2, 64, 16, "f32", "f16", seed=2, extra_rows=1).up()
    n_seq, at = 1 << 16, [0, 40000, (1 << 16) - 1]
    starts, lens = torch.zeros(n_seq + 2, dtype=torch.int32), torch.full((n_seq + 1,), 33, dtype=torch.int32)
    pages = torch.full((n_seq + 1, c.stride), -1, dtype=torch.int32)
    for s, i in enumerate(at):
        starts[i + 1:] = int(c.starts[s + 1])
        lens[i] = int(c.kv_len[s])
        pages[i] = torch.from_numpy(c.pages[s])
    starts, lens, pages = starts.cuda(), lens.cuda(), pages.cuda()
    before = {n: t.clone() for n, t in c.d.items()}

    def batch(n):
        return paged.Batch(n, c.n_tok, starts.data_ptr(), lens.data_ptr(), pages.data_ptr(), c.stride, max_q)

    with c.handle() as kv:
        for call in (lambda b: kv.attend_dev(0, b, "f32", c.ptr("q"), c.ptr("out")),
                     lambda b: kv.append_dev(0, b, "f32", c.ptr("k"), c.ptr("v"))):
            with pytest.raises(paged.PagedError, match="n_seq"):
                call(batch(n_seq + 1))
        kv.sync()
        for n, t in before.items():
            assert torch.equal(t.view(torch.uint8), c.d[n].view(torch.uint8)), n
        kv.append_dev(0, batch(n_seq), "f32", c.ptr("k"), c.ptr("v"))
        kv.attend_dev(0, batch(n_seq), "f32", c.ptr("q"), c.ptr("out"))
        kv.sync()
    for s, (n, kv_len) in enumerate(c.lens):
        for i in range(n):
            page, slot, row = int(c.pages[s, (kv_len - n + i) // 16]), (kv_len - n + i) % 16, int(c.starts[s]) + i
            for pool, x in (("k_pool", c.k), ("v_pool", c.v)):
                assert torch.equal(c.d[pool][0, page, :, slot].cpu(), x[row].half())
    c.k_pool, c.v_pool = c.d["k_pool"].cpu(), c.d["v_pool"].cpu()
    got = c.rows("out", 4)[0]
    assert (got[c.used:] == 77.0).all()
    check_rows(c, got, *c.exact())


def test_rotated_q_in_the_place_of_k_or_v():
    """q_out may be q and lie beside k and v in wide rows, but not on any of their bytes: it would be read after it is written."""
    from kore_amd import paged, rope
    E, D, n = 4 * 64, 2 * 64, 3
    c = Case([(n, 40)], 4, 2, 64, 16, "f32", "f16", seed=1).up()
    wide = torch.randn(n, E + 2 * D + 8, device="cuda")
    at = [wide.data_ptr() + 4 * x for x in (0, E, E + D, E + 2 * D)]
    step = wide.shape[1]
    torch.cuda.synchronize()
    with c.handle(rope.Config(64)) as kv:
        def call(q, q_out, k=at[1], v=at[2], qs=step, qo=step, ks=step, vs=step):
            kv.append_dev(0, c.batch(), "f32", k, v, q=q, q_out=q_out, k_stride=ks, v_stride=vs, q_stride=qs, q_out_stride=qo)

        before = wide.clone()
        for kw, text in [
                (dict(q=c.ptr("q"), qs=E, q_out=at[1]), "k and q_out"), (dict(q=c.ptr("q"), qs=E, q_out=at[0] + 4), "k and q_out"),
                (dict(q=c.ptr("q"), qs=E, q_out=at[2]), "v and q_out"), (dict(q=c.ptr("q"), qs=E, q_out=at[0], qo=E), "k and q_out"),
                (dict(q=c.ptr("q"), qs=E, q_out=c.ptr("out"), qo=E, k=c.ptr("out"), ks=D), "k and q_out"),
                (dict(q=c.ptr("q"), qs=E, q_out=c.ptr("out"), qo=E, v=c.ptr("out") + 4 * E, vs=D), "v and q_out")]:
            with pytest.raises(paged.PagedError, match=text):
                call(**kw)
        kv.sync()
        assert torch.equal(wide, before)
        call(q=at[0], q_out=at[0])                              # in place, beside k and v
        call(q=c.ptr("q"), qs=E, q_out=c.ptr("out"), qo=E)      # apart
        kv.sync()
    assert torch.equal(wide[:, E:], before[:, E:]) and not torch.equal(wide[:, :E], before[:, :E])


def test_a_layers_step_after_an_error_of_another_call():
    """As above for the layer's steps over either cache, and the attention, matvec and matmul calls that they are made of."""
    from kore_amd import KoreAttn, hip, paged, qmv, rope
    from kore_amd.layer import Layer
    from tests.test_gpu_layer_paged import E, FF, HD, KVD, NH, NKV, _weights
    L = hip.lib()
    L.hipPeekAtLastError.restype = L.hipGetLastError.restype = C.c_int
    n, w = 5, _weights(1)[0]
    x = torch.randn(n, E, device="cuda")
    q, k, v, out = (torch.randn(n, c, device="cuda") for c in (E, KVD, KVD, E))
    p = {m: t.data_ptr() for m, t in (("x", x), ("q", q), ("k", k), ("v", v), ("out", out))}
    starts, lens, pages = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, n], [n], [0]))
    torch.cuda.synchronize()
    try:
        with paged.PagedKV(1, 2, 16, NH, NKV, HD, "f32", rope.Config(HD)) as kv, Layer(E, FF, NH, NKV, 1e-6) as layer, \
                KoreAttn(1, 32, NH, NKV, HD, 1e6) as a, KoreAttn(1, 32, 6, 3, 36, 1e6) as generic:
            b = paged.Batch(1, n, starts.data_ptr(), lens.data_ptr(), pages.data_ptr(), 1, n)
            calls = [lambda: layer.paged_dev(w, kv, 0, b, p["x"]),
                     lambda: layer.prefill_dev(w, a, 0, 0, n, p["x"]),
                     lambda: layer.decode_dev(w, a, 0, n, p["x"]),
                     lambda: a.prefill_dev(0, 0, n, p["q"], p["k"], p["v"], p["out"]),
                     lambda: a.append_dev(0, n, 1, p["k"], p["v"]),
                     lambda: a.decode_dev(0, n, p["q"], p["k"], p["v"], p["out"]),
                     lambda: generic.decode_dev(0, 0, p["q"], p["k"], p["v"], p["out"]),
                     lambda: qmv.rmsnorm_rows_dev(p["x"], w.bufs["attn_norm"].ptr, E, n, 1e-6, p["out"]),
                     lambda: w.mats[0].mv_dev(p["x"], p["out"]),
                     lambda: w.mats[0].matmul_batch_dev(p["x"], n, p["out"])]
            for i, call in enumerate(calls):
                assert L.hipSetDevice(1 << 20) != 0      # no such device
                left = L.hipPeekAtLastError()
                try:
                    call()
                    assert L.hipPeekAtLastError() == left, i
                finally:
                    L.hipGetLastError()
            torch.cuda.synchronize()
    finally:
        w.close()
