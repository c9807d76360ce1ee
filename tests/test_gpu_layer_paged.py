"""kore_layer_paged_dev: a layer's step over the new rows of several sequences, the way a server runs it, against the same
sequences one after the other through kore_layer_prefill_dev and the contiguous cache."""
import numpy as np
import pytest
import torch

import oracle
from tests.test_gpu_layer import _synth

pytestmark = pytest.mark.gpu

E, FF, NH, NKV, HD = 512, 1024, 4, 2, 128
KVD = NKV * HD


def _weights(n_layer):
    from kore_amd import hip
    from kore_amd.layer import LayerWeights
    rng = np.random.default_rng(21)
    shapes = [(E, E), (KVD, E), (KVD, E), (E, E), (FF, E), (FF, E), (E, FF)]
    types = [oracle.TYPE_Q4K, oracle.TYPE_Q4K, oracle.TYPE_Q6K, oracle.TYPE_Q4K, oracle.TYPE_Q4K, oracle.TYPE_Q4K, oracle.TYPE_Q6K]
    out = []
    for l in range(n_layer):
        w = LayerWeights()
        w.mats = [_synth(t, r, c, 900 + 10 * l + j)[0] for j, (t, (r, c)) in enumerate(zip(types, shapes))]
        for name, n in (("attn_norm", E), ("ffn_norm", E), ("bq", E), ("bk", KVD), ("bv", KVD)):
            a = rng.standard_normal(n) * 0.2 + (1.0 if "norm" in name else 0.0)
            w.bufs[name] = hip.DeviceBuffer.from_array(a.astype(np.float32))
        out.append(w)
    return out


def test_steps_of_two_sequences():
    """Two layers; prompts in chunks beside single tokens.  Both sides share every kernel but the cache's and the
    attention's, whose outputs agree to 2 x 1e-4 of the largest (kore's tolerance, each side)."""
    from kore_amd import KoreAttn, paged, rope
    from kore_amd.layer import Layer
    rng = np.random.default_rng(5)
    total, n_layer, ps = [40, 23], 2, 16
    x0 = [rng.standard_normal((t, E)).astype(np.float32) for t in total]
    ws = _weights(n_layer)
    try:
        want = []
        with Layer(E, FF, NH, NKV, 1e-6) as L:
            for x in x0:
                d = torch.from_numpy(x).cuda()
                torch.cuda.synchronize()
                with KoreAttn(n_layer, len(x), NH, NKV, HD, 1e6) as a:
                    for l in range(n_layer):
                        L.prefill_dev(ws[l], a, l, 0, len(x), d.data_ptr())
                    L.sync()
                want.append(d.cpu().numpy())
            pages = torch.from_numpy(rng.permutation(6).astype(np.int32).reshape(2, 3)).cuda()
            done = [0, 0]
            with paged.PagedKV(n_layer, 6, ps, NH, NKV, HD, "f32", rope.Config(HD)) as kv:
                for step in [(17, 1), (1, 9), (0, 12), (21, 1), (1, 0)]:
                    rows = np.concatenate([x[d:d + m] for x, d, m in zip(x0, done, step)])
                    done = [d + m for d, m in zip(done, step)]
                    x = torch.from_numpy(rows).cuda()
                    starts = torch.tensor([0, step[0], sum(step)], dtype=torch.int32).cuda()
                    lens = torch.tensor(done, dtype=torch.int32).cuda()
                    torch.cuda.synchronize()
                    b = paged.Batch(2, sum(step), starts.data_ptr(), lens.data_ptr(), pages.data_ptr(), 3, max(step))
                    for l in range(n_layer):
                        L.paged_dev(ws[l], kv, l, b, x.data_ptr())
                    L.sync()
                    w = np.concatenate([o[d - m:d] for o, d, m in zip(want, done, step)])
                    assert np.abs(x.cpu().numpy() - w).max() <= 2e-4 * np.abs(w).max(), step
            assert done == total
    finally:
        for w in ws:
            w.close()


@pytest.mark.parametrize("cache", ["f32", "f16", "bf16"])
def test_a_layer_is_its_calls(cache):
    """The same bits as the library's calls that a layer is made of, one by one."""
    from kore_amd import hip, paged, qmv, rope
    from kore_amd.layer import Layer
    rng = np.random.default_rng(6)
    w = _weights(1)[0]
    lens, ps, n_pages = [(3, 20), (1, 33), (30, 30)], 16, 8
    n = sum(m for m, _ in lens)
    x = torch.from_numpy(rng.standard_normal((n, E)).astype(np.float32)).cuda()
    pool = (0.1 * torch.randn(2, 1, n_pages, NKV, ps, HD, generator=torch.Generator().manual_seed(1))).to(
        {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[cache])
    table = rng.permutation(n_pages).astype(np.int32)
    pages = torch.full((3, 3), -1, dtype=torch.int32)
    pages[0, :2], pages[1], pages[2, :2] = torch.from_numpy(table[:2]), torch.from_numpy(table[2:5]), torch.from_numpy(table[5:7])
    pages = pages.cuda()
    starts = torch.tensor([0, 3, 4, 34], dtype=torch.int32).cuda()
    kv_len = torch.tensor([kv for _, kv in lens], dtype=torch.int32).cuda()
    b = paged.Batch(3, n, starts.data_ptr(), kv_len.data_ptr(), pages.data_ptr(), 3, 30)
    got = []
    try:
        for whole in (True, False):
            k_pool, v_pool, y = pool[0].clone().cuda(), pool[1].clone().cuda(), x.clone()
            torch.cuda.synchronize()
            with paged.PagedKV(1, n_pages, ps, NH, NKV, HD, cache, rope.Config(HD), k_pool.data_ptr(), v_pool.data_ptr()) as kv, \
                    Layer(E, FF, NH, NKV, 1e-6) as L:
                if whole:
                    L.paged_dev(w, kv, 0, b, y.data_ptr())
                    L.sync()
                else:
                    t = {m: torch.empty(n, c, device="cuda") for m, c in (("h", E), ("q", E), ("k", KVD), ("v", KVD), ("a", E), ("g", FF), ("u", FF))}
                    p = {m: t[m].data_ptr() for m in t}
                    buf = {m: w.bufs[m].ptr for m in w.bufs}
                    s = torch.cuda.Stream()
                    st = s.cuda_stream
                    qmv.rmsnorm_rows_dev(y.data_ptr(), buf["attn_norm"], E, n, 1e-6, p["h"], st)
                    qmv.matmul_batch_group_ex_dev(w.mats[:3], p["h"], n, [p["q"], p["k"], p["v"]], [buf["bq"], buf["bk"], buf["bv"]], stream=st)
                    kv.append_dev(0, b, "f32", p["k"], p["v"], p["q"], p["q"], stream=st)
                    kv.attend_dev(0, b, "f32", p["q"], p["a"], stream=st)
                    qmv.matmul_batch_group_ex_dev([w.mats[3]], p["a"], n, [y.data_ptr()], accumulate=True, stream=st)
                    qmv.rmsnorm_rows_dev(y.data_ptr(), buf["ffn_norm"], E, n, 1e-6, p["h"], st)
                    qmv.matmul_batch_group_ex_dev(w.mats[4:6], p["h"], n, [p["g"], p["u"]], stream=st)
                    qmv.swiglu_dev(p["g"], p["u"], n * FF, st)
                    qmv.matmul_batch_group_ex_dev([w.mats[6]], p["g"], n, [y.data_ptr()], accumulate=True, stream=st)
                    s.synchronize()
            got.append([y.cpu(), k_pool.cpu(), v_pool.cpu()])
        assert torch.isfinite(got[0][0]).all() and not torch.equal(got[0][0], x.cpu())
        for a, c in zip(*got):
            assert torch.equal(a.contiguous().view(torch.uint8), c.contiguous().view(torch.uint8))
        hip.synchronize()
    finally:
        w.close()


def test_a_captured_step_follows_its_batch():
    """A layer's step captured once and replayed with other rows, lengths and pages, the program's own steps between the
    replays: the eager step's bits every time.  The captured step has a workspace of its own."""
    from kore_amd import paged, rope
    from kore_amd.layer import Layer
    ws = _weights(1)
    n_pages, ps, stride, n = 160, 32, 70, 7
    try:
        with paged.PagedKV(1, n_pages, ps, NH, NKV, HD, "f32", rope.Config(HD)) as kv, Layer(E, FF, NH, NKV, 1e-6) as L:
            starts = torch.zeros(4, dtype=torch.int32, device="cuda")
            kv_len = torch.zeros(3, dtype=torch.int32, device="cuda")
            pages = torch.full((3, stride), -1, dtype=torch.int32, device="cuda")
            x = torch.zeros(n, E, device="cuda")
            work = torch.empty(kv.workspace_bytes(), dtype=torch.uint8, device="cuda")
            b = paged.Batch(3, n, starts.data_ptr(), kv_len.data_ptr(), pages.data_ptr(), stride, 5)
            stream = torch.cuda.Stream()

            def fill(i):
                torch.cuda.synchronize()
                r = np.random.default_rng(100 + i)
                starts.copy_(torch.tensor([[0, 1, 2, 7], [0, 5, 6, 7], [0, 0, 4, 5], [0, 2, 4, 7]][i], dtype=torch.int32))
                kv_len.copy_(torch.tensor([[40, 2000, 5], [2200, 3, 33], [0, 900, 64], [2, 1500, 300]][i], dtype=torch.int32))
                order = r.permutation(n_pages)[:150].astype(np.int32)
                t = np.full((3, stride), -1, np.int32)
                t[0], t[1], t[2, :10] = order[:70], order[70:140], order[140:150]
                pages.copy_(torch.from_numpy(t))
                x.copy_(torch.from_numpy(r.standard_normal((n, E)).astype(np.float32)))
                torch.cuda.synchronize()

            fill(0)
            L.paged_dev(ws[0], kv, 0, b, x.data_ptr(), stream=stream.cuda_stream)
            fill(0)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                L.paged_dev(ws[0], kv, 0, b, x.data_ptr(), workspace=work.data_ptr(),
                            stream=torch.cuda.current_stream().cuda_stream)
            for i in (1, 0, 2, 3, 1):
                fill(i)
                L.paged_dev(ws[0], kv, 0, b, x.data_ptr(), stream=stream.cuda_stream)
                stream.synchronize()
                want = x[:int(starts[3])].clone()   # the rows behind the last sequence hold nothing of use
                fill(i)
                g.replay()
                torch.cuda.synchronize()
                got = x[:int(starts[3])]
                assert torch.isfinite(got).all() and torch.equal(got.view(torch.int32), want.view(torch.int32)), i
            del g
    finally:
        for w in ws:
            w.close()


def test_refusals():
    from kore_amd import paged
    from kore_amd.layer import Layer, LayerError
    ws = _weights(1)
    try:
        z = torch.zeros(64, dtype=torch.int32, device="cuda")
        x = torch.ones(64, E, device="cuda")
        torch.cuda.synchronize()
        good = paged.Batch(1, 2, z.data_ptr(), z.data_ptr(), z.data_ptr(), 4)
        with Layer(E, FF, NH, NKV, 1e-6) as L, paged.PagedKV(1, 4, 16, NH, NKV, HD) as kv, paged.PagedKV(1, 4, 16, NH, NH, HD) as other:
            def batch(**kw):
                b = paged.Batch(1, 2, z.data_ptr(), z.data_ptr(), z.data_ptr(), 4)
                for k, v in kw.items():
                    setattr(b.struct, k, v)
                return b

            for args, kw, text in [((other, 0, good, x.data_ptr()), {}, "geometry"), ((kv, 1, good, x.data_ptr()), {}, "layer"),
                                   ((kv, 0, good, x.data_ptr() + 4), {}, "unaligned"), ((kv, 0, batch(n_tok=65), x.data_ptr()), {}, "n_tok"),
                                   ((kv, 0, batch(n_tok=0), x.data_ptr()), {}, "n_tok"), ((kv, 0, batch(n_seq=0), x.data_ptr()), {}, "sequence"),
                                   ((kv, 0, batch(pages=None), x.data_ptr()), {}, "array"), ((kv, 0, good, x.data_ptr()), {"workspace": 8}, "workspace")]:
                with pytest.raises(LayerError) as e:
                    L.paged_dev(ws[0], *args, **kw)
                assert text in str(e.value)
            L.sync()
        assert (x == 1).all()
    finally:
        for w in ws:
            w.close()
