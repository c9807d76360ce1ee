"""Steps of drafted trees through whole layers, the way a server runs them: the step's tables made on the GPU, normalised heads
stored by slots, the trees attended, their accepted paths kept, eagerly and as one captured graph."""
import numpy as np
import pytest
import torch

from tests import step_ref
from tests.test_gpu_layer_paged import E, FF, HD, KVD, NH, NKV, _weights

pytestmark = pytest.mark.gpu

PS, STRIDE, N_PAGES, N_TOK, N_LAYER = 16, 12, 40, 24, 2


class Server:
    """Three sequences' state on the GPU, and the calls of a step over it."""

    def __init__(self, n_seq=3, seed=0, cache="f32"):
        from kore_amd import paged, rope
        from kore_amd.layer import Layer
        rng = np.random.default_rng(seed)
        self.n_seq = n_seq
        i32 = {"dtype": torch.int32, "device": "cuda"}
        self.t = {"n_new": torch.zeros(n_seq, **i32), "held": torch.zeros(n_seq, **i32), "kv_len": torch.zeros(n_seq, **i32),
                  "pages": torch.full((n_seq, STRIDE), -1, **i32), "free": torch.from_numpy(rng.permutation(N_PAGES).astype(np.int32)).cuda(),
                  "n_free": torch.full((1,), N_PAGES, **i32), "n_taken": torch.zeros(1, **i32), "parent": torch.zeros(N_TOK, **i32),
                  "q_start": torch.zeros(n_seq + 1, **i32), "pos": torch.zeros(N_TOK, **i32), "status": torch.zeros(1, **i32),
                  "slot": torch.zeros(N_TOK, dtype=torch.int64, device="cuda"), "mask": torch.zeros(N_TOK, dtype=torch.int64, device="cuda"),
                  "n_keep": torch.zeros(n_seq, **i32), "rows": torch.zeros(N_TOK, **i32), "x": torch.zeros(N_TOK, E, device="cuda"),
                  "q_norm": torch.from_numpy(1 + 0.3 * rng.standard_normal(HD).astype(np.float32)).cuda(),
                  "k_norm": torch.from_numpy(1 + 0.3 * rng.standard_normal(HD).astype(np.float32)).cuda()}
        ct = {"f32": torch.float32, "f16": torch.float16}[cache]
        for n in ("k_pool", "v_pool"):
            self.t[n] = torch.zeros(N_LAYER, N_PAGES, NKV, PS, HD, dtype=ct, device="cuda")
        p = self.p = {n: t.data_ptr() for n, t in self.t.items()}
        torch.cuda.synchronize()
        self.L = Layer(E, FF, NH, NKV, 1e-6)
        self.kv = paged.PagedKV(N_LAYER, N_PAGES, PS, NH, NKV, HD, cache, rope.Config(HD), p["k_pool"], p["v_pool"])
        self.plan = paged.Plan(n_seq, N_TOK, p["n_new"], p["held"], p["kv_len"], p["pages"], STRIDE, p["free"], p["n_free"], p["n_taken"],
                               p["q_start"], p["pos"], p["slot"], p["status"], p["parent"], p["mask"], 1)
        self.batch = paged.Batch(n_seq, N_TOK, p["q_start"], p["kv_len"], p["pages"], STRIDE, 16)
        self.tree = paged.Tree(p["mask"], 1)
        self.keep = paged.Keep(n_seq, N_TOK, p["q_start"], p["n_keep"], p["kv_len"], p["held"], p["pages"], STRIDE, p["rows"], p["free"],
                               p["n_taken"], p["n_free"])

    def step(self, ws, stream, workspace=None):
        p, st = self.p, stream.cuda_stream
        self.kv.plan_dev(self.plan, stream=st)
        for l, w in enumerate(ws):
            self.L.paged_ex_dev(w, self.kv, l, self.batch, p["x"], p["pos"], p["slot"], p["q_norm"], p["k_norm"], self.tree,
                                workspace=workspace, stream=st)
        self.kv.keep_dev(self.keep, stream=st)

    def fill(self, n_new, parents, x, paths):
        """A step's requests: rows' parents, their inputs, and the paths that will be kept (None: the sequence ends)."""
        torch.cuda.synchronize()
        flat = [q for s in parents for q in s]
        rows = np.zeros(N_TOK, np.int32)
        at = 0
        for n, path in zip(n_new, paths):
            rows[at:at + len(path or [])] = path or []
            at += n
        put = lambda n, v: self.t[n][:len(v)].copy_(torch.as_tensor(np.asarray(v), dtype=self.t[n].dtype))  # noqa: E731
        put("n_new", n_new)
        put("parent", flat)
        put("x", np.concatenate([x, np.zeros((N_TOK - len(x), E), np.float32)]))
        put("n_keep", [-1 if path is None else len(path) for path in paths])
        put("rows", rows)
        torch.cuda.synchronize()

    def close(self):
        self.kv.close()
        self.L.close()


def _path(rng, parent):
    """A root's path down a tree."""
    path, at = [], -1
    while True:
        below = [i for i, q in enumerate(parent) if q == at]
        if not below or (path and rng.random() < 0.2):
            return path
        at = int(rng.choice(below))
        path.append(at)


def _requests(rng, n_seq):
    """(rows, parents, paths) of a step."""
    n_new = [int(rng.integers(0, 9)) for _ in range(n_seq)]
    parents = [step_ref.tree(rng, n, 2) for n in n_new]
    return n_new, parents, [_path(rng, q) if q else [] for q in parents]


def test_accepted_paths_are_the_sequences():
    """Steps of drafted trees; then each sequence's accepted rows once more as one causal chunk of a fresh cache.  Both sides
    share every kernel but the attention, whose outputs agree to 2 x 1e-4 of the largest (each side's tolerance), and two layers
    pass it on; and the trees' rows that were refused leave nothing."""
    rng = np.random.default_rng(3)
    ws = _weights(N_LAYER)
    s, plain = Server(), Server(seed=1)
    try:
        for n in ("q_norm", "k_norm"):
            plain.t[n].copy_(s.t[n])
        stream = torch.cuda.Stream()
        kept_x, kept_y = [[] for _ in range(3)], [[] for _ in range(3)]
        for _ in range(9):
            n_new, parents, paths = _requests(rng, 3)
            x = rng.standard_normal((sum(n_new), E)).astype(np.float32)
            s.fill(n_new, parents, x, paths)
            s.step(ws, stream)
            torch.cuda.synchronize()
            assert int(s.t["status"]) == 0
            y = s.t["x"].cpu().numpy()
            at = 0
            for i, (n, path) in enumerate(zip(n_new, paths)):
                kept_x[i] += [x[at + r] for r in path]
                kept_y[i] += [y[at + r] for r in path]
                at += n
            lens = [len(k) for k in kept_x]
            assert s.t["held"].tolist() == lens
            assert int(s.t["n_free"]) == N_PAGES - sum(-(-n // PS) for n in lens)
        assert min(lens) > 8
        from kore_amd import paged
        for i in range(3):
            at = 0
            while at < lens[i]:
                n = min(16, lens[i] - at)
                plain.fill([n, 0, 0] if i == 0 else [0, n, 0] if i == 1 else [0, 0, n], [list(range(-1, n - 1))],
                           np.asarray(kept_x[i][at:at + n]), [list(range(n)) if j == i else [] for j in range(3)])
                p = plain.p
                plain.kv.plan_dev(plain.plan, stream=stream.cuda_stream)
                for l, w in enumerate(ws):
                    plain.L.paged_ex_dev(w, plain.kv, l, plain.batch, p["x"], p["pos"], p["slot"], p["q_norm"], p["k_norm"], stream=stream.cuda_stream)
                plain.kv.keep_dev(paged.Keep(3, N_TOK, p["q_start"], p["n_keep"], p["kv_len"], p["held"], p["pages"], STRIDE, None, p["free"],
                                             p["n_taken"], p["n_free"]), stream=stream.cuda_stream)
                torch.cuda.synchronize()
                got = plain.t["x"][:n].cpu().numpy()
                want = np.asarray(kept_y[i][at:at + n])
                assert np.isfinite(want).all() and np.abs(got - want).max() <= 4e-4 * np.abs(want).max()
                at += n
        assert plain.t["held"].tolist() == lens
    finally:
        s.close()
        plain.close()
        for w in ws:
            w.close()


@pytest.mark.parametrize("cache", ["f32", "f16"])
def test_a_captured_step_is_the_eager_one(cache):
    """Plan, layers and keep as one graph, replayed with other requests, the program's own steps between the replays: the same
    bits, sequences that end and a step that the free pages do not hold among them."""
    rng = np.random.default_rng(4)
    ws = _weights(N_LAYER)
    s, e = Server(cache=cache), Server(cache=cache)
    try:
        work = torch.empty(s.kv.workspace_bytes(), dtype=torch.uint8, device="cuda")
        stream = torch.cuda.Stream()
        s.step(ws, stream, work.data_ptr())   # (no rows)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            s.step(ws, torch.cuda.current_stream(), work.data_ptr())
        state = ("held", "kv_len", "pages", "free", "n_free", "n_taken", "q_start", "pos", "slot", "mask", "status", "k_pool", "v_pool")
        seen = set()
        for step in range(12):
            n_new, parents, paths = _requests(rng, 3)
            if step in (5, 9):
                paths[step % 3] = None
            x = rng.standard_normal((sum(n_new), E)).astype(np.float32)
            for t in (s, e):
                t.fill(n_new, parents, x, paths)
                if step == 7:
                    t.t["n_free"].zero_()      # others have taken them
                    torch.cuda.synchronize()
                if step == 8:
                    t.t["n_free"].fill_(20)
                    torch.cuda.synchronize()
            if step == 7:
                n_new[0] = 17
                for t in (s, e):
                    t.t["n_new"][0] = 17
                    torch.cuda.synchronize()
            e.step(ws, stream)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            seen.add(min(1, int(e.t["status"])))
            used = int(e.t["q_start"][3])
            assert torch.isfinite(e.t["x"][:used]).all()
            assert torch.equal(s.t["x"][:used].view(torch.int32), e.t["x"][:used].view(torch.int32)), step
            for n in state:
                assert torch.equal(s.t[n].contiguous().view(torch.uint8), e.t[n].contiguous().view(torch.uint8)), (step, n)
        assert seen == {0, 1}
        del g
    finally:
        s.close()
        e.close()
        for w in ws:
            w.close()


@pytest.mark.parametrize("with_tree", [False, True])
def test_a_layer_is_its_calls(with_tree):
    """The same bits as the library's calls that a layer is made of; without norms and tree, as kore_layer_paged_dev."""
    from kore_amd import paged, qmv
    rng = np.random.default_rng(6)
    ws = _weights(1)
    w = ws[0]
    got = []
    try:
        for how in ("whole", "calls") if with_tree else ("whole", "calls", "bare", "paged"):
            s = Server(seed=5)
            r = np.random.default_rng(7)
            n_new, parents = [7, 1, 12], [step_ref.tree(r, n, 2) for n in (7, 1, 12)]
            s.fill(n_new, parents if with_tree else [list(range(-1, n - 1)) for n in n_new], r.standard_normal((20, E)).astype(np.float32), [[0]] * 3)
            p, st = s.p, torch.cuda.Stream()
            c = st.cuda_stream
            for _ in range(2):   # once to have something cached
                s.kv.plan_dev(s.plan, stream=c)
                if how == "whole":
                    s.L.paged_ex_dev(w, s.kv, 0, s.batch, p["x"], p["pos"], p["slot"], p["q_norm"], p["k_norm"], s.tree if with_tree else None,
                                     stream=c)
                elif how == "bare":
                    s.L.paged_ex_dev(w, s.kv, 0, s.batch, p["x"], p["pos"], p["slot"], stream=c)
                elif how == "paged":
                    s.L.paged_dev(w, s.kv, 0, s.batch, p["x"], stream=c)
                else:
                    t = {m: torch.empty(N_TOK, d, device="cuda") for m, d in (("h", E), ("q", E), ("k", KVD), ("v", KVD), ("a", E), ("g", FF), ("u", FF))}
                    torch.cuda.synchronize()
                    b = {m: x.data_ptr() for m, x in t.items()}
                    buf = {m: w.bufs[m].ptr for m in w.bufs}
                    qmv.rmsnorm_rows_dev(p["x"], buf["attn_norm"], E, N_TOK, 1e-6, b["h"], c)
                    qmv.matmul_batch_group_ex_dev(w.mats[:3], b["h"], N_TOK, [b["q"], b["k"], b["v"]], [buf["bq"], buf["bk"], buf["bv"]], stream=c)
                    s.kv.append_rows_dev(0, paged.Rows(N_TOK, p["pos"], p["slot"], p["q_norm"], p["k_norm"]), "f32", b["k"], b["v"], b["q"], b["q"],
                                         stream=c)
                    if with_tree:
                        s.kv.attend_tree_dev(0, s.batch, s.tree, "f32", b["q"], b["a"], stream=c)
                    else:
                        s.kv.attend_dev(0, s.batch, "f32", b["q"], b["a"], stream=c)
                    qmv.matmul_batch_group_ex_dev([w.mats[3]], b["a"], N_TOK, [p["x"]], accumulate=True, stream=c)
                    qmv.rmsnorm_rows_dev(p["x"], buf["ffn_norm"], E, N_TOK, 1e-6, b["h"], c)
                    qmv.matmul_batch_group_ex_dev(w.mats[4:6], b["h"], N_TOK, [b["g"], b["u"]], stream=c)
                    qmv.swiglu_dev(b["g"], b["u"], N_TOK * FF, c)
                    qmv.matmul_batch_group_ex_dev([w.mats[6]], b["g"], N_TOK, [p["x"]], accumulate=True, stream=c)
                torch.cuda.synchronize()
                s.t["held"].copy_(s.t["kv_len"])
                s.t["n_free"].copy_(s.t["n_taken"])
                torch.cuda.synchronize()
            got.append([s.t[m].cpu() for m in ("x", "k_pool", "v_pool")])
            got[-1][0] = got[-1][0][:20]
            s.close()
        assert torch.isfinite(got[0][0]).all()
        for a, b in list(zip(got[0], got[1])) + ([] if with_tree else list(zip(got[2], got[3]))):
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
        if not with_tree:
            assert not torch.equal(got[0][0], got[2][0]), "the norms do something"
    finally:
        w.close()


def test_refusals():
    from kore_amd import paged
    from kore_amd.layer import Layer, LayerError
    ws = _weights(1)
    s = Server()
    try:
        p = s.p
        s.t["x"].fill_(1.0)
        torch.cuda.synchronize()
        good = dict(pos=p["pos"], slot=p["slot"], q_norm=p["q_norm"], k_norm=p["k_norm"], tree=s.tree)
        with paged.PagedKV(1, 4, 16, NH, NH, HD) as other, Layer(E, FF, NH, NKV, 0.0) as no_eps:
            for L, kv, layer, kw, text in [
                    (s.L, s.kv, 0, dict(pos=None), "pos"), (s.L, s.kv, 0, dict(slot=None), "slot"), (s.L, s.kv, 0, dict(slot=p["slot"] + 4), "slot"),
                    (s.L, s.kv, 0, dict(pos=p["pos"] + 1), "pos"), (s.L, s.kv, 0, dict(q_norm=p["q_norm"] + 2), "q_norm"), (s.L, s.kv, 0, dict(window=-1), "window"),
                    (s.L, s.kv, 0, dict(window=4), "pos"), (s.L, s.kv, 0, dict(tree=paged.Tree(None)), "mask"),
                    (s.L, s.kv, 0, dict(tree=paged.Tree(p["mask"], 17)), "mask_words"), (s.L, s.kv, 2, {}, "layer"), (s.L, other, 0, {}, "geometry"),
                    (s.L, s.kv, 0, dict(workspace=8), "workspace"), (no_eps, s.kv, 0, {}, "rms_eps")]:
                with pytest.raises(LayerError) as e:
                    L.paged_ex_dev(ws[0], kv, layer, s.batch, p["x"], **{**good, **kw})
                assert text in str(e.value)
            s.L.sync()
        assert (s.t["x"] == 1).all()
    finally:
        s.close()
        for w in ws:
            w.close()
