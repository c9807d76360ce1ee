"""A step of drafted tokens over the paged KV cache, as cases that can be timed and compared.

Five operators around the cache that a server runs between and within its layers: the step's tables made from the requests'
lengths (`plan`: pages, positions, slots, and the ancestors of a drafted tree), norms of q's and k's heads with the rotation
(`norm`) and with the store by slots (`store`), the attention of a tree of drafted tokens over a sequence's pages (`tree`),
and the accepted rows moved together in the cache of every layer (`keep`).  `run` computes them in plain torch operations
or, with `own` set, through the library.  Geometries are those of the benchmark and the tests (the Qwen2.5 widths, and one
outside that family); values are synthetic.
"""
from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BASE, EPS = 1e6, 1e-6

# (n_head, n_head_kv, head_dim) of the 0.5B, 1.5B, 3B and 7B models, and one that is none of them
FAMILY = [(14, 2, 64), (12, 2, 128), (16, 2, 128), (28, 4, 128)]
OTHER = (33, 3, 96)


def _geo(g):
    return {"nh": g[0], "nkv": g[1], "hd": g[2]}


def listed():
    return [
        # one more token of one conversation: all latency
        {"name": "plan_token", "op": "plan", "seqs": 1, "new": 1, "held": 500, "mix": "same", "page": 16, "width": 0, "words": 0,
         "short": False},
        # trees of 32 drafted tokens of 64 running sequences
        {"name": "plan_trees", "op": "plan", "seqs": 64, "new": 32, "held": 4000, "mix": "ragged", "page": 16, "width": 5, "words": 1,
         "short": False},
        # a thousand sequences' tokens beside chunks of prompts
        {"name": "plan_crowd", "op": "plan", "seqs": 1000, "new": 33, "held": 2000, "mix": "ragged", "page": 64, "width": 0, "words": 0,
         "short": False},
        # one token's q and k heads: all latency
        {"name": "norm_token", "op": "norm", "rows": 1, **_geo(FAMILY[3]), "rot": 128, "layout": "half", "type": "f32", "far": 4096},
        # a long prompt's rows
        {"name": "norm_prompt", "op": "norm", "rows": 4000, **_geo(FAMILY[3]), "rot": 128, "layout": "half", "type": "bf16", "far": 32768},
        # one token of each of 16 running sequences, stored
        {"name": "store_step", "op": "store", **_geo(FAMILY[3]), "seqs": 16, "new": 1, "held": 3000, "mix": "ragged", "page": 16,
         "width": 0, "type": "f32", "cache": "f16", "layout": "half"},
        # trees of up to 48 drafted tokens of 32 sequences
        {"name": "store_trees", "op": "store", **_geo(FAMILY[3]), "seqs": 32, "new": 48, "held": 1000, "mix": "ragged", "page": 32,
         "width": 6, "type": "f32", "cache": "bf16", "layout": "half"},
        # eight drafted tokens of one conversation on the smallest model: all latency
        {"name": "tree_small", "op": "tree", **_geo(FAMILY[0]), "seqs": 1, "new": 8, "held": 500, "mix": "same", "page": 16, "width": 2,
         "window": 0, "type": "f32", "cache": "f32"},
        # trees of 32 drafted tokens of 16 running sequences
        {"name": "tree_step", "op": "tree", **_geo(FAMILY[3]), "seqs": 16, "new": 32, "held": 8000, "mix": "ragged", "page": 16, "width": 5,
         "window": 0, "type": "f32", "cache": "f16"},
        # a tree over a very long context
        {"name": "tree_long", "op": "tree", **_geo(FAMILY[2]), "seqs": 1, "new": 63, "held": 131000, "mix": "same", "page": 256, "width": 8,
         "window": 0, "type": "bf16", "cache": "bf16"},
        # the accepted path of one conversation's tree, smallest model
        {"name": "keep_one", "op": "keep", "layers": 24, **_geo(FAMILY[0]), "seqs": 1, "new": 16, "kept": 4, "held": 100, "mix": "same",
         "page": 16, "cache": "f32", "end": 0},
        # the accepted paths of 32 sequences, two of which end
        {"name": "keep_step", "op": "keep", "layers": 28, **_geo(FAMILY[3]), "seqs": 32, "new": 32, "kept": 7, "held": 40, "mix": "ragged",
         "page": 16, "cache": "f16", "end": 2},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_geo(rng):
    if rng.random() < 0.35:
        nkv = rng.randint(1, 6)
        return nkv * rng.randint(1, 10), nkv, 8 * rng.randint(4, 20)
    return rng.choice(FAMILY + [OTHER])


def draw(rng):
    op = rng.choice(["plan", "norm", "store", "tree", "tree", "keep"])
    page, mix = rng.choice([16, 32, 64, 128, 256]), rng.choice(["same", "ragged", "ragged", "mixed"])
    if op == "plan":
        c = {"op": op, "seqs": _log_int(rng, 1, 1000), "new": _log_int(rng, 1, 2000), "mix": mix, "page": page, "width": 0, "words": 0,
             "short": rng.random() < 0.1}
        if rng.random() < 0.5:
            c["words"] = rng.choice([1, 1, 2, 5])
            c["new"] = _log_int(rng, 1, 64 * c["words"])
            c["width"] = _log_int(rng, 1, 1 + c["new"] // 4)
        while c["seqs"] * (c["new"] * (16 + 8 * c["words"] if c["words"] else 12) + 32) > 300_000:
            c["seqs"] = max(1, c["seqs"] // 2)
        return {**c, "held": _log_int(rng, 1, min(32000, 2_000_000 // c["seqs"]))}
    geo = _geo(_draw_geo(rng))
    layout = rng.choice(["half", "half", "interleaved"])
    act, cache = rng.choice([("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
    if op == "norm":
        rot = geo["hd"] if rng.random() < 0.6 else 2 * rng.randint(4, geo["hd"] // 2)
        kind = rng.choice(sorted(TYPES))
        most = 64_000_000 // (2 * (geo["nh"] + geo["nkv"]) * geo["hd"] * _SIZE[kind])
        return {"op": op, "rows": _log_int(rng, 1, min(3900, most)), **geo, "rot": rot, "layout": layout, "type": kind,
                "far": _log_int(rng, 4096, 1000000)}
    new = rng.choice([1, _log_int(rng, 2, 64), _log_int(rng, 2, 64)])
    c = {"op": op, **geo, "seqs": _log_int(rng, 1, 32), "new": new, "mix": mix, "page": page, "width": _log_int(rng, 1, 1 + new // 4)}
    if op == "store":
        while c["seqs"] * new * (2 * geo["nh"] * _SIZE[act] + 2 * geo["nkv"] * (_SIZE[act] + _SIZE[cache])) * geo["hd"] > 36_000_000:
            c["seqs"] = c["seqs"] * 3 // 4
        return {**c, "held": _log_int(rng, 1, 2000), "type": act, "cache": cache, "layout": layout}
    if op == "keep":
        row = 2 * geo["nkv"] * geo["hd"] * _SIZE[cache]
        c["held"] = _log_int(rng, 1, 100)
        c["layers"] = rng.randint(1, 28)
        while c["seqs"] * (c["held"] + c["new"] + page) * row * c["layers"] > 120_000_000 and c["seqs"] > 1:
            c["seqs"] = max(1, c["seqs"] // 2)
        while (c["held"] + c["new"] + page) * row * c["layers"] > 120_000_000 and c["layers"] > 1:
            c["layers"] = max(1, c["layers"] // 2)
        del c["width"]
        return {**c, "kept": rng.randint(1, min(8, (new + 1) // 2)), "cache": cache, "end": 1 if c["seqs"] > 4 and rng.random() < 0.4 else 0}
    if rng.random() < 0.15:  # a wide tree
        c["new"] = _log_int(rng, 65, 333)
        c["width"] = c["new"] // 8
    row = 2 * geo["nkv"] * geo["hd"] * _SIZE[cache]  # bytes of one position
    c["held"] = _log_int(rng, 1, max(2, min(131000, 130_000_000 // row // c["seqs"])))
    while c["seqs"] * c["new"] * geo["nh"] * (c["held"] + c["new"]) > 120_000_000:
        if c["seqs"] > 1:
            c["seqs"] = c["seqs"] * 3 // 4
        else:
            c["held"] = max(1, c["held"] // 2)
            c["new"] = max(1, c["new"] * 3 // 4)
            c["width"] = max(1, min(c["width"], c["new"]))
    return {**c, "window": 0 if rng.random() < 0.75 else _log_int(rng, 64, 2048), "type": act, "cache": cache}


# ---- inputs ------------------------------------------------------------------

_streams = []


def _stream():
    """The program's one stream: a pass starts when the one before it has ended."""
    if not _streams:
        _streams.append(torch.cuda.Stream())
    return _streams[0]


def _lengths(c):
    """(new rows, positions held before them) of each sequence: part of the case, not of its values."""
    r = random.Random("%d %d %d %s" % (c["seqs"], c["new"], c["held"], c["mix"]))
    got = []
    for s in range(c["seqs"]):
        n = c["new"] if c["mix"] == "same" or s == 0 else 1 if c["mix"] == "mixed" else r.randint((c["new"] + 1) // 2, c["new"])
        held = c["held"] if c["mix"] == "same" or s == 0 else r.randint(c["held"] // 8, c["held"])
        got.append((n, held))
    return got


def _kept(c):
    """How many of its new rows each sequence keeps (-1: it ends): part of the case."""
    r = random.Random("%d %d %d" % (c["seqs"], c["new"], c["kept"]))
    got = [min(r.randint(1, c["kept"]), (n + 1) // 2) for n, _ in _lengths(c)]
    for s in range(c["end"]):
        got[1 + s * (c["seqs"] // c["end"] // 2)] = -1
    got[0] = min(c["kept"], (c["new"] + 1) // 2)
    return got


def _acts(g, rows, heads, hd):
    """q or k rows: N(0, 1) with about one channel in a hundred six times as large, as activations have."""
    x = torch.randn(rows, heads, hd, generator=g, device="cuda")
    return x * torch.where(torch.rand(heads, hd, generator=g, device="cuda") < 0.01, 6.0, 1.0)


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype).cuda()


def _tables(c, g, lens, extra):
    """Pages in random order, enough for all rows: (table of what is held, free pages, number of free ones, pages)."""
    ps = c["page"]
    had = [-(-h // ps) for _, h in lens]
    has = [-(-(n + h) // ps) for n, h in lens]
    n_pages = sum(has) + extra
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).cpu()
    pages = torch.full((len(lens), max(has)), -1, dtype=torch.int32)
    at = 0
    for s, h in enumerate(had):
        pages[s, :h] = order[at:at + h]
        at += h
    free = torch.full((n_pages,), -1, dtype=torch.int32)
    free[:n_pages - at] = order[at:]
    return pages.cuda(), free.cuda(), n_pages - at, n_pages


def _trees(c, g, lens):
    """Every row's parent among its sequence's new rows, level by level: one of the `width` rows or so before it; without
    width a chain."""
    i = torch.cat([torch.arange(n) for n, _ in lens]).cuda()
    back = torch.rand(len(i), generator=g, device="cuda") * 2 * c["width"]
    p = (i - 1 - back.long()).clamp(min=0)
    return torch.where(i == 0, -1, torch.minimum(p, i - 1)).to(torch.int32)


def _ancestors(parent, start, words):
    """(depth, ancestors and itself as bits [row][words]) of rows in flat numbers: start, the first row of each row's tree."""
    row = torch.arange(len(parent), device="cuda")
    i = row - start
    up = torch.where(parent < 0, row, start + parent)
    depth = (parent >= 0).long()
    word = torch.arange(words, device="cuda")
    bits = torch.where(word == (i // 64)[:, None], torch.ones_like(i)[:, None] << (i % 64)[:, None], 0)
    for _ in range((64 * words - 1).bit_length()):  # ancestors 1, 2, 4, ... steps up
        depth = depth + depth[up]
        bits = bits | bits[up]
        up = up[up]
    return depth, bits


def _tensors(c, seed):
    """What a pass is given, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) % (1 << 62))
    t = {}
    if c["op"] == "norm":
        dt = TYPES[c["type"]]
        t["q"], t["k"] = (_acts(g, c["rows"], h, c["hd"]).to(dt) for h in (c["nh"], c["nkv"]))
        t["pos"] = torch.randint(0, c["far"], (c["rows"],), generator=g, device="cuda", dtype=torch.int32)
        t["q_norm"], t["k_norm"] = (1 + 0.3 * torch.randn(c["hd"], generator=g, device="cuda") for _ in range(2))
        return t
    lens, ps = _lengths(c), c["page"]
    n_tok = sum(n for n, _ in lens)
    t["pages"], t["free"], n_free, n_pages = _tables(c, g, lens, 3)
    first = [0]
    for n, _ in lens:
        first.append(first[-1] + n)
    t["held"] = _ints([h for _, h in lens])
    if c["op"] == "plan":
        if c["short"]:  # other sequences took what is missing
            n_free = n_free // 2
        t["n_new"], t["n_free"] = _ints([n for n, _ in lens]), _ints([n_free])
        if c["words"]:
            t["parent"] = _trees(c, g, lens)
        return t
    # the step's tables, as a plan leaves them
    at = sum(-(-h // ps) for _, h in lens)
    pages, top = t["pages"].cpu(), t["free"].cpu()[:n_free].tolist()
    for s, (n, h) in enumerate(lens):
        for j in range(-(-h // ps), -(-(n + h) // ps)):
            pages[s, j] = top.pop()
            at += 1
    t["pages"], t["n_free"] = pages.cuda(), _ints([n_pages - at])
    t["q_start"], t["kv_len"] = _ints(first), _ints([n + h for n, h in lens])
    geo, ct = (c["nkv"], c["hd"]), TYPES[c["cache"]]
    if c["op"] == "keep":
        for x in ("k_pool", "v_pool"):
            t[x] = torch.randn(c["layers"], n_pages, geo[0], ps, geo[1], generator=g, device="cuda", dtype=torch.float32).to(ct)
        r, rows = random.Random(seed), []
        for (n, _), k in zip(lens, _kept(c)):
            # the root, and a path below it behind the tree's first levels
            k = max(k, 1)
            path = [0] + sorted(r.sample(range(k, n), k - 1))
            rows += path + [-1] * (n - len(path))
        t["rows"], t["n_keep"] = _ints(rows), _ints(_kept(c))
        return t
    dt = TYPES[c["type"]]
    seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor([n for n, _ in lens])).cuda()
    start = t["q_start"][seq].long()
    words = -(-max(n for n, _ in lens) // 64)
    if c["width"]:
        depth, t["mask"] = _ancestors(_trees(c, g, lens).long(), start, words)
    else:
        depth = torch.arange(n_tok, device="cuda") - start
    t["pos"] = (t["held"][seq] + depth).to(torch.int32)
    t["q"] = _acts(g, n_tok, c["nh"], c["hd"]).to(dt)
    if c["op"] == "store":
        p = t["held"][seq].long() + torch.arange(n_tok, device="cuda") - start
        t["slot"] = t["pages"][seq, p // ps].long() * ps + p % ps
        t["k"] = _acts(g, n_tok, *geo).to(dt)
        t["v"] = torch.randn(n_tok, *geo, generator=g, device="cuda").to(dt)
        t["q_norm"], t["k_norm"] = (1 + 0.3 * torch.randn(c["hd"], generator=g, device="cuda") for _ in range(2))
        t["k_pool"] = torch.zeros(1, n_pages, c["nkv"], ps, c["hd"], dtype=ct, device="cuda")
        t["v_pool"] = torch.zeros_like(t["k_pool"])
    else:  # one layer's pages, [page][kv head][slot][head_dim]
        t["k_pool"] = _acts(g, n_pages * ps, *geo).to(ct).view(1, n_pages, ps, *geo).transpose(2, 3).contiguous()
        t["v_pool"] = torch.randn(1, n_pages, c["nkv"], ps, c["hd"], generator=g, device="cuda").to(ct)
    return t


class _State:
    """What the program keeps between calls."""


def _out_buffers(c, t):
    """The arrays that the calls fill."""
    if c["op"] == "norm":
        return {"q": torch.empty_like(t["q"]), "k": torch.empty_like(t["k"])}
    if c["op"] in ("store", "tree"):
        return {"q": torch.empty_like(t["q"])}
    n, dev = len(t["held"]), {"device": "cuda", "dtype": torch.int32}
    o = {"kv_len": torch.empty(n, **dev), "n_free": torch.empty(1, **dev)}
    if c["op"] == "plan":
        n_tok = sum(n for n, _ in _lengths(c))
        o.update(q_start=torch.empty(n + 1, **dev), pos=torch.empty(n_tok, **dev), status=torch.empty(1, **dev),
                 slot=torch.empty(n_tok, device="cuda", dtype=torch.int64))
        if c["words"]:
            o["mask"] = torch.empty(n_tok, c["words"], device="cuda", dtype=torch.int64)
    return o


def prepare(case, seed):
    c, s = case, _State()
    s.case, s.t, s.stream = c, _tensors(c, seed), _stream()
    t = s.t
    s.o = o = _out_buffers(c, t)
    s.lens = _lengths(c) if c["op"] != "norm" else None
    p = {k: v.data_ptr() for k, v in t.items()}
    if own:
        from kore_amd import paged, rope
        torch.cuda.synchronize()
        op = c["op"]
        if op == "norm":
            s.rope = rope.Rope(rope.Config(rot_dim=c["rot"], layout=c["layout"], base=BASE))
            s.sets = [rope.Heads(p["q"], o["q"].data_ptr(), c["nh"], c["hd"], norm=p["q_norm"]),
                      rope.Heads(p["k"], o["k"].data_ptr(), c["nkv"], c["hd"], norm=p["k_norm"])]
        elif op == "plan":
            # the tables are of a cache of any geometry
            s.kv = paged.PagedKV(n_layer=1, n_pages=len(t["free"]), page_size=c["page"], n_head=1, n_head_kv=1, head_dim=8, cache_type="f16")
            s.plan = paged.Plan(n_seq=c["seqs"], n_tok=len(o["pos"]), n_new=p["n_new"], kv_held=p["held"], kv_len=o["kv_len"].data_ptr(),
                                pages=p["pages"], pages_stride=t["pages"].shape[1], free_pages=p["free"], n_free=p["n_free"],
                                n_free_out=o["n_free"].data_ptr(), q_start=o["q_start"].data_ptr(), pos=o["pos"].data_ptr(),
                                slot=o["slot"].data_ptr(), status=o["status"].data_ptr(), parent=p.get("parent"),
                                mask=o["mask"].data_ptr() if c["words"] else None, mask_words=c["words"])
        else:
            s.kv = paged.PagedKV(n_layer=c.get("layers", 1), n_pages=t["k_pool"].shape[1], page_size=c["page"], n_head=c["nh"],
                                 n_head_kv=c["nkv"], head_dim=c["hd"], cache_type=c["cache"], k_pool=p["k_pool"], v_pool=p["v_pool"],
                                 rope=rope.Config(rot_dim=c["hd"], layout=c["layout"], base=BASE) if op == "store" else None)
            n_tok = sum(n for n, _ in s.lens)
            if op == "store":
                s.rows = paged.Rows(n_tok=n_tok, pos=p["pos"], slot=p["slot"], q_norm=p["q_norm"], k_norm=p["k_norm"], norm_eps=EPS)
            elif op == "tree":
                s.batch = paged.Batch(n_seq=c["seqs"], n_tok=n_tok, q_start=p["q_start"], kv_len=p["kv_len"], pages=p["pages"],
                                      pages_stride=t["pages"].shape[1], max_q=max(n for n, _ in s.lens))
                s.tree = paged.Tree(mask=p["mask"], mask_words=t["mask"].shape[1], pos=p["pos"])
            else:
                s.keep = paged.Keep(n_seq=c["seqs"], n_tok=n_tok, q_start=p["q_start"], n_keep=p["n_keep"], rows=p["rows"],
                                    kv_len=p["kv_len"], kv_out=o["kv_len"].data_ptr(), pages=p["pages"], pages_stride=t["pages"].shape[1],
                                    free_pages=p["free"], n_free=p["n_free"], n_free_out=o["n_free"].data_ptr())
    torch.cuda.synchronize()
    return s


# ---- the plain forms -----------------------------------------------------------

def _plain_plan(s):
    c, t, ps = s.case, s.t, s.case["page"]
    n, old, n_free = t["n_new"].long(), t["held"].long(), t["n_free"].long()
    n_tok, n_pages, stride = len(s.o["pos"]), len(t["free"]), t["pages"].shape[1]
    new = old + n
    had, has = (old + ps - 1) // ps, (new + ps - 1) // ps
    need = has - had
    bad = (n < 0).any() | (old < 0).any() | (new > stride * ps).any() | (n.sum() > n_tok) | (n_free < 0) | (n_free > n_pages)
    if c["words"]:
        bad = bad | (n > 64 * c["words"]).any()
    missing = (need.sum() - n_free).clamp(min=0)
    status = torch.where(bad, -1, missing)
    ok = status == 0
    n, new, need = torch.where(ok, n, 0), torch.where(ok, new, old), torch.where(ok, need, 0)
    q_start = torch.cat([torch.zeros_like(n[:1]), n.cumsum(0)])
    # the j-th new page of all is the j-th from the top of the free ones
    col = torch.arange(stride, device="cuda")
    j = (need.cumsum(0) - need)[:, None] + col - had[:, None]
    fresh = (col >= had[:, None]) & (col < (had + need)[:, None])
    pages = torch.where(fresh, t["free"][(n_free - 1 - j).clamp(0, n_pages - 1)], t["pages"])
    row = torch.arange(n_tok, device="cuda")
    seq = torch.searchsorted(q_start[1:], row, right=True)
    real = seq < len(n)
    seq = seq.clamp(max=len(n) - 1)
    i = row - q_start[seq]
    at = (old[seq] + i).clamp(min=0)
    page = pages[seq, (at // ps).clamp(max=stride - 1)].long()
    slot = torch.where(real & (page >= 0) & (page < n_pages), page * ps + at % ps, -1)
    depth, o = i, {}
    if c["words"]:
        parent = torch.where(real, t["parent"].long(), -1)
        depth, bits = _ancestors(parent, torch.where(real, q_start[seq], row), c["words"])
        o["mask"] = torch.where(real[:, None], bits, 0)
    pos = torch.where(real, old[seq] + depth, -1)
    t["pages"].copy_(pages)
    o.update(kv_len=new.int(), n_free=(n_free - need.sum()).int(), q_start=q_start.int(), pos=pos.int(), slot=slot, status=status.int())
    for k, v in o.items():
        s.o[k].copy_(v)


def _rotated(c, x, pos, rot, w):
    """The rows x [n][heads][hd] with their heads normalised and turned to the positions pos, in 32 bits."""
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f = torch.exp(i * (-2.0 / rot * math.log(BASE))).float().double()  # (the engine's table is one of floats)
    angle = pos.double()[:, None] * f[None, :]  # far positions need 64 bits
    cs, sn = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    out = x.clone()
    if c["layout"] == "half":
        a, b = slice(0, rot // 2), slice(rot // 2, rot)
    else:
        a, b = slice(0, rot, 2), slice(1, rot, 2)
    out[..., a] = x[..., a] * cs - x[..., b] * sn
    out[..., b] = x[..., a] * sn + x[..., b] * cs
    return out


def _plain_store(s):
    c, t, ps = s.case, s.t, s.case["page"]
    page, at = t["slot"] // ps, t["slot"] % ps
    t["k_pool"][0, page, :, at] = _rotated(c, t["k"], t["pos"], c["hd"], t["k_norm"]).to(t["k_pool"].dtype)
    t["v_pool"][0, page, :, at] = t["v"].to(t["v_pool"].dtype)
    s.o["q"].copy_(_rotated(c, t["q"], t["pos"], c["hd"], t["q_norm"]).to(t["q"].dtype))


def _plain_tree(s):
    c, t, dev = s.case, s.t, "cuda"
    nkv, hd, rep, n_seq = c["nkv"], c["hd"], c["nh"] // c["nkv"], c["seqs"]
    n_q, n_kv = max(n for n, _ in s.lens), max(n + h for n, h in s.lens)
    # the sequences side by side, padded to the longest
    page = t["pages"].clamp(min=0).long()
    k = t["k_pool"][0][page].transpose(1, 2).reshape(n_seq, nkv, -1, hd)[:, :, :n_kv].float()
    v = t["v_pool"][0][page].transpose(1, 2).reshape(n_seq, nkv, -1, hd)[:, :, :n_kv].float()
    i = torch.arange(n_q, device=dev)
    real = i < (t["q_start"][1:] - t["q_start"][:-1])[:, None]
    row = torch.where(real, t["q_start"][:-1, None] + i, 0).long()
    q = t["q"][row].float().view(n_seq, n_q, nkv, rep, hd).permute(0, 2, 3, 1, 4).reshape(n_seq, nkv, rep * n_q, hd)
    # a cached position, within the window; or a new row whose bit is set
    j = torch.arange(n_kv, device=dev)
    held = t["held"][:, None]
    cached = j < held
    new = (j - held).clamp(0, 64 * t["mask"].shape[1] - 1)
    bit = t["mask"][row][torch.arange(n_seq, device=dev)[:, None, None], i[:, None], new[:, None, :] // 64] >> (new % 64)[:, None, :]
    seen = torch.where(cached[:, None, :], j > t["pos"][row][:, :, None] - c["window"] if c["window"] else True, (bit & 1) == 1)
    seen = seen & (j < t["kv_len"][:, None])[:, None, :]
    w = torch.matmul(q, k.transpose(2, 3).contiguous()).view(n_seq, nkv, rep, n_q, n_kv)
    w.mul_(1 / math.sqrt(hd)).masked_fill_(~seen[:, None, None], -math.inf)
    m = w.amax(-1, keepdim=True)
    w.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(n_seq, nkv, rep * n_q, n_kv), v).view(n_seq, nkv, rep, n_q, hd)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(n_seq, n_q, c["nh"], hd)
    s.o["q"].copy_(o[real].to(t["q"].dtype))


def _plain_keep(s):
    c, t, ps = s.case, s.t, s.case["page"]
    start, kv = t["q_start"].long(), t["kv_len"].long()
    n = start[1:] - start[:-1]
    kept = torch.minimum(t["n_keep"].long(), n)
    row = torch.arange(len(t["rows"]), device="cuda")
    seq = torch.searchsorted(start[1:], row, right=True)
    i, src, held = row - start[seq], t["rows"].long(), (kv - n)[seq]
    moves = (i < kept[seq]) & (src >= 0) & (src < n[seq]) & (src != i)
    seq, a, b = seq[moves], (held + src)[moves], (held + i)[moves]
    pa, pb = t["pages"][seq, a // ps].long(), t["pages"][seq, b // ps].long()
    for pool in (t["k_pool"], t["v_pool"]):
        pool[:, pb, :, b % ps] = pool[:, pa, :, a % ps]
    new = torch.where(kept < 0, 0, kv - n + kept)
    # the pages behind the new ends, in the table's order
    col = torch.arange(t["pages"].shape[1], device="cuda")
    back = (col >= ((new + ps - 1) // ps)[:, None]) & (col < ((kv + ps - 1) // ps)[:, None])
    back &= (t["pages"] >= 0) & (t["pages"] < t["k_pool"].shape[1])
    gone = t["pages"][back]
    at = t["n_free"].long() + torch.arange(len(gone), device="cuda")
    t["free"][at] = gone
    s.o["kv_len"].copy_(new.int())
    s.o["n_free"].copy_(t["n_free"] + len(gone))


# ---- one pass ------------------------------------------------------------------

def _outputs(s):
    c, t, o = s.case, s.t, s.o
    if c["op"] == "plan":
        return {**o, "pages": t["pages"]}
    if c["op"] == "store":
        return {"q": o["q"], "k_pool": t["k_pool"], "v_pool": t["v_pool"]}
    if c["op"] == "keep":
        return {**o, "free": t["free"], "k_pool": t["k_pool"], "v_pool": t["v_pool"]}
    return o


def run(state):
    s, c, t = state, state.case, state.t
    op = c["op"]
    if not own:
        with torch.cuda.stream(s.stream):
            if op == "norm":
                for x in ("q", "k"):
                    s.o[x].copy_(_rotated(c, t[x], t["pos"], c["rot"], t[x + "_norm"]).to(t[x].dtype))
            else:
                {"plan": _plain_plan, "store": _plain_store, "tree": _plain_tree, "keep": _plain_keep}[op](s)
        return _outputs(s)
    st = s.stream.cuda_stream
    if op == "plan":
        s.kv.plan_dev(s.plan, stream=st)
    elif op == "norm":
        s.rope.norm_dev(c["type"], c["rows"], c["hd"], s.sets, t["pos"].data_ptr(), eps=EPS, stream=st)
    elif op == "store":
        s.kv.append_rows_dev(0, s.rows, c["type"], t["k"].data_ptr(), t["v"].data_ptr(), q=t["q"].data_ptr(), q_out=s.o["q"].data_ptr(),
                             stream=st)
    elif op == "tree":
        s.kv.attend_tree_dev(0, s.batch, s.tree, c["type"], t["q"].data_ptr(), s.o["q"].data_ptr(), window=c["window"], stream=st)
    else:
        s.kv.keep_dev(s.keep, stream=st)
    return _outputs(s)


# ---- what a pass cannot do without ---------------------------------------------

_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def work(case):
    c, op = case, case["op"]
    if op == "norm":
        heads = c["nh"] + c["nkv"]
        return {"bytes": 2 * c["rows"] * heads * c["hd"] * _SIZE[c["type"]] + 4 * c["rows"] + 8 * c["hd"],
                "flops": c["rows"] * heads * (4 * c["hd"] + 3 * c["rot"])}
    lens, ps = _lengths(c), c["page"]
    n_tok = sum(n for n, _ in lens)
    fresh = sum(-(-(n + h) // ps) - -(-h // ps) for n, h in lens)
    if op == "plan":
        row = 12 + (4 + 8 * c["words"] if c["words"] else 0)
        return {"bytes": 16 * len(lens) + 8 * fresh + row * n_tok + 16, "flops": 0}
    if op == "keep":
        e = 2 * c["layers"] * c["nkv"] * c["hd"] * _SIZE[c["cache"]]
        kept = _kept(c)
        moved = sum(max(0, k - 1) for k in kept)
        gone = sum(-(-(n + h) // ps) - -(-(h + k if k >= 0 else 0) // ps) for (n, h), k in zip(lens, kept))
        return {"bytes": 2 * moved * e + 16 * len(lens) + 8 * gone + 4 * moved, "flops": 0}
    e, ce = _SIZE[c["type"]], _SIZE[c["cache"]]
    if op == "store":
        rows = n_tok * c["nkv"] * c["hd"]
        return {"bytes": 2 * rows * (e + ce) + 2 * n_tok * c["nh"] * c["hd"] * e + 12 * n_tok + 8 * c["hd"],
                "flops": 7 * n_tok * (c["nh"] + c["nkv"]) * c["hd"]}
    w = c["window"] or 1 << 60
    tables = 4 * (2 * len(lens) + 1 + sum(-(-(n + h) // ps) for n, h in lens)) + 8 * n_tok * -(-c["new"] // 64)
    keys = sum(min(h, w) + n for n, h in lens)
    # a row's ancestors: the levels of a tree with some `width` rows each
    pairs = sum(min(h, w) + 1 + i // (c["width"] + 1) for n, h in lens for i in range(n))
    return {"bytes": 2 * keys * c["nkv"] * c["hd"] * ce + 2 * n_tok * c["nh"] * c["hd"] * e + tables,
            "flops": 4 * c["nh"] * c["hd"] * pairs}


# ---- the definition in 64 bits ---------------------------------------------------

def _exact_rotated(c, x, positions, rot, w):
    """Each head over its root mean square, each pair as a complex number, turned by its angle."""
    x = x.double()
    x = x / ((x.square().sum(-1, keepdim=True) / c["hd"] + EPS).sqrt()) * w.double()
    freq = torch.tensor([BASE ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float32).double().cuda()
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), positions.double()[:, None] * freq)[:, None]
    if c["layout"] == "half":
        z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * turn
        y = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) * turn
        y = torch.view_as_real(z).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _exact_plan(c, t):
    """Request by request on the host."""
    ps, words = c["page"], c["words"]
    pages, free = t["pages"].cpu().tolist(), t["free"].cpu().tolist()
    n_free, n_pages, stride = int(t["n_free"]), len(free), len(pages[0])
    lens = list(zip(t["n_new"].cpu().tolist(), t["held"].cpu().tolist()))
    n_tok = sum(n for n, _ in _lengths(c))
    parent = t["parent"].cpu().tolist() if words else None
    need = sum((h + n + ps - 1) // ps - (h + ps - 1) // ps for n, h in lens)
    status = max(0, need - n_free)
    if any(n < 0 or h < 0 or n + h > stride * ps or (words and n > 64 * words) for n, h in lens):
        status = -1
    o = {"kv_len": [h for _, h in lens], "n_free": [n_free], "q_start": [0] * (len(lens) + 1), "pos": [-1] * n_tok, "status": [status],
         "slot": [-1] * n_tok}
    mask = [[0] * max(words, 1) for _ in range(n_tok)]
    row = 0
    for s, (n, h) in enumerate(lens if status == 0 else []):
        for j in range(-(-h // ps), -(-(h + n) // ps)):
            n_free -= 1
            pages[s][j] = free[n_free]
        depth, seen = [], []
        for i in range(n):
            up = parent[row + i] if words else i - 1
            depth.append(depth[up] + 1 if up >= 0 else 0)
            seen.append((seen[up] if up >= 0 else 0) | 1 << i if words else 0)
            o["pos"][row + i] = h + depth[i]
            o["slot"][row + i] = pages[s][(h + i) // ps] * ps + (h + i) % ps
            for x in range(words):
                bits = seen[i] >> (64 * x) & (1 << 64) - 1
                mask[row + i][x] = bits - (1 << 64) if bits >> 63 else bits
        row += n
        o["q_start"][s + 1], o["kv_len"][s] = row, h + n
    o["n_free"] = [n_free]
    o = {k: _ints(v, torch.int64 if k == "slot" else torch.int32) for k, v in o.items()}
    if words:
        o["mask"] = _ints(mask, torch.int64)
    return {**o, "pages": _ints(pages)}


def _exact_keep(c, t):
    """Sequence by sequence, row by row on the host's lists."""
    ps = c["page"]
    k_pool, v_pool = t["k_pool"].double(), t["v_pool"].double()
    before = k_pool.clone(), v_pool.clone()
    start, kv, pages = t["q_start"].cpu().tolist(), t["kv_len"].cpu().tolist(), t["pages"].cpu().tolist()
    rows, keep, free, n_free = t["rows"].cpu().tolist(), t["n_keep"].cpu().tolist(), t["free"].cpu().tolist(), int(t["n_free"])
    ends = []
    for s, k in enumerate(keep):
        n = start[s + 1] - start[s]
        h = kv[s] - n
        for i in range(min(max(k, 0), n)):
            a, b = h + rows[start[s] + i], h + i
            for new, old in zip((k_pool, v_pool), before):
                new[:, pages[s][b // ps], :, b % ps] = old[:, pages[s][a // ps], :, a % ps]
        ends.append(h + min(k, n) if k >= 0 else 0)
        for j in range(-(-ends[s] // ps), -(-kv[s] // ps)):
            free[n_free] = pages[s][j]
            n_free += 1
    return {"kv_len": _ints(ends), "n_free": _ints([n_free]), "free": _ints(free), "k_pool": k_pool, "v_pool": v_pool}


def exact(case, seed):
    c, t = case, _tensors(case, seed)
    op = c["op"]
    if op == "norm":
        return {x: _exact_rotated(c, t[x], t["pos"], c["rot"], t[x + "_norm"]) for x in ("q", "k")}
    if op == "plan":
        return _exact_plan(c, t)
    if op == "keep":
        return _exact_keep(c, t)
    ps, lens, rep = c["page"], _lengths(c), c["nh"] // c["nkv"]
    if op == "store":
        k_pool, v_pool = t["k_pool"].double(), t["v_pool"].double()
        page = torch.div(t["slot"], ps, rounding_mode="floor")
        k_pool[0, page, :, t["slot"] - page * ps] = _exact_rotated(c, t["k"], t["pos"], c["hd"], t["k_norm"])
        v_pool[0, page, :, t["slot"] - page * ps] = t["v"].double()
        return {"q": _exact_rotated(c, t["q"], t["pos"], c["hd"], t["q_norm"]), "k_pool": k_pool, "v_pool": v_pool}
    out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    mask, at = t["mask"].cpu().tolist(), 0
    for s, (n, h) in enumerate(lens):
        j = torch.arange(n + h, device="cuda")
        where = t["pages"][s].long()[j // ps]
        hidden = torch.zeros(n, n + h, dtype=torch.bool)
        for i in range(n):
            bits = sum((w & (1 << 64) - 1) << (64 * x) for x, w in enumerate(mask[at + i]))
            hidden[i, h:] = torch.tensor([not bits >> x & 1 for x in range(n)])
            if c["window"]:
                hidden[i, :max(0, min(h, int(t["pos"][at + i]) - c["window"] + 1))] = True
        hidden = hidden.cuda()
        for kh in range(c["nkv"]):
            k, v = (t[x][0, where, kh, j % ps].double() for x in ("k_pool", "v_pool"))
            for x in range(kh * rep, (kh + 1) * rep):
                scores = t["q"][at:at + n, x].double() @ k.t().contiguous() / math.sqrt(c["hd"])
                out[at:at + n, x] = torch.softmax(scores.masked_fill(hidden, -math.inf), -1) @ v
        at += n
    return {"q": out}
