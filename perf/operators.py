"""Positions, the paged KV cache and the attention that reads it, as cases that can be timed and compared.

Three operators of a serving step: rotary positions (both layouts, part of the head, scaled), the append of new K and V
rows to a paged cache with the rotation on the way, and the attention of each sequence's new rows over its pages.  `run`
computes them in plain torch operations or, with `own` set, through the library.  Geometries are those of the benchmark
and the tests (the Qwen2.5 widths, and one outside that family); values are synthetic.
"""
from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BASE = 1e6

# (n_head, n_head_kv, head_dim) of the 0.5B, 1.5B, 3B and 7B models, and one that is none of them
FAMILY = [(14, 2, 64), (12, 2, 128), (16, 2, 128), (28, 4, 128)]
OTHER = (33, 3, 96)


def _geo(g):
    return {"nh": g[0], "nkv": g[1], "hd": g[2]}


def listed():
    half = {"layout": "half", "scaling": "none", "factor": 1.0}
    yarn = {"layout": "half", "scaling": "yarn", "factor": 4.0}
    return [
        # one token's q and k heads: all latency
        {"name": "rope_token", "op": "rope", "rows": 1, "heads": 32, "hd": 128, "rot": 128, "type": "f32", "far": 4096, **half},
        # the ragged end of a long prompt, past the trained context
        {"name": "rope_far_chunk", "op": "rope", "rows": 333, "heads": 18, "hd": 128, "rot": 128, "type": "f32", "far": 131072, **yarn},
        # a large batch of rows of a model that rotates two thirds of a head, neighbours as pairs
        {"name": "rope_part_interleaved", "op": "rope", "rows": 4096, "heads": 36, "hd": 96, "rot": 64, "type": "bf16", "far": 16384,
         "layout": "interleaved", "scaling": "linear", "factor": 4.0},
        # one token of each of 16 running sequences into a half-precision cache
        {"name": "append_step", "op": "append", **_geo(FAMILY[3]), "seqs": 16, "new": 1, "kv": 4096, "mix": "ragged", "page": 16,
         "type": "f32", "cache": "f16", **half},
        # prompts of uneven length at once
        {"name": "append_prompts", "op": "append", **_geo(FAMILY[3]), "seqs": 3, "new": 777, "kv": 2500, "mix": "ragged", "page": 64,
         "type": "f32", "cache": "bf16", **yarn},
        # one token of one conversation on the smallest model: all latency
        {"name": "attend_token", "op": "attend", **_geo(FAMILY[0]), "seqs": 1, "new": 1, "kv": 512, "mix": "same", "page": 16, "window": 0,
         "type": "f32", "cache": "f32"},
        # a decode step of 32 running sequences
        {"name": "attend_step", "op": "attend", **_geo(FAMILY[3]), "seqs": 32, "new": 1, "kv": 8192, "mix": "ragged", "page": 16,
         "window": 0, "type": "f32", "cache": "f16"},
        # one token over a very long context
        {"name": "attend_long_token", "op": "attend", **_geo(FAMILY[2]), "seqs": 1, "new": 1, "kv": 131072, "mix": "same", "page": 256,
         "window": 0, "type": "bf16", "cache": "bf16"},
        # a whole prompt
        {"name": "attend_prompt", "op": "attend", **_geo(FAMILY[3]), "seqs": 1, "new": 2048, "kv": 2048, "mix": "same", "page": 64,
         "window": 0, "type": "f16", "cache": "f16"},
        # a chunk of a long prompt behind what is cached of it
        {"name": "attend_long_chunk", "op": "attend", **_geo(FAMILY[3]), "seqs": 1, "new": 512, "kv": 32749, "mix": "same", "page": 32,
         "window": 0, "type": "f32", "cache": "bf16"},
        # a chunk of one prompt beside the tokens of eight running sequences, nothing rounded
        {"name": "attend_mixed", "op": "attend", **_geo(FAMILY[1]), "seqs": 9, "new": 700, "kv": 3000, "mix": "mixed", "page": 16,
         "window": 0, "type": "f32", "cache": "f32"},
        # uneven chunks of a geometry outside the family, each row seeing a window
        {"name": "attend_window", "op": "attend", **_geo(OTHER), "seqs": 4, "new": 333, "kv": 5001, "mix": "ragged", "page": 32,
         "window": 1024, "type": "f16", "cache": "f16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_positions(rng):
    return {"layout": rng.choice(["half", "interleaved"]),
            **rng.choice([{"scaling": "none", "factor": 1.0}, {"scaling": "linear", "factor": 2.5}, {"scaling": "yarn", "factor": 4.0}])}


def _draw_geo(rng):
    if rng.random() < 0.35:
        nkv = rng.randint(1, 6)
        return nkv * rng.randint(1, 10), nkv, 8 * rng.randint(4, 20)
    return rng.choice(FAMILY)


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend", "attend"])
    act, cache = rng.choice([("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
    if op == "rope":
        hd = 8 * rng.randint(4, 16)
        rot = hd if rng.random() < 0.6 else 2 * rng.randint(4, hd // 2)
        return {"op": op, "rows": _log_int(rng, 1, 4096), "heads": rng.randint(1, 36), "hd": hd, "rot": rot,
                "type": rng.choice(sorted(TYPES)), "far": _log_int(rng, 4096, 1000000), **_draw_positions(rng)}
    nh, nkv, hd = _draw_geo(rng)
    c = {"op": op, "nh": nh, "nkv": nkv, "hd": hd, "page": rng.choice([16, 32, 64, 128, 256]), "type": act, "cache": cache,
         "mix": rng.choice(["same", "ragged", "ragged", "mixed"])}
    if op == "append":
        c["seqs"], c["new"] = _log_int(rng, 1, 32), rng.choice([1, 1, _log_int(rng, 2, 700)])
        while c["seqs"] * c["new"] > 2331:
            c["seqs"] = max(1, c["seqs"] // 2)
        c["kv"] = c["new"] + _log_int(rng, 1, 2500)
        return {**c, **_draw_positions(rng)}
    if rng.random() < 0.5:  # a decode step
        c["seqs"], c["new"] = _log_int(rng, 1, 32), 1
        row = 2 * nkv * hd * _SIZE[cache]  # bytes of one position
        c["kv"] = _log_int(rng, 1, min(131072, 250_000_000 // row) // c["seqs"])
    else:  # chunks
        c["seqs"], c["new"] = _log_int(rng, 1, 6), _log_int(rng, 2, 1024)
        c["kv"] = c["new"] + rng.choice([0, _log_int(rng, 1, 16000)])
        while c["seqs"] * c["new"] * c["kv"] > 4_000_000:
            c["seqs"] = max(1, c["seqs"] - 1)
            c["kv"] = c["new"] + (c["kv"] - c["new"]) // 2
            c["new"] = max(2, c["new"] * 3 // 4) if c["seqs"] == 1 else c["new"]
    return {**c, "window": 0 if rng.random() < 0.75 else _log_int(rng, 64, 2048)}


# ---- inputs ------------------------------------------------------------------

_streams = []


def _stream():
    """The program's one stream: a pass starts when the one before it has ended."""
    if not _streams:
        _streams.append(torch.cuda.Stream())
    return _streams[0]


def _lengths(c):
    """(new rows, rows in the cache with them) of each sequence: part of the case, not of its values."""
    r = random.Random("%d %d %d %s" % (c["seqs"], c["new"], c["kv"], c["mix"]))
    got = []
    for s in range(c["seqs"]):
        n = c["new"] if c["mix"] == "same" or s == 0 else 1 if c["mix"] == "mixed" else r.randint((c["new"] + 1) // 2, c["new"])
        kv = c["kv"] if c["mix"] == "same" or s == 0 else r.randint(max(n, c["kv"] // 8), max(n, c["kv"]))
        got.append((n, kv))
    return got


def _acts(g, rows, heads, hd):
    """q or k rows: N(0, 1) with about one channel in a hundred six times as large, as activations have."""
    x = torch.randn(rows, heads, hd, generator=g, device="cuda")
    return x * torch.where(torch.rand(heads, hd, generator=g, device="cuda") < 0.01, 6.0, 1.0)


def _tensors(c, seed):
    """What a pass is given, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) % (1 << 62))
    dt = TYPES[c["type"]]
    t = {}
    if c["op"] == "rope":
        t["x"] = _acts(g, c["rows"], c["heads"], c["hd"]).to(dt)
        t["pos"] = torch.randint(0, c["far"], (c["rows"],), generator=g, device="cuda", dtype=torch.int32)
        return t
    nh, nkv, hd, ps, ct = c["nh"], c["nkv"], c["hd"], c["page"], TYPES[c["cache"]]
    lens = _lengths(c)
    n_tok = sum(n for n, _ in lens)
    held = [-(-kv // ps) for _, kv in lens]
    n_pages = sum(held) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).cpu()
    pages = torch.full((len(lens), max(held)), -1, dtype=torch.int32)
    at = 0
    for s, h in enumerate(held):
        pages[s, :h] = order[at:at + h]
        at += h
    t["pages"] = pages.cuda()
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    t["q_start"] = torch.tensor(starts, dtype=torch.int32).cuda()
    t["kv_len"] = torch.tensor([kv for _, kv in lens], dtype=torch.int32).cuda()
    t["q"] = _acts(g, n_tok, nh, hd).to(dt)
    if c["op"] == "append":
        t["k"] = _acts(g, n_tok, nkv, hd).to(dt)
        t["v"] = torch.randn(n_tok, nkv, hd, generator=g, device="cuda").to(dt)
        t["k_pool"] = torch.zeros(1, n_pages, nkv, ps, hd, dtype=ct, device="cuda")
        t["v_pool"] = torch.zeros_like(t["k_pool"])
    else:  # one layer's pages, [page][kv head][slot][head_dim]
        t["k_pool"] = _acts(g, n_pages * ps, nkv, hd).to(ct).view(1, n_pages, ps, nkv, hd).transpose(2, 3).contiguous()
        t["v_pool"] = torch.randn(1, n_pages, nkv, ps, hd, generator=g, device="cuda").to(ct)
    return t


class _State:
    """What the program keeps between calls."""


def _config(c, rot):
    from kore_amd import rope
    return rope.Config(rot_dim=rot, layout=c["layout"], base=BASE, scaling=c["scaling"], factor=c["factor"], orig_ctx=32768)


def prepare(case, seed):
    c, s = case, _State()
    s.case, s.t, s.stream = c, _tensors(c, seed), _stream()
    t = s.t
    if c["op"] == "rope":
        s.out = torch.empty_like(t["x"])
    else:
        s.lens = _lengths(c)
        s.rows = t["q"].shape[0]
        s.out = torch.empty_like(t["q"])
    if own:
        from kore_amd import paged, rope
        torch.cuda.synchronize()
        if c["op"] == "rope":
            s.rope = rope.Rope(_config(c, c["rot"]))
        else:
            s.kv = paged.PagedKV(n_layer=1, n_pages=t["k_pool"].shape[1], page_size=c["page"], n_head=c["nh"], n_head_kv=c["nkv"],
                                 head_dim=c["hd"], cache_type=c["cache"], k_pool=t["k_pool"].data_ptr(), v_pool=t["v_pool"].data_ptr(),
                                 rope=_config(c, c["hd"]) if c["op"] == "append" else None)
            s.batch = paged.Batch(n_seq=c["seqs"], n_tok=s.rows, q_start=t["q_start"].data_ptr(), kv_len=t["kv_len"].data_ptr(),
                                  pages=t["pages"].data_ptr(), pages_stride=t["pages"].shape[1], max_q=max(n for n, _ in s.lens))
    torch.cuda.synchronize()
    return s


# ---- the plain forms -----------------------------------------------------------

def _frequencies(c, rot):
    """The angle of each pair per position: base^(-2 i / rot), scaled, rounded to 32 bits (the engine's table), and the factor
    of the rotated pair."""
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f = torch.exp(i * (-2.0 / rot * math.log(BASE)))
    size = 1.0
    if c["scaling"] == "linear":
        f = f / c["factor"]
    elif c["scaling"] == "yarn":
        turn = lambda b: rot * math.log(32768 / (b * 2 * math.pi)) / (2 * math.log(BASE))  # noqa: E731
        low, high = max(math.floor(turn(32.0)), 0), min(math.ceil(turn(1.0)), rot - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / c["factor"] * ramp + f * (1 - ramp)
        size = 0.1 * math.log(c["factor"]) + 1.0
    return f.float().double(), size


def _rotated(c, x, pos, rot):
    """The rows x [n][heads][hd] at the positions pos, in 32 bits."""
    f, size = _frequencies(c, rot)
    angle = pos.double()[:, None] * f[None, :]  # far positions need 64 bits
    cs, sn = (size * angle.cos()).float()[:, None, :], (size * angle.sin()).float()[:, None, :]
    x = x.float()
    out = x.clone()
    if c["layout"] == "half":
        a, b = slice(0, rot // 2), slice(rot // 2, rot)
    else:
        a, b = slice(0, rot, 2), slice(1, rot, 2)
    out[..., a] = x[..., a] * cs - x[..., b] * sn
    out[..., b] = x[..., a] * sn + x[..., b] * cs
    return out


def _plain_append(s):
    c, t, ps = s.case, s.t, s.case["page"]
    row = torch.arange(s.rows, device="cuda")
    seq = (row[:, None] >= t["q_start"][None, 1:]).sum(1)
    pos = t["kv_len"][seq] - (t["q_start"][seq + 1] - row)
    page = t["pages"][seq, pos // ps].long()
    t["k_pool"][0, page, :, pos % ps] = _rotated(c, t["k"], pos, c["hd"]).to(t["k_pool"].dtype)
    t["v_pool"][0, page, :, pos % ps] = t["v"].to(t["v_pool"].dtype)
    s.out.copy_(_rotated(c, t["q"], pos, c["hd"]).to(t["q"].dtype))
    return {"q": s.out, "k_pool": t["k_pool"], "v_pool": t["v_pool"]}


def _plain_attend(s):
    c, t, ps, dev = s.case, s.t, s.case["page"], "cuda"
    nkv, hd, rep, n_seq = c["nkv"], c["hd"], c["nh"] // c["nkv"], c["seqs"]
    n_q, n_kv = max(n for n, _ in s.lens), max(kv for _, kv in s.lens)
    n_new = t["q_start"][1:] - t["q_start"][:-1]
    # the sequences side by side, padded to the longest
    page = t["pages"].clamp(min=0).long()
    k = t["k_pool"][0][page].transpose(1, 2).reshape(n_seq, nkv, -1, hd)[:, :, :n_kv].float()
    v = t["v_pool"][0][page].transpose(1, 2).reshape(n_seq, nkv, -1, hd)[:, :, :n_kv].float()
    i = torch.arange(n_q, device=dev)
    row = (t["q_start"][:-1, None] + i).clamp(max=s.rows - 1).long()
    q = t["q"][row].float().view(n_seq, n_q, nkv, rep, hd).permute(0, 2, 3, 1, 4).reshape(n_seq, nkv, rep * n_q, hd)
    j = torch.arange(n_kv, device=dev)
    pos = (t["kv_len"] - n_new)[:, None] + i
    seen = (j <= pos[:, :, None]) & (j < t["kv_len"][:, None, None])
    if c["window"]:
        seen &= j > pos[:, :, None] - c["window"]
    w = torch.matmul(q, k.transpose(2, 3).contiguous()).view(n_seq, nkv, rep, n_q, n_kv)
    w.mul_(1 / math.sqrt(hd)).masked_fill_(~seen[:, None, None], -math.inf)
    m = w.amax(-1, keepdim=True)
    w.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(n_seq, nkv, rep * n_q, n_kv), v).view(n_seq, nkv, rep, n_q, hd)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(n_seq, n_q, c["nh"], hd)
    real = i < n_new[:, None]
    s.out.copy_(o[real].to(t["q"].dtype))
    return s.out


# ---- one pass ------------------------------------------------------------------

def run(state):
    s, c, t = state, state.case, state.t
    if not own:
        with torch.cuda.stream(s.stream):
            if c["op"] == "rope":
                s.out.copy_(_rotated(c, t["x"], t["pos"], c["rot"]).to(t["x"].dtype))
                return s.out
            return _plain_append(s) if c["op"] == "append" else _plain_attend(s)
    st = s.stream.cuda_stream
    if c["op"] == "rope":
        s.rope.apply_dev(c["type"], c["rows"], c["heads"], c["hd"], t["x"].data_ptr(), t["pos"].data_ptr(), s.out.data_ptr(), stream=st)
        return s.out
    if c["op"] == "append":
        s.kv.append_dev(0, s.batch, c["type"], t["k"].data_ptr(), t["v"].data_ptr(), q=t["q"].data_ptr(), q_out=s.out.data_ptr(), stream=st)
        return {"q": s.out, "k_pool": t["k_pool"], "v_pool": t["v_pool"]}
    s.kv.attend_dev(0, s.batch, c["type"], t["q"].data_ptr(), s.out.data_ptr(), window=c["window"], stream=st)
    return s.out


# ---- what a pass cannot do without ---------------------------------------------

_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def work(case):
    c, e = case, _SIZE[case["type"]]
    if c["op"] == "rope":
        n = c["rows"] * c["heads"] * c["hd"]
        return {"bytes": 2 * n * e + 4 * c["rows"], "flops": 6 * c["rows"] * c["heads"] * (c["rot"] // 2)}
    lens, ce = _lengths(c), _SIZE[c["cache"]]
    n_tok = sum(n for n, _ in lens)
    tables = 4 * (2 * len(lens) + 1 + sum(-(-kv // c["page"]) for _, kv in lens))
    if c["op"] == "append":
        rows = n_tok * c["nkv"] * c["hd"]
        return {"bytes": 2 * rows * (e + ce) + 2 * n_tok * c["nh"] * c["hd"] * e + tables,
                "flops": 3 * n_tok * (c["nh"] + c["nkv"]) * c["hd"]}
    w = c["window"] or 1 << 60
    keys = sum(min(kv, n - 1 + w) for n, kv in lens)
    pairs = sum(min(p + 1, w) for n, kv in lens for p in range(kv - n, kv))
    return {"bytes": 2 * keys * c["nkv"] * c["hd"] * ce + 2 * n_tok * c["nh"] * c["hd"] * e + tables,
            "flops": 4 * c["nh"] * c["hd"] * pairs}


# ---- the definition in 64 bits ---------------------------------------------------

def _exact_rope(c, x, positions, rot):
    """Each pair as a complex number, turned by its angle."""
    freq, size = [], 1.0
    for i in range(rot // 2):
        f = BASE ** (-2.0 * i / rot)
        if c["scaling"] == "linear":
            f /= c["factor"]
        if c["scaling"] == "yarn":
            edge = [rot * math.log(32768 / (2 * math.pi * b)) / (2 * math.log(BASE)) for b in (32.0, 1.0)]
            lo, hi = max(0, math.floor(edge[0])), min(rot - 1, math.ceil(edge[1]))
            g = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f, size = (1 - g) * f + g * f / c["factor"], 1 + 0.1 * math.log(c["factor"])
        freq.append(f)
    freq = torch.tensor(freq, dtype=torch.float32).double().cuda()  # the table is one of floats
    turn = torch.polar(torch.full((1,), size, dtype=torch.float64, device="cuda"), positions.double()[:, None] * freq)[:, None]
    x = x.double()
    if c["layout"] == "half":
        z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * turn
        y = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) * turn
        y = torch.view_as_real(z).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def exact(case, seed):
    c, t = case, _tensors(case, seed)
    if c["op"] == "rope":
        return _exact_rope(c, t["x"], t["pos"], c["rot"])
    ps, lens, rep = c["page"], _lengths(c), c["nh"] // c["nkv"]
    if c["op"] == "append":
        k_pool, v_pool, q = t["k_pool"].double(), t["v_pool"].double(), t["q"].double()
        at = 0
        for s, (n, kv) in enumerate(lens):
            p = torch.arange(kv - n, kv, device="cuda")
            where = t["pages"][s].long()[p // ps]
            k_pool[0, where, :, p % ps] = _exact_rope(c, t["k"][at:at + n], p, c["hd"])
            v_pool[0, where, :, p % ps] = t["v"][at:at + n].double()
            q[at:at + n] = _exact_rope(c, t["q"][at:at + n], p, c["hd"])
            at += n
        return {"q": q, "k_pool": k_pool, "v_pool": v_pool}
    out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for s, (n, kv) in enumerate(lens):
        j = torch.arange(kv, device="cuda")
        where = t["pages"][s].long()[j // ps]
        p = torch.arange(kv - n, kv, device="cuda")[:, None]
        hidden = (j > p) | (j <= p - c["window"]) if c["window"] else j > p
        for h in range(c["nh"]):
            k, v = (t[x][0, where, h // rep, j % ps].double() for x in ("k_pool", "v_pool"))
            scores = t["q"][at:at + n, h].double() @ k.t().contiguous() / math.sqrt(c["hd"])
            out[at:at + n, h] = torch.softmax(scores.masked_fill(hidden, -math.inf), -1) @ v
        at += n
    return out
