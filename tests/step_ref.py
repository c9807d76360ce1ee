"""Plain implementations of the tables of a step of drafted tokens, of what is kept of it, and of heads that are normalised and
turned, for their tests."""
import math

import numpy as np
import torch

from tests.paged_ref import UNIT, rope_rows


def plan(n_new, held, pages, free, n_free, n_tok, ps, n_pages, parent=None, words=0):
    """The outputs of kore_paged_plan_dev, request by request; pages is a copy."""
    pages = [list(r) for r in pages]
    stride = len(pages[0]) if pages else 1
    need = [(h + n + ps - 1) // ps - (h + ps - 1) // ps for n, h in zip(n_new, held)]
    status = max(0, sum(need) - n_free)
    if (any(n < 0 or h < 0 or n + h > stride * ps or (words and n > 64 * words) for n, h in zip(n_new, held))
            or sum(n_new) > n_tok or not 0 <= n_free <= n_pages):
        status = -1
    o = {"kv_len": list(held), "q_start": [0] * (len(held) + 1), "pos": [-1] * n_tok, "slot": [-1] * n_tok, "status": [status]}
    mask = np.zeros((n_tok, words), np.uint64)
    row = 0
    for s, (n, h) in enumerate(zip(n_new, held) if status == 0 else []):
        for j in range((h + ps - 1) // ps, (h + n + ps - 1) // ps):
            n_free -= 1
            pages[s][j] = int(free[n_free])
        depth, seen = [], []
        for i in range(n):
            up = int(parent[row + i]) if words else i - 1
            up = up if 0 <= up < i else -1
            depth.append(depth[up] + 1 if up >= 0 else 0)
            seen.append((seen[up] if words and up >= 0 else 0) | 1 << i)
            o["pos"][row + i] = h + depth[i]
            page = pages[s][(h + i) // ps]
            o["slot"][row + i] = page * ps + (h + i) % ps if 0 <= page < n_pages else -1
            for w in range(words):
                mask[row + i, w] = seen[i] >> (64 * w) & (1 << 64) - 1
        row += n
        o["q_start"][s + 1], o["kv_len"][s] = row, h + n
    o["n_free"] = [n_free]
    return {**{k: np.asarray(v, np.int64) for k, v in o.items()}, "pages": np.asarray(pages, np.int64).reshape(-1, stride), "mask": mask}


def keep(pools, starts, n_keep, rows, kv_len, pages, free, n_free, ps):
    """The outputs of kore_paged_keep_dev: pools (torch [layer][page][head][slot][hd]) and free in place."""
    ends, n_pages = [], pools[0].shape[1]
    for s, k in enumerate(n_keep):
        n = starts[s + 1] - starts[s]
        h = kv_len[s] - n

        def place(p):
            page = pages[s][p // ps] if 0 <= p < len(pages[s]) * ps else -1
            return (page, p % ps) if 0 <= page < n_pages else None

        k = min(k, n)
        for pool in pools:
            moved = []
            for i in range(max(k, 0)):
                r = rows[starts[s] + i] if rows is not None else i
                if 0 <= r < n and r != i and place(h + r) and place(h + i):
                    a, b = place(h + r), place(h + i)
                    moved.append((b, pool[:, a[0], :, a[1]].clone()))
            for b, x in moved:
                pool[:, b[0], :, b[1]] = x
        ends.append(max(0, h + k) if k >= 0 else 0)
        for j in range(-(-ends[s] // ps), min(-(-kv_len[s] // ps), len(pages[s]))):
            if 0 <= pages[s][j] < n_pages and n_free < n_pages:
                free[n_free] = pages[s][j]
                n_free += 1
    return ends, n_free


def tree(rng, n, width):
    """Parents of n rows: each one of the `width` or so before it; the first, and now and then another, is a root."""
    return [-1 if i == 0 or rng.random() < 0.02 else max(0, i - 1 - int(rng.integers(0, 2 * width + 1))) for i in range(n)]


def heads(x, pos, freqs, m, layout, w, eps):
    """x [n][heads][hd] normalised (w None: not) and turned in 64 bits: (y, the sum of the magnitudes of each one's products)."""
    x = np.asarray(x, np.float64)
    if w is not None:
        x = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * np.asarray(w, np.float64)
    return rope_rows(x, pos, freqs, m, layout)


def heads_bound(y, size, dtype, normed):
    """As rope_bound, four half steps of fp32; and of a normalised head three more, of 1 / root and of the two products."""
    b = (7 if normed else 4) * UNIT["f32"] * size * (1 + 2.0 ** -20)
    return b if dtype == "f32" else b + UNIT[dtype] * (np.abs(y) + b) + (2.0 ** -25 if dtype == "f16" else 0.0)


def tree_exact(c, mask, pos=None, layer=0, window=0, scale=0.0):
    """Case.exact for rows that attend what their sequence held, in the window behind pos, and the new rows of their mask
    ([n_tok][words] uint64); the bound is derived there."""
    out = np.full((c.n_tok, c.nh, c.hd), np.nan)
    bound = np.full_like(out, np.nan)
    q, kp, vp = (t.detach().to(torch.float64).numpy() for t in (c.q, c.k_pool[layer], c.v_pool[layer]))
    scale = scale or 1 / math.sqrt(c.hd)
    rep = c.nh // c.nkv
    for s, (n, _) in enumerate(c.lens):
        kv = int(c.kv_len[s])
        h = kv - n
        for i in range(n):
            row = int(c.starts[s]) + i
            bits = sum(int(w) << (64 * x) for x, w in enumerate(mask[row]))
            lo = 0
            if window:
                lo = max(0, min(max(int(pos[row]), h), kv - 1) - window + 1)
            p = np.asarray(list(range(lo, h)) + [h + j for j in range(n) if bits >> j & 1 and h + j >= 0], np.int64)
            p = p[p < c.stride * c.ps]
            page = c.pages[s, p // c.ps]
            p = p[(page >= 0) & (page < c.n_pages)]
            if len(p) == 0:
                out[row], bound[row] = 0, 0
                continue
            page = c.pages[s, p // c.ps]
            for hd in range(c.nh):
                K, V = kp[page, hd // rep, p % c.ps], vp[page, hd // rep, p % c.ps]
                with np.errstate(invalid="ignore", over="ignore"):
                    sc = K @ q[row, hd] * scale
                    w = np.exp(sc - sc.max())
                    w /= w.sum()
                    out[row, hd] = w @ V
                    S = scale * float((np.abs(K) @ np.abs(q[row, hd])).max())
                    u = UNIT[c.dtype] if c.dtype != "f32" else 2.0 ** -21
                    e = 2 * S * ((c.hd + 8) * UNIT["f32"] + 2.0 ** -21) + u + (len(p) / 8 + 16) * UNIT["f32"]
                    bound[row, hd] = e * (w @ np.abs(V)) + UNIT[c.dtype] * np.abs(out[row, hd]) + (2.0 ** -24 if c.dtype == "f16" else 0.0)
    return out, bound
