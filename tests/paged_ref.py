"""Inputs, plain implementations in 64 bits and error bounds for the tests of the rotary positions and the paged cache."""
import math

import numpy as np
import torch

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# half a step relative to the value
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]


def rope_freqs(rot, base=1e6, scaling="none", factor=1.0, orig_ctx=0, fast=32.0, slow=1.0, factors=None):
    """The float frequencies of include/kore_rope.h and the magnitude."""
    out, m = [], 1.0
    base, factor = float(np.float32(base)), float(np.float32(factor))
    for i in range(rot // 2):
        f = base ** (-2.0 * i / rot)
        if scaling == "linear":
            f /= factor
        if scaling == "yarn":
            corr = lambda b: rot * math.log(orig_ctx / (b * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            lo, hi = max(math.floor(corr(fast)), 0), min(math.ceil(corr(slow)), rot - 1)
            g = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f, m = f / factor * g + f * (1 - g), 0.1 * math.log(factor) + 1.0
        if factors is not None:
            f /= float(np.float32(factors[i]))
        out.append(f)
    return np.asarray(out, np.float32), m


def rope_rows(x, pos, freqs, m, layout, transpose=False):
    """x [n][heads][hd] (any float) turned in 64 bits: (y, the sum |x0 c| + |x1 s| of each element)."""
    x = np.asarray(x, np.float64)
    half = len(freqs)
    rot = 2 * half
    ang = np.asarray(pos, np.float64)[:, None] * freqs.astype(np.float64)
    c, s = m * np.cos(ang)[:, None], m * np.sin(ang)[:, None]
    if transpose:
        s = -s
    a, b = (slice(0, half), slice(half, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    y, size = x.copy(), np.abs(x)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    size[..., a] = np.abs(x[..., a] * c) + np.abs(x[..., b] * s)
    size[..., b] = np.abs(x[..., a] * s) + np.abs(x[..., b] * c)
    return y, size


def rope_bound(y, size, dtype):
    """c, s, each product and the sum are rounded to fp32 (three halves of a step of each product, one of the sum), then
    the result to dtype (an fp16 result under 2^-14: half of its smallest step, 2^-25)."""
    b = 4 * UNIT["f32"] * size * (1 + 2.0 ** -20)
    return b if dtype == "f32" else b + UNIT[dtype] * (np.abs(y) + b) + (2.0 ** -25 if dtype == "f16" else 0.0)


def to64(t):
    return t.detach().cpu().to(torch.float64).numpy()


class Case:
    """A batch over a pool: lens = [(new rows, positions with them)], random pages, values as given.  Everything in the pool
    that no sequence holds is NaN."""

    def __init__(self, lens, nh, nkv, hd, ps, dtype, cache, seed=0, extra_rows=0, extra_pages=2, size=1.0, n_layer=1,
                 row_pad=0, row_off=0):
        self.lens, self.nh, self.nkv, self.hd, self.ps = lens, nh, nkv, hd, ps
        self.dtype, self.cache, self.n_layer = dtype, cache, n_layer
        rng = np.random.default_rng(seed)
        self.rng = rng
        held = [-(-kv // ps) for _, kv in lens]
        self.n_pages = sum(held) + extra_pages
        order = rng.permutation(self.n_pages)
        self.stride = max(held + [1])
        self.pages = np.full((max(1, len(lens)), self.stride), -1, np.int32)
        at = 0
        for s, h in enumerate(held):
            self.pages[s, :h] = order[at:at + h]
            at += h
        self.starts = np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32)
        self.kv_len = np.asarray([kv for _, kv in lens] or [0], np.int32)
        self.used = int(self.starts[-1])
        self.n_tok = self.used + extra_rows
        dt = DTYPE[dtype]
        gen = torch.Generator().manual_seed(seed)
        self.q = (size * torch.randn(self.n_tok, nh, hd, generator=gen)).to(dt)
        self.k = (size * torch.randn(self.n_tok, nkv, hd, generator=gen)).to(dt)
        self.v = torch.randn(self.n_tok, nkv, hd, generator=gen).to(dt)
        shape = (n_layer, self.n_pages, nkv, ps, hd)
        self.k_pool = torch.full(shape, math.nan, dtype=DTYPE[cache])
        self.v_pool = torch.full(shape, math.nan, dtype=DTYPE[cache])
        for s, (n, kv) in enumerate(lens):
            p = np.arange(kv)
            page = self.pages[s, p // ps]
            self.k_pool[:, page, :, p % ps] = (size * torch.randn(n_layer, kv, nkv, hd, generator=gen)).to(DTYPE[cache]).transpose(0, 1)
            self.v_pool[:, page, :, p % ps] = torch.randn(n_layer, kv, nkv, hd, generator=gen).to(DTYPE[cache]).transpose(0, 1)
        self.row_pad, self.row_off = row_pad, row_off

    # -- device side
    def up(self):
        self.d = {k: getattr(self, k).cuda() for k in ("k_pool", "v_pool")}
        for k in ("pages", "starts", "kv_len"):
            self.d[k] = torch.from_numpy(getattr(self, k)).cuda()
        for k in ("q", "k", "v"):
            self.d[k] = self.wide(getattr(self, k))
        self.d["out"] = self.wide(torch.full_like(self.q, 77.0))
        return self

    def wide(self, x):
        """x's rows in a wider buffer: self.row_off elements in, self.row_pad behind."""
        n = x[0].numel() if x.shape[0] else x.shape[1] * x.shape[2]
        w = torch.full((max(1, x.shape[0]), self.row_off + n + self.row_pad), 55.0, dtype=x.dtype)
        w[:x.shape[0], self.row_off:self.row_off + n] = x.reshape(x.shape[0], n)
        return w.cuda()

    def ptr(self, name):
        t = self.d[name]
        return t.data_ptr() + self.row_off * t.element_size()

    def step(self, name):
        return self.d[name].shape[1]

    def rows(self, name, heads):
        """The rows in a wide buffer, and whether what lies around them is untouched."""
        t = self.d[name].cpu()
        n = heads * self.hd
        inner = t[:self.n_tok, self.row_off:self.row_off + n]
        around = torch.cat([t[:, :self.row_off], t[:, self.row_off + n:]], 1)
        return inner.reshape(self.n_tok, heads, self.hd), bool((around == 55.0).all())

    def handle(self, rope=None):
        from kore_amd import paged
        return paged.PagedKV(self.n_layer, self.n_pages, self.ps, self.nh, self.nkv, self.hd, self.cache, rope,
                             self.d["k_pool"].data_ptr(), self.d["v_pool"].data_ptr())

    def batch(self, max_q=None):
        from kore_amd import paged
        return paged.Batch(len(self.lens), self.n_tok, self.d["starts"].data_ptr(), self.d["kv_len"].data_ptr(),
                           self.d["pages"].data_ptr(), self.stride,
                           max([n for n, _ in self.lens] + [0]) if max_q is None else max_q)

    def attend(self, kv, layer=0, window=0, scale=0.0, max_q=None, workspace=None, stream=None):
        kv.attend_dev(layer, self.batch(max_q), self.dtype, self.ptr("q"), self.ptr("out"), q_stride=self.step("q"),
                      out_stride=self.step("out"), scale=scale, window=window, workspace=workspace, stream=stream)
        if stream is None:
            kv.sync()

    # -- the oracle
    def exact(self, layer=0, window=0, scale=0.0):
        """(out, bound) of every row in 64 bits from the tensors as they are (self.q, the pools); bound as derived below.
        Rows behind the last sequence: NaN in both.

        A score's error: hd products summed in fp32 in any order, (hd + 8) half steps of the sum of their magnitudes S, and
        what operands in parts leave (2^-21 of it).  A weight's relative error is twice the largest score's error of its
        row.  The weights are rounded to half a step of the rows' type (fp32 rows: parts that hold 2^-21 at least).  Sums
        over n keys run in blocks of 16 and more: n / 8 + 16 half steps; the result is rounded once."""
        out = np.full((self.n_tok, self.nh, self.hd), np.nan)
        bound = np.full_like(out, np.nan)
        q, kp, vp = to64(self.q), to64(self.k_pool[layer]), to64(self.v_pool[layer])
        scale = scale or 1 / math.sqrt(self.hd)
        rep = self.nh // self.nkv
        for s, (n, _) in enumerate(self.lens):
            kv_len = int(self.kv_len[s])
            for i in range(n):
                row = int(self.starts[s]) + i
                pos = kv_len - n + i
                p = np.arange(max(0, pos - window + 1 if window else 0), max(0, min(pos + 1, self.stride * self.ps)))
                page = self.pages[s, p // self.ps]
                p = p[(page >= 0) & (page < self.n_pages)]
                if len(p) == 0:
                    out[row], bound[row] = 0, 0
                    continue
                page = self.pages[s, p // self.ps]
                for h in range(self.nh):
                    K, V = kp[page, h // rep, p % self.ps], vp[page, h // rep, p % self.ps]
                    with np.errstate(invalid="ignore", over="ignore"):
                        sc = K @ q[row, h] * scale
                        w = np.exp(sc - sc.max())
                        w /= w.sum()
                        out[row, h] = w @ V
                        S = scale * float((np.abs(K) @ np.abs(q[row, h])).max())
                        u = UNIT[self.dtype] if self.dtype != "f32" else 2.0 ** -21
                        e = 2 * S * ((self.hd + 8) * UNIT["f32"] + 2.0 ** -21) + u + (len(p) / 8 + 16) * UNIT["f32"]
                        bound[row, h] = e * (w @ np.abs(V)) + UNIT[self.dtype] * np.abs(out[row, h]) + \
                            (2.0 ** -24 if self.dtype == "f16" else 0.0)
        return out, bound


def check_rows(case, got, want, bound, name=""):
    """got (torch) against want (numpy) where want is a number; NaN and infinities the same."""
    g = to64(got)[:case.used]
    w, b = want[:case.used], bound[:case.used]
    fine = np.isfinite(w)
    assert np.array_equal(np.isnan(g), np.isnan(w)), name + ": NaN elsewhere"
    assert np.array_equal(g[~fine & ~np.isnan(w)], w[~fine & ~np.isnan(w)]), name + ": infinities elsewhere"
    over = np.abs(g - w)[fine] - b[fine]
    assert over.size == 0 or over.max() <= 0, "%s: %.3g over the bound (largest error %.3g)" % (name, over.max(), np.abs(g - w)[fine].max())
