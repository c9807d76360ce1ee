"""The paged attention's values at their ends, against plain implementations in 64 bits."""
import math

import numpy as np
import pytest
import torch

from tests.paged_ref import DTYPE, UNIT, Case, to64

pytestmark = pytest.mark.gpu


# ---- scores far from 0 ---------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("common", [2 ** 10, 2 ** 13, 2 ** 14, 2 ** 17, 2 ** 21, 2 ** 23, -2 ** 14, -2 ** 23])
@pytest.mark.parametrize("lens", ["short", "split"])
@pytest.mark.parametrize("max_q", [1, 64])
def test_scores_with_a_common_part(dtype, common, lens, max_q):
    """Every score has the same large part, which softmax takes out again; what they differ by decides.  q and K are whole
    numbers, so that scores are exact in fp32.  Neighbouring 64 keys have different largest scores: the reference moves, and
    differs between the waves, teams and splits whose sums are joined.

    A weight's relative error: half a step of the type in the chunks (u, in the numerator and in the sum), the scale's and
    the exponent's rounding (distances of up to 60 binades times 2^-23, under 2^-17), and what the common part's own rounding
    may leave between two sums: 2^-13.  Sums: n / 8 + 16 half steps.  The result is rounded once."""
    c = Case({"short": [(40, 700), (1, 700), (64, 64)], "split": [(70, 3000), (2, 2500)]}[lens], 6, 2, 64, 32, dtype, dtype, seed=5)
    g = torch.Generator().manual_seed(abs(common) + len(c.lens))
    c.q = torch.randint(-1, 2, c.q.shape, generator=g).to(DTYPE[dtype])
    k = torch.randint(-2, 3, c.k_pool.shape, generator=g).to(DTYPE[dtype])
    a = 2 ** (int(math.log2(abs(common))) // 2)
    c.q[..., 0], k[..., 0] = math.copysign(a, common), abs(common) // a
    c.q[..., 1] = 1
    for s, (_, kv) in enumerate(c.lens):
        p = np.arange(kv)
        k[0, c.pages[s, p // 32], :, p % 32, 1] = torch.from_numpy(8.0 * (p // 64 * 5 % 9)).to(DTYPE[dtype])[:, None]
    c.k_pool = torch.where(torch.isnan(c.k_pool), c.k_pool, k)
    c.up()
    with c.handle() as kv_:
        c.attend(kv_, max_q=max_q)
    got = to64(c.rows("out", 6)[0])
    q, kp, vp = to64(c.q), to64(c.k_pool[0]), to64(c.v_pool[0])
    u = UNIT[dtype]
    for s, (n, kv) in enumerate(c.lens):
        for i in range(n):
            row, p = int(c.starts[s]) + i, np.arange(kv - n + i + 1)
            K, V = (x[c.pages[s, p // 32], :, p % 32] for x in (kp, vp))
            for h in range(6):
                sc = K[:, h // 3] @ q[row, h] / 8
                w = np.exp(sc - sc.max())
                w /= w.sum()
                want, size = w @ V[:, h // 3], w @ np.abs(V[:, h // 3])
                e = (2 * u + 2.0 ** -13 + 2.0 ** -17 + (len(p) / 8 + 16) * 2.0 ** -24) * size + u * np.abs(want) + 2.0 ** -24
                assert (np.abs(got[row, h] - want) <= e).all(), (row, h, float((np.abs(got[row, h] - want) / e).max()))


# ---- units of q and K ----------------------------------------------------------------

@pytest.mark.parametrize("cache", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("max_q", [1, 64])
def test_large_values_that_meet_zeros(cache, max_q):
    """q and K are large, each where the other is 0: scores of 0, the mean of V, whatever the scale."""
    c = Case([(20, 90), (1, 40)], 4, 2, 64, 16, "f32", cache, seed=7)
    c.q[:] = 0
    c.q[..., 3] = 2.0 ** 100
    c.k_pool = torch.where(torch.isnan(c.k_pool), c.k_pool, torch.zeros_like(c.k_pool))
    c.k_pool[..., 5] = torch.where(torch.isnan(c.k_pool[..., 5]), c.k_pool[..., 5], torch.full_like(c.k_pool[..., 5], 2.0 ** (15 if cache == "f16" else 100)))
    c.up()
    with c.handle() as kv:
        for scale in (0.0, 1.0, 1e30, 1e-30):
            c.attend(kv, max_q=max_q, scale=scale)
            got = to64(c.rows("out", 4)[0])
            vp = to64(c.v_pool[0])
            for s, (n, kv_len) in enumerate(c.lens):
                for i in range(n):
                    p = np.arange(kv_len - n + i + 1)
                    V = vp[c.pages[s, p // 16], :, p % 16].repeat(2, 1)
                    e = (2.0 ** -20 + (len(p) / 8 + 16) * 2.0 ** -24) * np.abs(V).mean(0)
                    assert (np.abs(got[int(c.starts[s]) + i] - V.mean(0)) <= e).all(), scale
