"""The paged attention's values at their ends, and the precision that the header states, against plain implementations in
64 bits."""
import math

import numpy as np
import pytest
import torch

from tests.paged_ref import DTYPE, PAIRS, UNIT, Case, check_rows, to64

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


# ---- infinities of V --------------------------------------------------------------

def _by_weight(c, window=0):
    """(out, bound): keys whose score is -inf have no weight and give nothing; of the others, however small their weight, an
    infinity or NaN of V reaches its dim.  Finite dims as Case.exact's, with its bound."""
    kp, vp, q = to64(c.k_pool[0]), to64(c.v_pool[0]), to64(c.q)
    out = np.zeros((c.n_tok, c.nh, c.hd))
    bound = np.zeros_like(out)
    rep = c.nh // c.nkv
    for s, (n, kv) in enumerate(c.lens):
        for i in range(n):
            row = int(c.starts[s]) + i
            pos = kv - n + i
            p = np.arange(max(0, pos - window + 1 if window else 0), pos + 1)
            for h in range(c.nh):
                K, V = kp[c.pages[s, p // c.ps], h // rep, p % c.ps], vp[c.pages[s, p // c.ps], h // rep, p % c.ps]
                with np.errstate(invalid="ignore"):
                    sc = K @ q[row, h] / math.sqrt(c.hd)
                on = sc > -np.inf
                if not on.any():
                    continue
                K, V, sc = K[on], V[on], sc[on]
                w = np.exp(sc - sc.max())
                w /= w.sum()
                F = np.where(np.isfinite(V), V, 0)
                out[row, h] = w @ F
                S = float((np.abs(K[w > 0]) @ np.abs(q[row, h])).max()) / math.sqrt(c.hd)   # (errors of a weight of 0 are none)
                u = UNIT[c.dtype] if c.dtype != "f32" else 2.0 ** -21
                e = 2 * S * ((c.hd + 8) * UNIT["f32"] + 2.0 ** -21) + u + (len(p) / 8 + 16) * UNIT["f32"]
                bound[row, h] = e * (w @ np.abs(F)) + UNIT[c.dtype] * np.abs(out[row, h]) + 2.0 ** -24
                up, down = ((V == np.inf) | np.isnan(V)).any(0), ((V == -np.inf) | np.isnan(V)).any(0)
                out[row, h] = np.where(up & down, np.nan, np.where(up, np.inf, np.where(down, -np.inf, out[row, h])))
    return out, bound


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("hd", [64, 96, 256])
@pytest.mark.parametrize("lens", ["short", "split"])
@pytest.mark.parametrize("max_q", [1, 64])
def test_infinities_reach_a_row_by_its_scores_alone(dtype, cache, hd, lens, max_q):
    """Infinities and NaN of V in keys of ordinary weight, of a weight far under the smallest float (before and behind the
    largest score of the row, near it and a split away) and of none (a score of -inf): where tiles and splits are cut, and
    which kernel is taken, changes nothing."""
    lens = {"short": [(40, 330), (1, 200)], "split": [(3, 2900), (1, 2500)]}[lens]
    c = Case(lens, 2, 1, hd, 32, dtype, cache, seed=hd)
    c.q[..., 7] = c.q[..., 7].abs() + 4.0
    c.k_pool[..., 7] = torch.where(torch.isnan(c.k_pool[..., 7]), c.k_pool[..., 7], torch.zeros_like(c.k_pool[..., 7]))

    def put(s, p, dim, v, k7=None):
        c.v_pool[0, c.pages[s, p // 32], 0, p % 32, dim] = v
        if k7 is not None:
            c.k_pool[0, c.pages[s, p // 32], 0, p % 32, 7] = k7

    far, gone = -8.0 * 2000, -math.inf
    put(0, 3, 0, math.inf)                      # of ordinary weight: in tiles that all see it
    put(0, 40, 1, -math.inf)
    put(0, 41, 2, math.nan)
    put(0, 50, 3, math.inf)
    put(0, 150, 3, -math.inf)                   # both in one dim
    put(0, 9, 4, math.inf, far)                 # weights of 2^-2000 and less
    put(0, 130, 5, -math.inf, far)
    put(0, lens[0][1] - 2, 6, math.inf, far)    # that the last rows alone see
    put(0, 20, 7, math.nan, far)
    put(0, 10, 8, math.inf, gone)               # no weight
    put(0, 140, 9, math.nan, gone)
    put(0, lens[0][1] - 1, 10, -math.inf, gone)
    for p in range(64):                         # sequence 1: nothing but far keys, then ordinary ones
        put(1, p, 11, math.inf if p == 5 else 1.0, far)
    put(1, 199, 12, -math.inf, gone)
    put(1, 100, 13, math.inf)
    c.up()
    with c.handle() as kv:
        c.attend(kv, max_q=max_q)
        check_rows(c, c.rows("out", 2)[0], *_by_weight(c))
        c.attend(kv, max_q=max_q, window=170)
        check_rows(c, c.rows("out", 2)[0], *_by_weight(c, 170), "window")


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("max_q", [1, 64])
def test_rows_without_weight_get_zeros_beside_infinities(dtype, cache, bad, max_q):
    """Every attended score is -inf: zeros, whatever V holds, in whole and in split tiles."""
    c = Case([(3, 40), (20, 300), (1, 3000)], 6, 2, 64, 16, dtype, cache, seed=3)
    c.q[..., 7] = c.q[..., 7].abs() + 0.5
    c.k_pool[..., 7] = -math.inf
    c.v_pool[..., ::5] = bad
    c.up()
    with c.handle() as kv:
        c.attend(kv, max_q=max_q)
    assert (to64(c.rows("out", 6)[0]) == 0).all()


@pytest.mark.parametrize("dtype,cache", [p for p in PAIRS if p[1] != "f16"])
@pytest.mark.parametrize("max_q", [1, 64])
def test_an_infinity_at_the_other_end_of_the_scores(dtype, cache, max_q):
    """Scores of +-2^127 (before the scale), further apart than fp32 reaches: the lower keys' infinities count, and nothing else
    of them."""
    c = Case([(40, 150), (1, 70)], 2, 1, 64, 16, dtype, cache, seed=6)
    c.q[:] = 0
    c.q[..., 0] = 2.0 ** 63
    for s, (_, kv) in enumerate(c.lens):
        for p in range(kv):
            at = (0, c.pages[s, p // 16], 0, p % 16)
            c.k_pool[at] = 0
            c.k_pool[at + (0,)] = 2.0 ** 64 if p % 3 == 0 else -2.0 ** 64
        c.v_pool[0, c.pages[s, 0], 0, 5, 3 + s] = math.inf       # position 5, low
    c.up()
    with c.handle() as kv:
        c.attend(kv, max_q=max_q)
    got = to64(c.rows("out", 2)[0])
    for s, (n, kv_len) in enumerate(c.lens):
        for i in range(n):
            p = np.arange(0, kv_len - n + i + 1, 3)     # those of the high score share the weight
            V = to64(c.v_pool[0, c.pages[s, p // 16], 0, p % 16])
            want, e = V.mean(0), (2 * UNIT[dtype] + 2.0 ** -20 + (len(p) / 8 + 16) * 2.0 ** -24) * np.abs(V).mean(0)
            row = got[int(c.starts[s]) + i]
            assert (row[:, 3 + s] == math.inf).all()
            row[:, 3 + s] = want[3 + s]
            assert (np.abs(row - want) <= e).all()


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("max_q", [1, 64])
def test_other_rows_do_not_notice_a_q_that_is_not_finite(dtype, cache, bad, max_q):
    """A row, a head and a single value of q are not finite: the others' bits are those of a finite q."""
    c = Case([(30, 200), (1, 2500), (2, 40)], 6, 2, 64, 16, dtype, cache, seed=11).up()
    with c.handle() as kv:
        c.attend(kv, max_q=max_q)
        want = c.rows("out", 6)[0].clone()
        odd = torch.zeros(c.n_tok, 6, dtype=torch.bool)
        odd[4], odd[11, 2], odd[31, 5], odd[20, 0] = True, True, True, True
        c.q[4], c.q[11, 2], c.q[31, 5] = bad, bad, bad
        c.q[20, 0, 17] = bad
        c.d["q"].copy_(c.wide(c.q))
        torch.cuda.synchronize()
        c.attend(kv, max_q=max_q)
    got = c.rows("out", 6)[0]
    assert torch.equal(got[~odd].view(torch.uint8), want[~odd].view(torch.uint8))


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


# ---- the precision that the header states -------------------------------------------

def _cut(x, bits):
    """fp32 values cut to their first `bits` bits."""
    m, e = np.frexp(np.asarray(x, np.float64))
    return np.ldexp(np.trunc(np.ldexp(m, bits)), e - bits)


@pytest.mark.parametrize("cache", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("max_q", [1, 64])
def test_fp32_rows_root_mean_square(cache, hd, max_q):
    """fp32 rows of N(0, 1) values: the root mean square error, relative to the outputs'.  With values of independent sign, a
    score's error is what hd products and sums leave, sqrt(hd) half steps of fp32 at most, and q's and K's parts, half of 2^-21
    each (22 bits).  An error d of the scores is one of d in the outputs (sum w d v beside sum w v).  The weights' parts, 2^-21
    at most, the sums' n / 8 + 16 roundings as roots, and the result's own follow.  A q of 16 bits, as two bf16 parts hold, is
    beyond it: shown on the oracle."""
    n, kv = 48, 600
    c = Case([(n, kv)], 4, 2, hd, 32, "f32", cache, seed=hd).up()
    with c.handle() as h:
        c.attend(h, max_q=max_q)
    got = to64(c.rows("out", 4)[0])
    want, _ = c.exact()
    rms = lambda x: float(np.sqrt(np.mean(np.square(x))))  # noqa: E731
    bound = math.sqrt(sum(x * x for x in (math.sqrt(hd) * 2.0 ** -24, 2.0 ** -22, 2.0 ** -22, 2.0 ** -21, math.sqrt(kv / 8 + 16) * 2.0 ** -24, 2.0 ** -24)))
    assert rms(got - want) <= bound * rms(want), (rms(got - want) / rms(want), bound)
    c.q = torch.from_numpy(_cut(c.q.numpy(), 16)).float()
    assert rms(c.exact()[0] - want) > 2 * bound * rms(want)
