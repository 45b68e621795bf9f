"""Trees whose outputs rest on one product of 16-bit terms each.

The tree attention takes each operand as a sum of 16-bit terms (bf16: K and V of an
f32 cache, q and the weights P three; f16: all of a q8_0 cache's two; a bf16 cache's
K and V are one) and sums the products of terms that matter.  A case here cancels
all of these but one, (a, b): term a of K or V with term b of q or P.  Its output is
about 1 where that product counts and far from it where it is lost.

`emulate` is the arithmetic in numpy, products left out at will.
"""
import numpy as np

import kv_plain

SCALE = float(np.float32(np.log(2.0)))  # scale * log2(e) is 1 in f32: scores are in base 2
assert np.float32(SCALE) * np.float32(1.44269504088896) == 1.0

PRODUCTS = {"F32": [(2, 0), (1, 1), (0, 2), (1, 0), (0, 1), (0, 0)], "BF16": [(0, 2), (0, 1), (0, 0)],
            "Q8_0": [(1, 0), (0, 1), (0, 0)]}
T1, T2 = 2.0 ** -9, 2.0 ** -18  # what the second and the third bf16 term of 1 + T1 + T2 are
HIDDEN = 31                     # a column of each block that q leaves out: it sets the block's scale


def split(x, dtype, cached):
    """The terms of f64 values that f32 (K, V of a cache: its type) holds."""
    if dtype == "Q8_0":
        hi = x.astype(np.float16).astype(np.float64)
        return [hi, (x - hi).astype(np.float16).astype(np.float64)]
    terms = []
    for _ in range(1 if cached and dtype == "BF16" else 3):
        t = (kv_plain.bf16_bits(x.astype(np.float32)).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        terms.append(t)
        x = x - t
    return terms


def emulate(dtype, q, k, v, lost_scores=(), lost_values=()):
    """One row: q [hd] f32, k and v [positions, hd] as the cache holds them."""
    q = q.astype(np.float64)
    up = 2.0 ** (10 - np.floor(np.log2(np.abs(q).max()))) if dtype == "Q8_0" and q.any() else 1.0
    qt, kt, vt = split(q * up, dtype, False), split(k, dtype, True), split(v, dtype, True)
    s = sum(kt[a] @ qt[b] for a, b in PRODUCTS[dtype] if (a, b) not in lost_scores) / up
    p = np.exp2(s - s.max() + 7.0).astype(np.float32).astype(np.float64)
    pt = split(p, dtype, False)
    return sum(pt[b] @ vt[a] for a, b in PRODUCTS[dtype] if (a, b) not in lost_values) / p.sum()


def _two_terms():
    """(scale, code, hi, lo) of a q8_0 value scale * code = hi + lo with the largest lo."""
    best = None
    for m in range(1025, 2048, 2):
        for code in range(65, 127):
            x = m * code
            step = 2.0 ** (np.floor(np.log2(x)) - 10)
            hi = float(np.float16(x / step)) * step  # 11 bits, nearest even
            if best is None or abs(x - hi) / x > abs(best[3]) / (best[2] + best[3]):
                best = (float(m), code, hi, x - hi)
    m, code, hi, lo = best
    return m / 256, code, hi / 256, lo / 256


def _unit(rows, hd, dims):
    """K rows that are 1 in one column each (and 127 / 64 where q is 0, for q8_0)."""
    k = np.zeros((rows, hd))
    k[:, HIDDEN::32] = 127.0 / 64.0
    k[np.arange(rows), dims] = 1.0
    return k


def cases(dtype, hd, at):
    """{(part, a, b): (q, k, v)}: the row's q [hd], K and V [positions, hd]; the columns
    that matter start at `at`.  part 0: a product of the scores, 1: of the values."""
    got = {}
    ones = np.zeros((2, hd))
    ones[1] = 1.0  # position 1 has the score in question, position 0 zero
    ones[1, HIDDEN::32] = 127.0 / 64.0

    def scores(a, b, qs, ks, x):
        q, k = np.zeros(hd), np.zeros((2, hd))
        k[:, HIDDEN::32] = 127.0 / 64.0
        q[at:at + len(qs)], k[1, at:at + len(ks)] = x * np.array(qs), ks
        got[0, a, b] = (q, k, ones)

    def values(a, b, log2p, vs, x):
        n = len(vs)
        q, dims = np.zeros(hd), at + np.arange(n)
        q[dims] = log2p
        v = np.repeat(x * np.array(vs, np.float64)[:, None], hd, axis=1)
        if dtype == "Q8_0":  # 64 steps of the block's scale
            v[:, HIDDEN::32] = v[:, :1] * 127.0 / 64.0
        got[1, a, b] = (q, _unit(n, hd, dims), v)

    less = np.log2(1.0 - 2.0 ** -10)
    if dtype == "Q8_0":
        scores(0, 1, [1 + 2.0 ** -12, -1], [1, 1], 2.0 ** 14)
        values(0, 1, [0, np.log2(1.0 - 2.0 ** -13)], [1, -1], 2.0 ** 14)
        m, code, hi, lo = _two_terms()
        # K and V hold hi + lo in a block of scale m, hi in one of scale hi / 64
        q, k = np.zeros(hd), np.zeros((2, hd))
        other = (at + 32) % hd
        k[1, at], k[1, at // 32 * 32 + HIDDEN] = m * code, m * 127
        k[1, other], k[1, other // 32 * 32 + HIDDEN] = hi, hi / 64 * 127
        x = 2.0 ** np.round(np.log2(4.0 / abs(lo)))
        q[at], q[other] = x * np.sign(lo), -x * np.sign(lo)
        got[0, 1, 0] = (q, k, ones)
        v = np.zeros((2, hd))
        v[0], v[1] = m * code, -hi
        v[0, HIDDEN::32], v[1, HIDDEN::32] = m * 127, -hi / 64 * 127
        q = np.zeros(hd)
        got[1, 1, 0] = (q, _unit(2, hd, at + np.arange(2)), v * 2.0 ** (1 - np.round(np.log2(abs(lo)))))
        return got
    scores(0, 1, [1 + T1, -1], [1, 1], 2.0 ** 11)
    scores(0, 2, [1 + T1 + T2, -1 - T1], [1, 1], 2.0 ** 20)
    values(0, 1, [0, less], [1, -1], 2.0 ** 11)
    # (the third term of P: near half a step of the second, as f32 exponents of 7 hold them)
    values(0, 2, [less, np.log2(1 - 2.0 ** -10 - 1.75 * 2.0 ** -19), 0], [1, -1, 0], 2.0 ** 20)
    if dtype == "F32":
        scores(1, 0, [1, -1], [1 + T1, 1], 2.0 ** 11)
        scores(2, 0, [1, -1], [1 + T1 + T2, 1 + T1], 2.0 ** 20)
        scores(1, 1, [1 + T1, -1 - T1, -1, 1], [1 + T1, 1, 1 + T1, 1], 2.0 ** 20)
        values(1, 0, [0, 0], [1 + T1, -1], 2.0 ** 10)
        values(2, 0, [0, 0], [1 + T1 + T2, -1 - T1], 2.0 ** 19)
        values(1, 1, [less, less, 0, 0], [1 + T1, -1, -1 - T1, 1], 2.0 ** 21)
    return got


def padded(case, before, far):
    """`before` positions of no weight in front: their column `far` of K is 1, q's there -64."""
    q, k, v = case
    q, hd = q.copy(), len(q)
    if before:
        q[far] = -64.0
    return (q.astype(np.float32), np.concatenate([_unit(before, hd, np.full(before, far)), k]),
            np.concatenate([np.zeros((before, hd)), v]))
