"""The 8-bit KV cache and attention over caches in float64, from their
definitions, for the tests of kv_append_rows_*, attn_*_fp8 and
attn_decode_prefix_*."""
import numpy as np

# e4m3 magnitudes in the order of their codes (4 exponent bits of bias 7, 3 of mantissa; code 127 is NaN)
LEVELS = np.array([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)][:127])


def encode(x):
    """Codes [..., hd] and scale bytes [...] of f32 x: the smallest scale 2^e, e >= -127, that
    brings the largest magnitude to at most 448, then the nearest level, between two the even code."""
    x = np.asarray(x, np.float64)
    amax = np.abs(x).max(-1)
    bad = ~np.isfinite(amax)
    e = np.full(amax.shape, -127)
    for cand in range(121, -128, -1):
        with np.errstate(invalid="ignore", over="ignore"):
            e[amax <= 448 * 2.0 ** cand] = cand
    a = np.abs(np.where(bad[..., None], 0, x)) * 2.0 ** -e[..., None].astype(np.float64)
    mid = (LEVELS[1:] + LEVELS[:-1]) / 2
    low, high = np.searchsorted(mid, a, side="left"), np.searchsorted(mid, a, side="right")
    code = np.where(low % 2 == 0, low, high) | np.where(np.signbit(x) & ~bad[..., None], 128, 0)
    return code.astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def decode(codes, scales):
    """f64 values of codes [..., hd] with scale bytes [...]."""
    table = np.concatenate((LEVELS, [np.nan], -LEVELS, [np.nan]))
    s = scales.astype(np.float64)
    return table[codes] * np.where(s == 255, np.nan, 2.0 ** (s - 127))[..., None]


def attend(q, k, v):
    """softmax(q k^T / sqrt(hd)) v in f64, q [rows][hd], k and v [keys][hd], and what the bound of
    a result needs: A, the largest sum |q k| / sqrt(hd) of a row."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    if not len(k):
        return np.zeros_like(q), 0.0
    s = q @ k.T / np.sqrt(q.shape[1])
    p = np.exp(s - s.max(-1, keepdims=True))
    return p @ v / p.sum(-1, keepdims=True), float((np.abs(q) @ np.abs(k).T / np.sqrt(q.shape[1])).max())


def bound(A, keys, vmax):
    """How far an output may be from the exact one.  A score: q in two fp16
    terms (2^-22 of each product), K exact, f32 sums of up to 2 x 128 products
    (MFMA steps of 32: 8 roundings, 2^-21), scaled and subtracted in one
    rounding of at most twice the score (2^-23): under 2^-20 A.  A probability
    is off by that factor, by the hardware 2^x (2^-22) and its two terms
    (2^-22); l adds up to keys / 4 terms a lane in f32 and the merges a few
    more; O as many MFMA steps.  Numerator and denominator: twice."""
    return 2 * vmax * (2.0 ** -20 * (A + 1) + (keys / 4 + 64) * 2.0 ** -24)
