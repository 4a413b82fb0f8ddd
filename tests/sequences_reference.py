"""Attention over packed sequences, e4m3 rows and the paged cache in 64 bits, with how far a kernel's rounding may be off (numpy, CPU)."""
import numpy as np

HALF = 2.0 ** -8                # half a step of bf16, relative


def bf16_round(x):
    """float32 -> bf16 bits, ties to even; NaN stays NaN"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(np.asarray(x, np.float32)), np.uint16(0x7fc0), r).astype(np.uint16).reshape(np.shape(x))


def bf16_value(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def e4m3_value(codes):
    c = np.asarray(codes, np.uint8).astype(np.int64)
    e, f = (c >> 3) & 15, (c & 7) / 8.0
    v = np.where(e == 0, np.ldexp(f, -6), np.ldexp(1 + f, e - 7))
    v = np.where((c & 0x7f) == 0x7f, np.nan, v)
    return np.where(c >> 7, -v, v)


def scale_value(s):
    return np.where(np.asarray(s) == 255, np.nan, np.ldexp(1.0, np.asarray(s, np.int64) - 127))


E4M3 = e4m3_value(np.arange(127, dtype=np.uint8))                  # the values >= 0, rising with their codes


def quantise(x):
    """(codes, scales) of rows in the last dimension, from the definition"""
    x = np.asarray(x, np.float64)
    top = np.abs(x).max(-1)
    bad = ~np.isfinite(top)
    safe = np.where(bad | (top == 0), 1.0, top)
    e = np.ceil(np.log2(safe / 448.0)).astype(np.int64)
    e = np.where(np.ldexp(448.0, e - 1) >= safe, e - 1, np.where(np.ldexp(448.0, e) < safe, e + 1, e))     # the logarithm's own rounding
    e = np.where(top == 0, -127, np.maximum(e, -127))
    r = np.where(bad[..., None], 0.0, np.abs(np.where(np.isfinite(x), x, 0.0))) * np.ldexp(1.0, -e)[..., None]
    hi = np.clip(np.searchsorted(E4M3, r), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = E4M3[hi] - r, r - E4M3[lo]
    code = np.where(up < down, hi, np.where(down < up, lo, np.where(hi % 2 == 0, hi, lo))).astype(np.uint8)
    code = np.where(bad[..., None], 0x7f, code | (np.signbit(x).astype(np.uint8) << 7)).astype(np.uint8)
    return code, np.where(bad, 255, e + 127).astype(np.uint8)


def spans(first, limit):
    """[from, to) of every sequence: a value counts as the largest up to its place, limited to 0 .. limit"""
    at = np.clip(np.maximum.accumulate(np.maximum(np.asarray(first, np.int64), 0)), 0, limit)
    return list(zip(at[:-1], at[1:]))


def softmax_rows(q, k, v, scale, limit):
    """q [n, heads, hd], k, v [m, kv, hd] in float64; row i sees the keys below limit[i] (or limit[i] is a set of truth values). Returns the
    result and the sizes that errors are relative to: sum p |v| / sum p, and the largest scale * sum |q| |k| of the row"""
    n, heads, hd = q.shape
    out, weight, size = np.zeros((n, heads, hd)), np.zeros((n, heads, hd)), np.zeros((n, heads, 1))
    if not k.shape[0]:
        return out, weight, size
    group = heads // k.shape[1]
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        for i in range(n):
            sees = np.arange(len(kh)) < limit[i] if np.ndim(limit[i]) == 0 else limit[i]
            if not sees.any():
                continue
            s = scale * (kh[sees] @ q[i, h])
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ vh[sees]
            weight[i, h] = p @ np.abs(vh[sees])
            size[i, h] = abs(scale) * (np.abs(kh[sees]) @ np.abs(q[i, h])).max()
    return out, weight, size


def bound(out, weight, size, hd, rounded):
    """The output's rounding; where P is rounded to bf16 (`rounded`) half a step of every term and of the sum that divides them; f32
    arithmetic: a product of hd terms and its scaling, the exponential, and the sums over keys, at a few units in the 24th place."""
    f32 = (2 * (hd + 8) * size + 64) * 2.0 ** -24
    return HALF * np.abs(out) + (2 * HALF * weight if rounded else 0.0) * (1 + HALF) + f32 * weight + 2.0 ** -126


def check(got, want, what=""):
    out, limit = want
    bad = ~(np.abs(got - out) <= limit)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} values, first at {np.argwhere(bad)[0]}: {got[bad][:3]} for {out[bad][:3]} within {limit[bad][:3]}"
