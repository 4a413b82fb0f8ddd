"""MXFP4 (blocks of 32, power-of-two scales, E2M1 codes) in numpy and 64 bits: the plain form the GPU tests compare with."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def blocks(cols):
    return (cols + 31) // 32


def bf16_round(x):
    """float32 -> nearest bf16, as uint16 (finite values, infinities; NaN stays NaN)"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + np.uint32(0x7fff) + ((u >> np.uint32(16)) & np.uint32(1))) >> np.uint32(16)).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def bf16_value(h):
    return (np.asarray(h, np.uint16).astype(np.uint32) << np.uint32(16)).view(np.float32)


def encode(x):
    """x float32 [rows, cols] -> codes uint8 [rows, 16 nb], scales uint8 [rows, nb]"""
    x = np.asarray(x, np.float32).astype(np.float64)
    rows, cols = x.shape
    nb = blocks(cols)
    b = np.zeros((rows, nb * 32))
    b[:, :cols] = x
    b = b.reshape(rows, nb, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    e = np.clip(np.where(top > 0, np.frexp(top)[1] - 1, -1000) - 2, -127, 127)
    v = np.minimum(np.abs(b) * np.ldexp(1.0, -e)[..., None], 6.0)
    d = np.abs(v[..., None] - GRID)
    code = np.argmin(d, -1)                                       # the lower one of two as near
    tie = (code < 7) & (np.take_along_axis(d, code[..., None], -1)[..., 0] == np.abs(GRID[np.minimum(code + 1, 7)] - v))
    code = np.where(tie & (code % 2 == 1), code + 1, code)
    code = code | np.where(np.signbit(b), 8, 0)
    code = np.where(bad[..., None], 0, code).reshape(rows, nb * 16, 2)
    return (code[..., 0] | code[..., 1] << 4).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def decode(codes, scales, cols):
    """float64 [..., cols]"""
    grid = np.concatenate([GRID, -GRID])
    v = np.stack([grid[codes & 15], grid[codes >> 4]], -1).reshape(*codes.shape[:-1], -1, 32)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    with np.errstate(invalid="ignore"):
        return (v * s[..., None]).reshape(*codes.shape[:-1], -1)[..., :cols]


def random_codes(rng, rows, cols, scale_from, scale_to):
    """Codes and scales of any rows x cols values, the columns behind the last one zero"""
    nb = blocks(cols)
    half = rng.integers(0, 16, (rows, nb * 32))
    half[:, cols:] = 0
    half = half.reshape(rows, nb * 16, 2)
    return (half[..., 0] | half[..., 1] << 4).astype(np.uint8), rng.integers(scale_from, scale_to, (rows, nb), endpoint=True).astype(np.uint8)
