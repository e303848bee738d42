"""E4M3 and the block-scaled products in 64 bits, in numpy: what the GPU tests of the FP8 operators compare with."""
import numpy as np


def decode(b):
    """E4M3 bytes -> float64 (0x7F, 0xFF: NaN)."""
    b = np.asarray(b, np.uint8).astype(np.int64)
    e, m = b >> 3 & 15, b & 7
    v = np.where(e > 0, (8 + m) * np.exp2(e - 10.0), m * 2.0**-9)
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b >= 128, -v, v)


_CODES = decode(np.arange(127))                       # 0 .. 448, ascending


def encode(v):
    """float64 -> E4M3 bytes, to nearest, ties to the even code; |v| <= 448 or NaN."""
    v = np.asarray(v, np.float64)
    a = np.where(np.isnan(v), 0, np.abs(v))
    hi = np.searchsorted(_CODES, a).clip(0, 126)
    lo = np.maximum(hi - 1, 0)
    d_hi, d_lo = _CODES[hi] - a, a - _CODES[lo]
    code = np.where((d_lo < d_hi) | ((d_lo == d_hi) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.isnan(v), 127, code) | np.where(np.signbit(v), 128, 0)
    return code.astype(np.uint8)


def blocks(n):
    return (n + 127) // 128


def quantize(x):
    """(bytes, f32 scales) of f32 rows."""
    n, K = x.shape
    v = np.zeros((n, blocks(K) * 128))
    v[:, :K] = x
    v = v.reshape(n, -1, 128)
    v = np.where(np.isfinite(v), v, np.nan)
    most = np.nan_to_num(np.abs(v), nan=0.0).max(2)
    m, e = np.frexp(most)                             # most = m * 2^e; 448 = 0.875 * 2^9
    scale = np.where(most > 0, np.exp2(np.maximum(e - 9 + (m > 0.875), -126).astype(np.float64)), 1.0)
    return encode(v / scale[:, :, None]).reshape(n, -1)[:, :K], scale.astype(np.float32)


def weights(rng, M, K, mats=None, spread=0.02):
    """Random E4M3 matrices and scales that are no powers of two."""
    shape = (M, K) if mats is None else (mats, M, K)
    q = encode(np.clip(rng.standard_normal(shape) * 100, -448, 448))
    s = (spread / 100 * rng.uniform(0.5, 2.0, shape[:-2] + (blocks(M), blocks(K)))).astype(np.float32)
    return q, s


def expand(q, scale, rows):
    """float64 values of E4M3 with a scale for each `rows` x 128."""
    s = scale.astype(np.float64).repeat(rows, -2)[..., :q.shape[-2], :].repeat(128, -1)[..., :q.shape[-1]]
    with np.errstate(invalid="ignore"):
        return decode(q) * s


def product(w, w_scale, xq, x_scale):
    """(y, bound): the product in 64 bits, and how far f32 sums may be from it.  Per column block 128 products are added, exact products with one
    rounding each (the tensor cores may cut instead of rounding: 2^-23 of the sum of magnitudes), then the scales' product, the scaling and the
    addition of every block round once, and the result once more."""
    W, X = expand(w, w_scale, 128), expand(xq, x_scale, 1)
    size = np.abs(X) @ np.abs(W).T
    return X @ W.T, size * 2.0**-23 * (128 + blocks(W.shape[1]) + 4)
