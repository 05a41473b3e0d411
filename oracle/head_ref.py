"""CPU oracle (test infrastructure only) for the operators of the fully connected head: layer norm, dropout without a stored
mask, and the 8-bit product with block scales.  numpy in 64 bits, written from the formulas; the reference has no code for
any of them.  Philox and the rounding to bf16 come from fc_ref."""
import numpy as np

from .fc_ref import philox4x32_10

E4M3_MAX = 448.0


# ---- layer norm ------------------------------------------------------------------------------------------------------
def layer_norm(x, w=None, b=None, eps=1e-5):
    """-> y, mean, rstd, h in 64 bits; x [rows, cols]."""
    x = np.asarray(x, np.float64)
    mu = x.mean(1, keepdims=True)
    r = 1.0 / np.sqrt(((x - mu) ** 2).mean(1, keepdims=True) + eps)
    h = (x - mu) * r
    y = h if w is None else h * np.asarray(w, np.float64)
    return (y if b is None else y + np.asarray(b, np.float64)), mu, r, h


def layer_norm_bwd(dy, x, w=None, eps=1e-5):
    """-> dx, dw, db in 64 bits."""
    dy = np.asarray(dy, np.float64)
    _, _, r, h = layer_norm(x, eps=eps)
    g = dy if w is None else dy * np.asarray(w, np.float64)
    dx = r * (g - g.mean(1, keepdims=True) - h * (g * h).mean(1, keepdims=True))
    return dx, (dy * h).sum(0), dy.sum(0)


# ---- dropout ---------------------------------------------------------------------------------------------------------
def keep_mask(seed, n, p):
    """True where element e of a row-major tensor is kept: (r >> 8) * 2^-24 >= p in fp32."""
    r = philox4x32_10(seed, np.arange((n + 3) // 4, dtype=np.uint64)).reshape(-1)[:n]
    return (r >> np.uint32(8)).astype(np.float32) * np.float32(2.0 ** -24) >= np.float32(p)


def dropout(x, p, seed, slope=1.0):
    """-> y in 64 bits.  p decides as an fp32 number, its scale is 1 / (1 - p); slope is the fp32 number the kernels get."""
    x = np.asarray(x, np.float64)
    keep = keep_mask(seed, x.size, p).reshape(x.shape)
    scale = 0.0 if np.float32(p) >= 1 else 1.0 / (1.0 - p)
    with np.errstate(invalid="ignore"):
        return np.where(keep, np.where(x > 0, x, x * float(np.float32(slope))) * scale, 0.0)


def dropout_bwd(dy, y, p, seed, slope=1.0):
    dy = np.asarray(dy, np.float64)
    keep = keep_mask(seed, dy.size, p).reshape(dy.shape)
    scale = 0.0 if np.float32(p) >= 1 else 1.0 / (1.0 - p)
    with np.errstate(invalid="ignore"):
        return np.where(keep, dy * scale * (1.0 if slope == 1.0 else np.where(np.asarray(y, np.float64) > 0, 1.0, float(np.float32(slope)))), 0.0)


# ---- e4m3 blocks of 128 ----------------------------------------------------------------------------------------------
def to_e4m3(v):
    """Round to e4m3 (1 sign, 4 exponent, 3 mantissa bits, no infinities), to nearest, ties to even; what lies beyond 448
    by half a step or more, infinities and NaN give NaN.  Values, in 64 bits."""
    v = np.asarray(v, np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        _, e = np.frexp(np.where(np.isfinite(v), v, 1.0))
        step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
        q = np.rint(v / step) * step
        return np.where(np.isfinite(v) & (np.abs(q) <= E4M3_MAX), q, np.nan)


def scale_exponent(amax):
    """Smallest whole e >= -127 with amax <= 448 * 2^e; 0 for amax = 0."""
    amax = np.asarray(amax, np.float64)
    m, e = np.frexp(amax)                  # 448 = 0.875 * 2^9
    e = e - 9 + (m > 0.875)
    return np.where(amax > 0, np.maximum(e, -127), 0).astype(np.int64)


def quantize(x, rows, cols):
    """Blocks of rows x cols -> (values on the e4m3 grid, block exponents [blocks down, blocks across]); the scale is taken
    from the block's finite elements."""
    x = np.asarray(x, np.float64)
    r, c = x.shape
    p = np.zeros((-(-r // rows) * rows, -(-c // cols) * cols))
    p[:r, :c] = x
    t = p.reshape(p.shape[0] // rows, rows, p.shape[1] // cols, cols)
    e = scale_exponent(np.where(np.isfinite(t), np.abs(t), 0.0).max((1, 3)))
    q = to_e4m3(np.ldexp(t, -e[:, None, :, None]))
    return q.reshape(p.shape)[:r, :c], e


def rounded(x, rows, cols):
    """The values x stands for after quantize(x, rows, cols)."""
    q, e = quantize(x, rows, cols)
    return np.ldexp(q, np.repeat(np.repeat(e, rows, 0)[: q.shape[0]], cols, 1)[:, : q.shape[1]])
