"""Attention of new rows over cached ones in 64 bits, with a bound on the error of the device's result."""
import numpy as np

EPS = {"f32": 2.0 ** -23, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}


def to_bits(a):
    """float32 -> bf16 bits, to the nearest, ties to even."""
    u = np.ascontiguousarray(a, dtype=np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r)


def rounded(a, kind):
    """float32 values as `kind` holds them, in float32."""
    a = np.ascontiguousarray(a, dtype=np.float32)
    if kind == "f16":
        with np.errstate(over="ignore"):
            return a.astype(np.float16).astype(np.float32)
    if kind == "bf16":
        return (to_bits(a).astype(np.uint32) << 16).view(np.float32)
    return a


def stored(a, kind):
    """float32 values as the session's host arrays of `kind`."""
    return to_bits(a) if kind == "bf16" else rounded(a, kind).astype(np.float16 if kind == "f16" else np.float32)


def loaded(a, kind):
    """The session's host arrays as float32."""
    return (a.astype(np.uint32) << 16).view(np.float32) if kind == "bf16" else a.astype(np.float32)


def sees(count, context, parents=None):
    """[count][context + count]: whether a row sees a position."""
    if parents is None:
        return np.arange(context + count)[None] <= context + np.arange(count)[:, None]
    out = np.zeros((count, context + count), dtype=bool)
    out[:, :context] = True
    for j in range(count):
        n = j
        while n >= 0:
            out[j, context + n] = True
            n = parents[n]
    return out


def attention(q, keys, values, visible, scale, row_kind, cache_kind):
    """y [rows][heads][dim] of q [rows][heads][dim] over keys, values [positions][kv_heads][dim] (as the
    cache holds them), and how far the device may be from it.

    The bound, with u = 2^-24.  A score's parts: q in the cache's type is exact (rows of 16 bits, f32, three
    parts of bf16: 2^-24) or, as two parts of f16, off by 2^-22 of the row's largest at each element; a sum of
    dim products, each at most u off at each of dim additions; two roundings by the factor.  A score's error e
    makes a probability's relative one e, and as much in their sum.  The exponential, the probabilities' split and
    the joins' factors: 16 u, and u of the exponent's argument; parts of f16 are off by 2^-25 at least, next to
    2^9 or more for the row's largest probability (a half of the smallest step, and as much of the second part).  Sums over n positions: no longer chain of additions than n / 8 + 64 (a lane adds
    every eighth probability; a product sums 16 at a time).  Probabilities of 16-bit rows are rounded once, and
    so is their output."""
    rows, heads, dim = q.shape
    group = heads // keys.shape[1]
    y, bound = np.zeros(q.shape), np.zeros(q.shape)
    u = 2.0 ** -24
    for h in range(heads):
        k, v = keys[:, h // group].astype(np.float64), values[:, h // group].astype(np.float64)
        x = q[:, h].astype(np.float64)
        live = visible.any(0)
        kf = np.where(live[:, None], k, 0)
        with np.errstate(invalid="ignore", over="ignore"):
            s = np.where(visible, scale * (x @ kf.T), -np.inf)
            size = scale * (np.abs(x) @ np.abs(kf).T)
            e = (dim + 4) * u * size
            if row_kind == "f32" and cache_kind == "f16":
                e += scale * 2.0 ** -22 * np.abs(x).max(1, keepdims=True) * np.abs(kf).sum(1)[None]
            elif row_kind == "f32" and cache_kind == "bf16":
                e += u * size
            e = np.where(visible, e, 0).max(1, keepdims=True)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            vf = np.where(live[:, None], v, 0)
            y[:, h] = p @ vf
            reach = p @ np.abs(vf)
            far = (p * np.where(p > 0, s.max(1, keepdims=True) - s, 0)) @ np.abs(vf)
            chain = visible.sum(1, keepdims=True) / 8 + 64
            bound[:, h] = (2 * e + (16 + chain) * u) * reach + 2 * u * far
            if cache_kind == "f16":
                bound[:, h] += 2.0 ** -33 * visible @ np.abs(vf)
            if row_kind != "f32":
                bound[:, h] += 1.001 * EPS[row_kind] / 2 * (reach + np.abs(y[:, h])) + 2.0 ** -24
    return y, bound
