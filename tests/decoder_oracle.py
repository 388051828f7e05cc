"""What the decoder's operators compute, written down in float64 from their definitions: rotary positions and norms of heads,
slots of a paged cache, attention over it.  Plain numpy, no device; the tests hold the kernels to it."""
import numpy as np

STEP = 2.0 ** -24  # the largest relative rounding of an fp32 operation


def bf16(x):
    """fp32 values rounded to the nearest bf16, ties to even, as fp32."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return np.where(np.isfinite(x), r, np.asarray(x, np.float32))


def normed(x, gamma, epsilon):
    x = x.astype(np.float64)
    return x if gamma is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + epsilon) * gamma.astype(np.float64)


def turned(x, positions, frequencies, interleaved, magnitude=1.0):
    """x [..., heads, d] (float64) at positions [...]; the first 2 len(frequencies) channels turn."""
    y, half = x.copy(), len(frequencies)
    if half == 0:
        return y
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
    t = (np.asarray(positions, np.float64)[..., None] * frequencies)[..., None, :]
    y[..., a] = magnitude * (x[..., a] * np.cos(t) - x[..., b] * np.sin(t))
    y[..., b] = magnitude * (x[..., a] * np.sin(t) + x[..., b] * np.cos(t))
    return y


def turned_bound(x, half, interleaved, gamma, magnitude=1.0):
    """How far fp32 may be off for the same rows (x: normed, float64).  Sine and cosine of the reduced angle are off by at most
    2 steps (the angle's rounding, the polynomial's last operations), each product and the sum by 1, the magnitude by 1; a norm adds a sum
    of squares in chains of 8 and a tree of 6 (half of 14 steps behind the root), a mean, a root, a division and two products."""
    bound, i = np.abs(x).copy(), np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
    if half:
        both = abs(magnitude) * (np.abs(x[..., a]) + np.abs(x[..., b]))
        bound[..., a] = bound[..., b] = 5 * both
    return (bound + (13 * np.maximum(bound, np.abs(x)) if gamma is not None else 0)) * STEP


def ranges(n, length, causal, window, prefix, first):
    """[low, high) and place of each of a sequence's n rows."""
    place = np.arange(length - n, length, dtype=np.int64)
    high = place + 1 if causal else np.full(n, length, np.int64)
    if prefix is not None:
        high = np.maximum(high, prefix)
    high = np.minimum(high, length)
    low = np.maximum(0, place - window + 1) if window else np.zeros(n, np.int64)
    if first is not None:
        low = np.maximum(low, first)
    return low, high, place


def attended(q, k, v, low, high, place, scale, cap, slopes):
    """One sequence: q [n, heads, d], k / v [length, kv heads, d]; the result and how far fp32 may be off.

    The bound is that of the summation orders a kernel may take: a dot product of d terms is off by at most (d + 4) steps of the
    sum of its terms' magnitudes (scale and log2 among the 4); a cap adds 8 steps of itself (tanh, two products), a bias 3 of itself.
    An exponential is off by what its argument is, in units of 1, and 2 steps; so is the sum of weights, relative to itself, and a sum
    of n terms by n steps more."""
    n, heads, d = q.shape
    group = heads // k.shape[1]
    out, bound = np.zeros((n, heads, v.shape[2])), np.zeros((n, heads, v.shape[2]))
    key = np.arange(k.shape[0])
    seen = (key >= low[:, None]) & (key < high[:, None])
    rows = seen.any(1)
    for h in range(heads):
        kk, vv, qq = k[:, h // group].astype(np.float64), v[:, h // group].astype(np.float64), q[:, h].astype(np.float64)
        with np.errstate(invalid="ignore", over="ignore"):
            kk, vv = np.where(seen.any(0)[:, None], kk, 0.0), np.where(seen.any(0)[:, None], vv, 0.0)
            x = qq @ kk.T * scale
            off = (d + 4) * (np.abs(qq) @ np.abs(kk).T) * abs(scale)
            if cap:
                x = cap * np.tanh(x / cap)
                off = off + 8 * cap
            if slopes is not None:
                bias = slopes[h].astype(np.float64) * np.abs(place[:, None] - key)
                x, off = x - bias, off + 3 * np.abs(bias)
            off = np.where(np.isfinite(x), off, 0.0)
            x = np.where(seen, x, -np.inf)
            top = x.max(1, keepdims=True, initial=-np.inf)
            p = np.where(seen, np.exp(x - np.where(rows[:, None], top, 0.0)), 0.0)
            p = p / np.where(rows[:, None], p.sum(1, keepdims=True), 1.0)
            for r in np.flatnonzero(rows):  # a key that a row does not see has no part in it, whatever it holds
                s = seen[r]
                out[r, h] = p[r, s] @ vv[s]
                worst = np.where(s, off[r], 0.0).max()
                bound[r, h] = (2 * worst + 2 * s.sum() + 8) * STEP * (p[r, s] @ np.abs(vv[s]))
    return out, bound
