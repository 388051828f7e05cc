"""What the operators around a paged cache compute, in float64 from their definitions: trees of drafted tokens, masses of keys, who stays in a full
cache, pages chosen by their means.  Plain numpy, no device."""
import numpy as np

from decoder_oracle import STEP


def attended_where(q, k, v, seen, distance, scale, cap, slopes):
    """One sequence: q [n, heads, d], k / v [length, kv heads, d], seen and distance [n, length] or [n, kv heads, length].  The result and how far fp32 may be
    off, and the weights [n, heads, length] with theirs.

    The bound is decoder_oracle.attended's: a product of d terms is off by (d + 4) steps of its terms' magnitudes, a cap adds 8 steps of itself, a bias 3; a
    weight is off by what its argument and the largest argument are, a step for each term of the sum it is divided by, and 8 more."""
    n, heads, d = q.shape
    length, group = k.shape[0], heads // k.shape[1]
    out, bound = np.zeros((n, heads, v.shape[2])), np.zeros((n, heads, v.shape[2]))
    weights, off_weights = np.zeros((n, heads, length)), np.zeros((n, heads, length))
    for h in range(heads):
        g = h // group
        mine = seen[:, g] if seen.ndim == 3 else seen
        some = mine.any(0)[:, None]
        kk, vv, qq = np.where(some, k[:, g].astype(np.float64), 0.0), v[:, g].astype(np.float64), q[:, h].astype(np.float64)
        with np.errstate(invalid="ignore", over="ignore"):
            x = qq @ kk.T * scale
            off = (d + 4) * (np.abs(qq) @ np.abs(kk).T) * abs(scale)
            if cap:
                x = cap * np.tanh(x / cap)
                off = off + 8 * cap
            if slopes is not None:
                bias = slopes[h].astype(np.float64) * np.abs(distance)
                x, off = x - bias, off + 3 * np.abs(bias)
            off = np.where(np.isfinite(x), off, 0.0)
            for r in np.flatnonzero(mine.any(1)):
                s = mine[r]
                p = np.exp(x[r, s] - x[r, s].max())
                p = p / p.sum()
                worst = (2 * off[r, s].max() + 2 * s.sum() + 8) * STEP
                weights[r, h, s], off_weights[r, h, s] = p, p * worst
                out[r, h], bound[r, h] = p @ vv[s], worst * (p @ np.abs(vv[s]))
    return out, bound, weights, off_weights


def tree(parents, length, window=0, first=None):
    """seen and distance [n, length] of the rows of a tree, the newest n tokens of a sequence of `length`."""
    n = len(parents)
    base = length - n
    depth = np.zeros(n, np.int64)
    for t in range(n):
        depth[t] = depth[parents[t]] + 1 if parents[t] >= 0 else 0
    key = np.arange(length)
    position = np.where(key < base, key, base + depth[np.clip(key - base, 0, n - 1)])
    distance = (base + depth)[:, None] - position
    seen = np.zeros((n, length), bool)
    for t in range(n):
        seen[t] = (key < base) & (key >= (first[t] if first is not None else 0))
        u = t
        while u >= 0:
            if base + u >= 0:
                seen[t, base + u] = True
            u = parents[u]
    return seen & (distance < window) if window else seen, distance


def stays(mass, position, budget, recent, first):
    """Which slots of one head stay, places in order."""
    length = len(mass)
    if length <= budget:
        return np.ones(length, bool)
    safe = (position.astype(np.int64) < first) | (position > int(position.max()) - recent)
    value = np.where(np.isnan(mass), -np.inf, mass.astype(np.float64))
    # The last key counts most: those kept by their position (by place alone), numbers, by mass, by place.
    order = np.lexsort((np.arange(length), np.where(safe, 0.0, -value), ~safe & np.isnan(mass), ~safe))
    out = np.zeros(length, bool)
    out[order[:budget]] = True
    return out


def chosen_pages(q, means, place, page, most, first, last):
    """The pages that a row at `place` sees for one head of keys: q [group, d], means [pages, d] (fp32)."""
    mine = place // page
    if mine + 1 <= most:
        return np.arange(mine + 1)
    with np.errstate(invalid="ignore", over="ignore"):
        # Summed the same way for each page, so that pages of the same mean have the same score (a matrix product treats its last columns differently).
        products = np.stack([(row.astype(np.float64) * means[:mine + 1].astype(np.float64)).sum(-1) for row in q])
    score = np.where(np.isnan(products).all(0), np.nan, np.where(np.isnan(products), -np.inf, products).max(0))
    number = np.arange(mine + 1)
    always = (number < first) | (number > mine - last)
    rest = number[~always]
    order = rest[np.lexsort((rest, -np.where(np.isnan(score[rest]), -np.inf, score[rest]), np.isnan(score[rest])))]
    return np.sort(np.concatenate([number[always], order[:most - always.sum()]]))
