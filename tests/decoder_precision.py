"""Attention over a cache where a lost bit shows: the worst case of a dot product of d terms hides whether a kernel that splits fp32
into three bf16 numbers kept the third.  Here every score is one product, every sum of weights has two terms, or every weight is one.
Plain numpy, no device: the inputs, how far fp32 may be off, and the kernels' arithmetic with a part or a product left out, which has to
show (test_decoder_precision.py)."""
import numpy as np

from decoder_oracle import STEP, bf16

WINDOWS = {"values": 1, "weights": 2, "scores": 8}


def queries(rng, what, rows, d):
    """[rows, d]: one pair of neighbouring channels a row for the scores, any values otherwise."""
    if what != "scores":
        return rng.standard_normal((rows, d)).astype(np.float32)
    q = np.zeros((rows, d), np.float32)
    pair = 2 * rng.integers(0, d // 2, rows)
    for i in range(2):
        q[np.arange(rows), pair + i] = 1 + rng.random(rows) / 256
    return q


def keys(rng, what, shape, elem):
    """[..., slots, d], slots in the order of places, an even number: near 256 in every other channel and 0 between, the next key the other way
    round, so that a row's scores are single products near 256, by one channel of its query or the other."""
    k = rng.standard_normal(shape).astype(np.float32)
    if what == "scores":
        at = (np.arange(shape[-2])[:, None] + np.arange(shape[-1])) % 2
        k = np.where(at == 0, 256 + k, 0).astype(np.float32)
    return bf16(k) if elem == "bf16" else k


def values(rng, what, shape, elem):
    v = np.ones(shape, np.float32) if what == "weights" else rng.standard_normal(shape).astype(np.float32)
    return bf16(v) if elem == "bf16" else v


def expected(what, q, k, v, seen):
    """q [rows, d], k and v [keys, d], seen [rows, keys] (scale 1): the result in float64 and how far fp32 may be off.

    values: the weight is 1, so the result is the value, bit for bit: the sum of its three parts is exact in any order that starts
    with the smaller two.  weights: two weights a and b, and (a + b) / (a + b): the sum of their parts is off by 2 steps for each of up to three
    instructions that add them, the sum of the weights by 1; a rescaling rounds both once, a join each twice; a reciprocal and a product
    follow: 16 steps at most.  scores: the scaled query is off by 3 steps (log2(e), the scale, the product), the products of the parts
    that are left out are 2 steps, their sum is off by 2, an exponential by 1: 8 steps of the largest score in every weight's exponent, to first
    order times the spread of the values around the result (2% more for the second), and the sums' and weights' own 2 n + 16 steps."""
    if what == "weights":
        return np.ones((len(q), v.shape[1])), np.full((len(q), v.shape[1]), 16 * STEP)
    x = np.where(seen, q.astype(np.float64) @ k.T.astype(np.float64), -np.inf)
    p = np.exp(x - x.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    want = p @ v.astype(np.float64)
    if what == "values":
        return want, np.zeros_like(want)
    largest = np.abs(np.where(seen, x, 0)).max(1)
    spread = np.stack([p[r] @ np.abs(v - want[r]) for r in range(len(q))])
    return want, STEP * (1.02 * 8 * largest[:, None] * spread + (2 * seen.sum(1)[:, None] + 16) * (p @ np.abs(v)))


def parts_of(x, keep=3):
    """fp32 as three bf16 numbers, of which `keep` are kept."""
    out = []
    for _ in range(3):
        out.append(bf16(x))
        x = (x - out[-1]).astype(np.float32)
    return out[:keep]


def by_parts(q, k, v, seen, elem, keep=(3, 3, 3, 3), without=()):
    """The kernels' arithmetic: products of parts whose numbers add up to 2 at most, but those left out `without`, in fp32 otherwise.  keep:
    parts of queries, keys, weights, values."""
    def product(a, b, a_keep, b_keep):
        total = np.zeros((a.shape[0], b.shape[1]))
        for i, x in enumerate(parts_of(a, a_keep)):
            for j, y in enumerate(parts_of(b, b_keep)):
                if i + j <= 2 and (i, j) not in without:
                    total = total + x.astype(np.float64) @ y.astype(np.float64)
        return total.astype(np.float32)

    one = 1 if elem == "bf16" else None
    x = product((q * np.float32(1.44269504)).astype(np.float32), np.ascontiguousarray(k.T), keep[0], one or keep[1])
    x = np.where(seen, x, -np.inf).astype(np.float32)
    p = np.exp2((x - x.max(1, keepdims=True)).astype(np.float32)).astype(np.float32)
    return product(p, v, keep[2], one or keep[3]) / p.sum(1, keepdims=True, dtype=np.float32)
