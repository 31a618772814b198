"""The 8-bit K/V cache and its attention in 64 bits: the definition that the
CUDA kernels are held to. Plain numpy, one sequence at a time."""
import numpy as np

BLOCK, E_MIN, E_MAX = 16, -48, 64


def exponent(amax):
    """The smallest e in [E_MIN, E_MAX] with amax <= 127 * 2^e."""
    for e in range(E_MIN, E_MAX):
        if amax <= 127.0 * 2.0 ** e:
            return e
    return E_MAX


class Held:
    """One sequence's keys (or values): integers [positions][heads][dim] and a
    scale's exponent per block and head."""

    def __init__(self, heads, dim):
        self.codes = np.zeros((0, heads, dim))
        self.exps = np.zeros((0, heads), np.int64)

    def append(self, rows):
        rows = np.asarray(rows, np.float64)
        rows = np.where(np.isfinite(rows), rows, 0.0)
        if not len(rows):
            return
        heads = rows.shape[1]
        start, end = len(self.codes), len(self.codes) + len(rows)
        self.codes = np.concatenate([self.codes, np.zeros_like(rows)])
        for b in range(start // BLOCK, -(-end // BLOCK)):
            lo, hi = max(start, b * BLOCK), min(end, (b + 1) * BLOCK)
            if b == len(self.exps):
                self.exps = np.concatenate([self.exps, np.full((1, heads), E_MIN)])
            for h in range(heads):
                x = rows[lo - start:hi - start, h]
                was = self.exps[b, h] if lo > b * BLOCK else E_MIN
                e = max(was, exponent(np.abs(x).max()))
                old = self.codes[b * BLOCK:lo, h]
                self.codes[b * BLOCK:lo, h] = np.rint(old * 2.0 ** (was - e))
                self.codes[lo:hi, h] = np.clip(np.rint(x / 2.0 ** e), -127, 127)
                self.exps[b, h] = e

    def values(self):
        n = len(self.codes)
        return self.codes * (2.0 ** self.exps.repeat(BLOCK, 0)[:n])[..., None]


def attention(q, keys, values, window=0, scale=None):
    """q [rows][heads][dim] at the last `rows` positions of keys, values
    [length][kv_heads][dim]; returns the output and, per row and head, the
    largest sum of |scale q k| over a key's dims, the bound of its scores."""
    rows, heads, dim = q.shape
    length, kv_heads = keys.shape[:2]
    scale = dim ** -0.5 if scale is None else scale
    q = q.astype(np.float64)
    out, size = np.zeros(q.shape), np.zeros((rows, heads))
    for r in range(rows):
        at = length - rows + r
        first = max(0, at - window + 1) if window else 0
        if at < 0:
            continue
        for h in range(heads):
            k, v = keys[first:at + 1, h * kv_heads // heads], values[first:at + 1, h * kv_heads // heads]
            s = scale * (k @ q[r, h])
            size[r, h] = scale * (np.abs(k) @ np.abs(q[r, h])).max()
            p = np.exp(s - s.max())
            out[r, h] = (p @ v) / p.sum()
    return out, size


def attention_bound(size, biggest, out, dim, length, bf16):
    """How far a kernel that keeps the documented precision may be from the
    exact output, per element. size: attention()'s bound of a row's scores;
    biggest: the largest |value|. u = 2^-23 is twice fp32's half step, the
    worst of a truncating addition.

    A score: q in 22 bits (2u: two halves; as bytes it has 23 or, in bf16,
    15, which hold its 8) and at most dim/8 + 8 rounded additions and products
    of partial sums, each below the score's own bound. A weight: the error of
    its exponent, the exponential (within 2u) and the rounding to two halves
    (2u; as bytes 32 bits of the largest). The output: a weighted mean, whose
    numerator and denominator each take a weight's error and one rounded
    addition per block and per merged share. Rows in bf16 add a weight's
    rounding to one half, 2^-12 (numerator only), and the output's, 2^-8."""
    u = 2.0 ** -23
    score = size * (dim / 8 + 10) * u
    weight = score + 4 * u
    steps = (length / 16 + 128) * u
    bound = 2 * (weight + steps) * (1 + weight)
    if bf16:
        bound = bound + 2.0 ** -12
    bound = bound[..., None] * biggest
    return bound + (2.0 ** -8 if bf16 else u) * np.abs(out) + 1e-30
