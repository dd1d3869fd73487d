"""The 8-bit KV cache's definition in numpy, for the tests: blocks of 32 rows,
scale = fp32(amax / 127), code = nearest integer to value / scale (ties to
even, on the exact quotient), attention and eviction in float64."""
import numpy as np

BLOCK = 32
TINY = 127.0 * float(np.finfo(np.float32).tiny)


def quantise(x):
    """Blocks of float32 rows x [n, D] (n counted from a block's edge): codes, scales."""
    x = np.asarray(x, np.float32)
    n = len(x)
    codes, scales = np.zeros(x.shape, np.int8), np.zeros((n + BLOCK - 1) // BLOCK, np.float32)
    for b in range(len(scales)):
        v = x[b * BLOCK:(b + 1) * BLOCK]
        if not np.isfinite(v).all():
            scales[b] = np.nan
            continue
        top = np.abs(v).max()
        if float(top) < TINY:
            continue
        s = np.float32(np.float64(top) / 127.0)
        scales[b] = s
        # a quotient of two fp32 numbers is a multiple of 2^-24 of its size away from a tie or on it:
        # float64 (2^-53) rounds it on the right side
        codes[b * BLOCK:(b + 1) * BLOCK] = np.rint(v.astype(np.float64) / np.float64(s))
    return codes, scales


def values(codes, scales):
    """fp32 values of codes [n, D] with their blocks' scales."""
    return codes.astype(np.float32) * np.repeat(np.asarray(scales, np.float32), BLOCK)[:len(codes), None]


def attention(q, k, v, past, scale):
    """q [n, heads, D], k and v [H, rows, D] in float64: out, the weight of each row [H, rows],
    and the largest sum of |q||k| of a row's scores (for the tolerance)."""
    n, heads, D = q.shape
    H = len(k)
    out, w, big = np.zeros((n, heads, D)), np.zeros(k.shape[:2]), np.zeros((n, heads))
    for j in range(heads):
        h = j // (heads // H)
        for t in range(n):
            r = max(0, min(past + t + 1, k.shape[1]))
            if r == 0:
                continue
            s = scale * (k[h, :r] @ q[t, j])
            big[t, j] = abs(scale) * (np.abs(k[h, :r]) @ np.abs(q[t, j])).max()
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, j] = p @ v[h, :r]
            w[h, :r] += p
    return out, w, big


def evicted(w, length, keep, sink, recent):
    """The rows that a head keeps, in order."""
    if length <= keep:
        return np.arange(length)
    mid = np.arange(sink, length - recent)
    order = mid[np.lexsort((mid, -w[mid].astype(np.float64)))][:keep - sink - recent]
    return np.concatenate([np.arange(sink), np.sort(order), np.arange(length - recent, length)])


def moved(x, kept, codes, scales):
    """Codes and scales of the kept rows packed down: x [rows, D] their fp32 values, blocks in place as they were."""
    c, s = quantise(x[kept])
    for b in range(len(s)):
        r = kept[b * BLOCK:(b + 1) * BLOCK]
        if (r == np.arange(b * BLOCK, b * BLOCK + len(r))).all():
            c[b * BLOCK:(b + 1) * BLOCK], s[b] = codes[r], scales[b]
    return c, s
