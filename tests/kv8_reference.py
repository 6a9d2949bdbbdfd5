"""The 8-bit paged cache and its operators from their definitions (include/strata_cuda.h), in NumPy:
whole numbers and scales exactly, attention in 64 bits. One sequence and head at a time."""
import numpy as np

BLOCK = 64
TINY = np.float32(2.0 ** -100)


def padded(dim):
    return 64 if dim <= 64 else 128 if dim <= 128 else 256


def quantise(rows):
    """rows [n <= 64, dim] f32 -> codes [n, dim] int, scale (f32)"""
    rows = np.where(np.isfinite(rows), rows, 0).astype(np.float32)
    amax = np.float32(np.abs(rows).max()) if rows.size else np.float32(0)
    if amax < TINY:
        return np.zeros(rows.shape, np.int64), np.float32(0)
    scale = np.float32(amax / np.float32(127))
    return np.clip(np.rint(rows * np.float32(np.float32(1) / scale)), -127, 127).astype(np.int64), scale


def pack_keys(codes, dim):
    """codes [n, dim] -> a page's key bytes"""
    p = padded(dim)
    full = np.zeros((BLOCK, p), np.int8)
    full[: codes.shape[0], :dim] = codes
    return full.reshape(BLOCK, p // 64, 64).transpose(1, 0, 2).reshape(-1)


def pack_values(codes, dim):
    full = np.zeros((padded(dim), BLOCK), np.int8)
    full[:dim, : codes.shape[0]] = codes.T
    return full.reshape(-1)


def blocks_of(keys, values):
    """One head's rows [n, dim] -> per block (key codes, key scale, value codes, value scale)"""
    out = []
    for at in range(0, keys.shape[0], BLOCK):
        kc, ks = quantise(keys[at:at + BLOCK])
        vc, vs = quantise(values[at:at + BLOCK])
        out.append((kc, ks, vc, vs))
    return out


def dequantised(blocks):
    """-> keys, values [n, dim] in 64 bits, as the cache holds them"""
    k = np.concatenate([b[0] * np.float64(b[1]) for b in blocks])
    v = np.concatenate([b[2] * np.float64(b[3]) for b in blocks])
    return k, v


def attend(q, k, v, scale, allowed):
    """q [n, dim], k, v [keys, dim], allowed [n, keys] -> (y [n, dim], bound [n]): the result in 64 bits and how
    far an evaluation with the products' and sums' rounding may be from it, for each row.

    The bound, with u = 2^-24 the unit of F32 and the two FP16 halves of a query or a weight exact to
    2^-22 of their row's largest: a logit of terms a_d = scale q_d k_d is off by at most
    (4 u + (dim + 8) u) sum |a_d| (representation, then one rounding for each of dim sums and of the few scalings),
    the exponent adds 4 u times the span of the logits, so each weight has at most a relative error e = their sum;
    the normalised sum moves by at most 2 e max|v|. Adding up n weighted values in blocks of 64 rounds at most
    64 + n / 64 + 16 times on the way of any term, and a weight's halves add 4 u of the largest weight, of
    which there are n at most against a sum of at least 1: (80 + n / 64 + 4 n) u max|v|, taken for
    the n that matter, the sum of the weights over the largest."""
    u = 2.0 ** -24
    n, dim = q.shape
    q, k, v = q.astype(np.float64), np.asarray(k, np.float64), np.asarray(v, np.float64)
    a = (q @ k.T) * scale
    size = (np.abs(q) @ np.abs(k).T) * abs(scale) + np.abs(q).max(-1, keepdims=True) * np.abs(k).sum(-1)[None] * abs(scale) * 0.5
    y, bound = np.zeros((n, v.shape[1])), np.zeros(n)
    for i in range(n):
        at = allowed[i]
        if not at.any():
            continue
        row = a[i, at]
        w = np.exp(row - row.max())
        y[i] = (w / w.sum()) @ v[at]
        top = np.abs(v[at]).max()
        e = (dim + 12) * u * size[i, at].max() + 4 * u * (row.max() - row.min())
        count = at.sum()
        bound[i] = top * (2 * e + (80 + count / 64) * u + 4 * u * count / w.sum())
    return y, bound


def select(q, marks, key_scales, have, top, first, last):
    """q [group, dim] f32, marks (lo, hi) [blocks, dim], key_scales [blocks] -> picked blocks, ascending"""
    if have <= top:
        return np.arange(have)
    q = np.where(np.isfinite(q), q, 0).astype(np.float32)
    amax = np.float32(np.abs(q).max())
    unit = np.float32(0) if amax < TINY else np.float32(np.float32(32767) / amax)
    r = np.rint(q * unit).astype(np.int64)
    pos, neg = np.maximum(r, 0).sum(0), np.minimum(r, 0).sum(0)
    big = np.float32(max(pos.max(), -neg.min()))
    fine = np.float32(0) if big == 0 else np.float32(np.float32(127) / big)
    p, m = np.rint(pos.astype(np.float32) * fine).astype(np.int64), np.rint(neg.astype(np.float32) * fine).astype(np.int64)
    lo, hi = marks
    score = ((hi[:have].astype(np.int64) @ p) + (lo[:have].astype(np.int64) @ m)).astype(np.float32) * key_scales[:have].astype(np.float32)
    score = score.astype(np.float64)
    score[:first] = np.inf
    score[have - last:] = np.inf
    order = np.argsort(-score, kind="stable")[:top]
    return np.sort(order)
