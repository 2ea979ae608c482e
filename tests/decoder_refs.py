"""64-bit references of the decoder's operators, from their definitions: 8-bit products with scales for
blocks of 128, 8-bit rows of caches, attention to the states of an encoder."""
import numpy as np

from tests.token_refs import EPS, HALF, attend, attention_tolerance, quantise

BLOCK = 128


def blocks_of(n):
    return -(-n // BLOCK)


def quantise_blocks(x):
    """Rows in blocks of 128: (values, scales [.., blocks])."""
    x = np.asarray(x, np.float32)
    q, scales = np.empty_like(x), np.empty(x.shape[:-1] + (blocks_of(x.shape[-1]),), np.float32)
    for j in range(scales.shape[-1]):
        c = slice(j * BLOCK, (j + 1) * BLOCK)
        q[..., c], scales[..., j] = quantise(x[..., c])
    return q, scales


def quantise_tiles(w):
    """Weights in blocks of 128 x 128: (values, scales)."""
    w = np.asarray(w, np.float32)
    q, scales = np.empty_like(w), np.empty((blocks_of(w.shape[0]), blocks_of(w.shape[1])), np.float32)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            at = slice(i * BLOCK, (i + 1) * BLOCK), slice(j * BLOCK, (j + 1) * BLOCK)
            flat, s = quantise(w[at].reshape(1, -1))
            q[at], scales[i, j] = flat.reshape(w[at].shape), s[0]
    return q, scales


def spread_scales(scales, shape, rows=1):
    """Each value's scale, as 64-bit numbers: blocks of `rows` x 128."""
    s = np.repeat(np.asarray(scales, np.float64), BLOCK, -1)[..., :shape[-1]]
    return np.repeat(s, rows, -2)[:shape[-2]] if rows > 1 else s


def linear_blocks(xq, xs, wq, ws, bias):
    """(y before the activation, sum of magnitudes) in 64 bits."""
    x = xq.astype(np.float64) * spread_scales(xs, xq.shape)
    w = wq.astype(np.float64) * spread_scales(ws, wq.shape, BLOCK)
    y = x @ w.T
    return (y if bias is None else y + bias), np.abs(x) @ np.abs(w).T


def held_rows(x, heads):
    """Rows [.., heads * hd] as an 8-bit cache holds them: (values, scales [.., heads])."""
    x = np.asarray(x, np.float32)
    q, s = quantise(x.reshape(*x.shape[:-1], heads, x.shape[-1] // heads))
    return q.reshape(x.shape), s


def values_of(q, scales):
    """What 8-bit rows stand for, in 64 bits."""
    heads = scales.shape[-1]
    x = q.astype(np.float64).reshape(*q.shape[:-1], heads, q.shape[-1] // heads)
    return (x * scales.astype(np.float64)[..., None]).reshape(q.shape)


def memory(q, k, v, heads, kv_heads, scale):
    """One sequence's tokens on all of k and v; zeros where there are none: (out, spread, size)."""
    if len(k) == 0:
        z = np.zeros(q.shape)
        return z, z, z
    return attend(q, k, v, np.ones((len(q), len(k)), bool), heads, kv_heads, scale)


def held_tolerance(spread, size, hd, keys, dtype):
    """attention_tolerance, and the roundings of the scales: of each score's product with its key's scale
    and the scores' own, of each probability's with its value's scale, and of the sums' order."""
    return attention_tolerance(spread, size, hd + 8, keys + 8, dtype)


def split_tolerance(spread, size, hd, keys, dtype):
    """attention_tolerance where keys are split into ranges that are joined: a factor a range and side."""
    return attention_tolerance(spread, size, hd, keys + 16, dtype)


__all__ = ["BLOCK", "EPS", "HALF", "blocks_of", "held_rows", "held_tolerance", "linear_blocks", "memory",
           "quantise_blocks", "quantise_tiles", "split_tolerance", "spread_scales", "values_of"]
