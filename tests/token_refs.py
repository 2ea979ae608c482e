"""64-bit references of the token operators, from their definitions, and the helpers of their tests."""
import numpy as np

from metalaudio_amd import nn

EPS = 2.0 ** -24  # half a step of fp32, relative to the value
HALF = {"f32": EPS, "bf16": 2.0 ** -8, "e4m3": 2.0 ** -4}  # half a step of each type
TINY = np.float32(2.0 ** -100)


def rounded(x, dtype):
    """The values that a tensor of `dtype` holds of x."""
    x = np.asarray(x, np.float32)
    if dtype == "bf16":
        return (nn.bf16_bits(x).astype(np.uint32) << 16).view(np.float32)
    if dtype == "e4m3":
        return nn.E4M3_VALUES[nn.e4m3_bits(x)]
    return x


def row_scales(x):
    """(scale, factor) of each fp32 row, the steps as they are defined."""
    top = np.maximum(np.abs(x).max(-1), TINY).astype(np.float32)
    return top * np.float32(1 / 448), np.float32(448) * (np.float32(1) / top)


def quantise(x):
    x = np.asarray(x, np.float32)
    scale, inv = row_scales(x)
    return rounded(x * inv[..., None], "e4m3"), scale


def rmsnorm(h, w, eps):
    h = np.asarray(h, np.float64)
    return h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)


def rotary(x, pos, heads, hd, dims, base=10000.0, interleaved=False):
    """x [B, S, heads * hd], pos [S or B, S, axes]."""
    B, S = x.shape[:2]
    y = np.asarray(x, np.float64).reshape(B, S, heads, hd).copy()
    pos = np.broadcast_to(np.asarray(pos, np.float64), (B, S, len(dims)))
    off = 0
    for a, d in enumerate(dims):
        ang = pos[..., a, None] * float(np.float32(base)) ** (-2.0 * np.arange(d // 2) / d)
        c, s = np.cos(ang)[:, :, None], np.sin(ang)[:, :, None]
        i = np.arange(d // 2)
        p, q = (off + 2 * i, off + 2 * i + 1) if interleaved else (off + i, off + d // 2 + i)
        u, v = y[..., p].copy(), y[..., q].copy()
        y[..., p], y[..., q] = u * c - v * s, v * c + u * s
        off += d
    return y.reshape(x.shape)


def attend(q, k, v, seen, heads, kv_heads, scale):
    """One sequence: q [T, H * hd] on k, v [S, KV * hd], seen [T, S]. Keys that a query does not see
    have no part in it, whatever they hold. Also gives max |score| sums for tolerances."""
    T, hd = q.shape[0], q.shape[1] // heads
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    out = np.zeros((T, heads * hd))
    spread = np.zeros((T, heads * hd))  # bound of sum_d |q k| scale, and of |v|
    size = np.zeros((T, heads * hd))
    finite = np.isfinite(k).all() and np.isfinite(v).all()
    for h in range(heads):
        c = slice(h * hd, (h + 1) * hd)
        g = h * kv_heads // heads
        kc = slice(g * hd, (g + 1) * hd)
        if finite:  # all queries at once: what is not seen has weight 0
            s = np.where(seen, q[:, c] @ k[:, kc].T * scale, -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[:, c], size[:, c] = p @ v[:, kc], p @ np.abs(v[:, kc])
            spread[:, c] = np.where(seen, np.abs(q[:, c]) @ np.abs(k[:, kc]).T, 0).max(
                -1, keepdims=True) * abs(scale)
            continue
        for t in range(T):
            at = np.nonzero(seen[t])[0]
            kk, vv = k[at][:, kc], v[at][:, kc]
            s = kk @ q[t, c] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, c] = p @ vv
            spread[t, c] = (np.abs(kk) @ np.abs(q[t, c])).max() * abs(scale)
            size[t, c] = p @ np.abs(vv)
    return out, spread, size


def window_seen(n, left, right, sinks):
    i, j = np.arange(n)[:, None], np.arange(n)[None]
    return (j <= i + right) & ((j >= i - left) | (j < sinks))


def attention_tolerance(spread, size, hd, keys, dtype):
    """Scores are sums of hd products, each off by a half step of the running sum at most, and in
    powers of two (a product with log2 e): delta = (hd + 4) EPS spread + 4 EPS moves each probability
    by a factor e^delta, numerator and denominator; sums over the keys add a half step a key; in bf16
    the probabilities are rounded to bf16, and so is the result."""
    delta = (hd + 4) * EPS * spread + 4 * EPS
    rel = 2 * np.expm1(delta) + (keys + 8) * EPS
    if dtype == "bf16":
        rel = rel + 2 * HALF["bf16"]
    return rel * size + 1e-37


def slot_of(p, sinks, slots):
    return p if p < sinks else sinks + (p - sinks) % (slots - sinks)
