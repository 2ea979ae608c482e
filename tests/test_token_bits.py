"""The distances of token_bits.py tell fp32 work from work with fewer bits (no GPU)."""
import numpy as np
import pytest

from tests import token_bits as bits
from tests.token_refs import attend, quantise, window_seen


@pytest.mark.parametrize("S,hd,left,right,sinks", [
    (33, 48, 5, 0, 2), (65, 128, 1000, 1000, 70), (130, 32, 16, 16, 4), (257, 72, 100, 0, 33),
    (300, 96, 0, 299, 3), (400, 48, 168, 168, 4), (700, 64, 300, 1, 129)])
def test_attention_by_three_products_is_seen(S, hd, left, right, sinks):
    rng = np.random.default_rng(S)
    q, k, v = (rng.standard_normal((S, hd)).astype(np.float32) * s for s in (1.3, 1.3, 1))
    q, k, v = (x.astype(np.float32) for x in (q, k, v))
    seen = window_seen(S, left, right, sinks)
    want = attend(q, k, v, seen, 1, 1, hd ** -0.5)[0]
    assert bits.distance(bits.attention(q, k, v, seen, 6), want) <= bits.ATTENTION_F32
    assert bits.distance(bits.attention(q, k, v, seen, 3), want) > 2 * bits.ATTENTION_F32


@pytest.mark.parametrize("K", [128, 384, 1536, 2048])
def test_linear_with_narrow_sums_is_seen(K):
    """Sums that drop what lies 14 bits below the largest product of each 64."""
    rng = np.random.default_rng(K)
    x, _ = quantise(rng.standard_normal((40, K)).astype(np.float32))
    w, _ = quantise((rng.standard_normal((50, K)) / np.sqrt(K)).astype(np.float32))
    p = x.astype(np.float64)[:, None] * w[None]
    want = p.sum(-1)
    g = p.reshape(40, 50, K // 64, 64)
    unit = np.exp2(np.floor(np.log2(np.abs(g).max(-1, keepdims=True))) - 14)
    narrow = (np.trunc(g / unit) * unit).sum((-1, -2))
    wide = np.zeros((40, 50), np.float32)
    for i in range(0, K, 16):
        wide = (wide + p[..., i:i + 16].sum(-1)).astype(np.float32)
    assert bits.distance(wide, want) <= bits.linear_f32(K)
    assert bits.distance(narrow, want) > 2 * bits.linear_f32(K)
