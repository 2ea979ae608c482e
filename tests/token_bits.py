"""Distances in the 2-norm that the token operators keep, and fp32 attention with a number of partial
products to see that those distances tell them apart."""
import numpy as np

from tests.token_refs import EPS

# fp32 attention: a score is off by its products' sums (below 1e-7 of ordinary scores) and, as a power of
# two minus the reference, by a half step of an argument up to about 10 (rms 2e-7 or below); exp2, the sums and
# the quotient add a few half steps (0.42 * 2^-24 rms each). An output is off by as much relative to itself as
# the probabilities, whose errors and whose values are averaged over the same keys: 3e-7, three times that here.
ATTENTION_F32 = 1e-6
# bf16 results: a rounding is 0.42 half steps rms of values of all sizes, 1.65e-3. Whole sequences round the
# probabilities as well, which comes to the same again: 2.3e-3.
ATTENTION_BF16 = 2.6e-3
STEP_BF16 = 1.9e-3


def linear_f32(K):
    """One rounding of about 2^-25 rms of the running sum for each of the K / 16 matrix instructions behind
    one another, 3e-8 sqrt(K / 16) of the result where the sums grow evenly (their mean square is half the
    last one's), and as much again for the scales."""
    return 3e-8 * np.sqrt(K / 16) / np.sqrt(2) + 6e-8


def distance(got, want):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    return np.linalg.norm(got - want) / np.linalg.norm(want)


def bf16(x):
    """fp32 rounded to bf16, as 64-bit numbers (finite values)."""
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32).astype(np.float64)


def parts(x):
    """x as three bf16 values."""
    x = np.asarray(x, np.float32).astype(np.float64)
    h = bf16(x)
    m = bf16(x - h)
    return h, m, x - h - m


def product(a, b, kept):
    """a @ b.T of fp32 values by `kept` (3 or 6) partial products of their parts, the sum rounded to fp32."""
    a, b = parts(a), parts(b)
    pairs = [(0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0)][:kept]
    return sum(a[i] @ b[j].T for i, j in pairs).astype(np.float32)


def attention(q, k, v, seen, kept):
    """One head in fp32, its two products by `kept` partial products."""
    scale = np.float32(q.shape[1] ** -0.5 * np.log2(np.e))
    s = np.where(seen, product(q * scale, k, kept), np.float32(-np.inf))
    p = np.exp2(s - s.max(-1, keepdims=True)).astype(np.float32)
    return product(p, v.T, kept) / p.sum(-1, keepdims=True, dtype=np.float32)
