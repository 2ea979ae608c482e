"""The bits that the token operators hold, through the C ABI against 64-bit references: sums of products
that cancel, and distances in the 2-norm, which the bounds of single elements are too wide to see.
Tolerances count roundings (token_refs.py) and were fixed before the first run."""
import numpy as np
import pytest

from metalaudio_amd import nn
from tests import token_bits as bits
from tests.test_gpu_tokens import linear_case
from tests.token_refs import (EPS, HALF, TINY, attend, attention_tolerance, quantise, rmsnorm, rotary,
                              rounded, slot_of, window_seen)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return nn.AudioDevice(0)


@pytest.fixture(scope="module")
def stream(dev):
    return nn.Stream(dev)


def say(msg):
    print(f"[case] {msg}", flush=True)


def tensor(dev, x, dtype):
    return nn.Tensor.from_numpy(dev, x, dtype=dtype)


# -------------------------------------------------------------------------------- 8-bit linear
def linear(dev, stream, x, xs, w, out):
    layer = nn.Linear(dev, w.shape[1], w.shape[0], use_bias=False, precision="e4m3")
    layer.load_weights(w)
    y = nn.Tensor(dev, (x.shape[0], w.shape[0]), dtype=out)
    layer.forward_scaled(tensor(dev, x, "e4m3"), tensor(dev, xs, "f32"), y, stream=stream)
    stream.sync(60000)
    return y.to_numpy()


# rows of each of the kernel's forms: few, then tiles of 64 to 256
LINEARS = [(5, 256, 96), (200, 384, 320), (2500, 256, 1400), (3001, 384, 1240), (4000, 256, 4090)]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,K,N", LINEARS)
def test_linear_e4m3_sums_that_cancel(dev, stream, M, K, N, out):
    """Two products of 448 x 448 cancel beside small ones, near each other or far apart in the depth. All
    products are multiples of 1/16, and no sum of some of them reaches 2^19: 23 bits, so no fp32 sum is
    rounded, in whichever order, and only the row scales' roundings and the result's are left."""
    say(f"linear that cancels {M}x{K}x{N} {out}")
    rng = np.random.default_rng(M + K + N)
    for gap in (1, 5, 40, 130):
        x = rng.integers(-4, 5, (M, K)).astype(np.float32) / 4
        w = rng.integers(-4, 5, (N, K)).astype(np.float32) / 4
        at = int(rng.integers(0, K - gap))
        x[:, [at, at + gap]] = 448
        w[:, at], w[:, at + gap] = 448, -448
        wq, ws = quantise(w)
        np.testing.assert_array_equal(wq, w)
        want = (x.astype(np.float64) @ w.astype(np.float64).T) * ws
        got = linear(dev, stream, x, np.ones(M, np.float32), w, out).astype(np.float64)
        err = np.abs(got - want)
        tol = (4 * EPS + HALF[out] * (out == "bf16")) * np.abs(want)
        assert (err <= tol).all(), (f"gap {gap}: {(err > tol).mean():.3g} of the results off, the worst by "
                                    f"{err.max():.3g}, results up to {np.abs(want).max():.3g}")


@pytest.mark.parametrize("M,K,N", [(24, 2048, 4096), (300, 1536, 384), (2500, 384, 1400),
                                   (4000, 512, 4090)])
def test_linear_e4m3_distance(dev, stream, M, K, N):
    """fp32 output: one rounding of about 2^-25 rms of the running sum for each of the K / 16 matrix
    instructions behind one another, 3e-8 sqrt(K / 16) of the result where the sums grow evenly (their mean
    square is half the last one's), and as much again for the scales. bf16 output: the share of results that
    are not the nearest bf16 values is twice their distance over a step of 2^-8 to 2^-7, below 2^-7.5 / 4e-7 =
    7e-5 at that distance."""
    say(f"linear distance {M}x{K}x{N}")
    rng = np.random.default_rng(M + K)
    x, xs = quantise(rng.standard_normal((M, K)).astype(np.float32))
    w = (rng.standard_normal((N, K)) / np.sqrt(K)).astype(np.float32)
    wq, ws = quantise(w)
    want = (x.astype(np.float64) * xs[:, None]) @ (wq.astype(np.float64) * ws[:, None]).T
    got = linear(dev, stream, x, xs, w, "f32")
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    print(f"distance {off:.3g}")
    assert off <= 3e-8 * np.sqrt(K / 16) / np.sqrt(2) + 6e-8
    got = linear(dev, stream, x, xs, w, "bf16")
    share = (got != rounded(want, "bf16")).mean()
    print(f"not the nearest: {share:.3g}")
    assert share <= 3e-4


@pytest.mark.parametrize("M,K,N", [(3999, 256, 4089), (4090, 100, 4088), (10752, 128, 1536)])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_linear_e4m3_full_rounds(dev, stream, M, K, N, out):
    """Grids that fill the compute units with the largest tile, odd rows and columns, the residual in place."""
    say(f"linear full rounds {M}x{K}x{N} {out}")
    linear_case(dev, stream, M, K, N, act="swish", residual=True, out=out, in_place=True)


# ------------------------------------------------------------------------------------- RMS norm
@pytest.mark.parametrize("F", [8, 384, 1001, 1536, 5000])  # a wave a row, three passes, a workgroup a row
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("eps", [1e-5, 0.0, 1e-30])
def test_rmsnorm_sizes_whose_squares_leave_fp32(dev, stream, F, dtype, eps):
    """Finite rows whose squares overflow or underflow, ordinary ones between them."""
    say(f"rmsnorm sizes {F} {dtype} epsilon {eps}")
    rng = np.random.default_rng(F)
    sizes = [1.0, 1e25, 3e37, 1e-25, 1e19, 1e-20, 2.0 ** -120, 1.0, 1e-12, 1e-40]
    x = rng.standard_normal((len(sizes) + 2, F)).clip(-3, 3)
    x[:len(sizes)] *= np.array(sizes)[:, None]
    x[len(sizes)] *= 1e-3
    x[len(sizes), F // 2] = 1e30  # one large value takes all of the norm
    x[len(sizes) + 1] *= np.exp2(rng.integers(-60, 60, F))
    x = rounded(x, dtype)
    if dtype == "bf16":
        x[9] = 1  # bf16 rounds the smallest row to few bits, or to zeros
    w = (1 + 0.2 * rng.standard_normal(F)).astype(np.float32)
    layer = nn.RMSNorm(dev, F, eps)
    layer.load_parameters(w)
    rows = x.shape[0]
    y32, y8, s8 = nn.Tensor(dev, (rows, F)), nn.Tensor(dev, (rows, F), dtype="e4m3"), nn.Tensor(dev, (rows,))
    total = nn.Tensor(dev, (rows, F), dtype=dtype)
    layer.forward_residual(tensor(dev, x, dtype), None, y32, sum=total, stream=stream)
    layer.forward_residual(tensor(dev, x, dtype), None, y8, scales=s8, stream=stream)
    stream.sync(60000)
    np.testing.assert_array_equal(total.to_numpy(), x)
    want = rmsnorm(x, w, float(np.float32(eps)))
    # as in test_rmsnorm_residual; a power of two in between rounds nothing
    rel = (F / 64 + 24) * EPS
    got = y32.to_numpy().astype(np.float64)
    err = np.abs(got - want)
    bad = ~(err <= rel * np.abs(want) + 1.5e-45)  # the smallest results have a step of 2^-149
    assert not bad.any(), f"rows {sorted(set(np.argwhere(bad)[:, 0]))}: {got[bad][:3]} for {want[bad][:3]}"
    top = np.maximum(np.abs(want).max(-1), TINY)
    scales = s8.to_numpy().astype(np.float64)
    assert (np.abs(scales - top / 448) <= (rel + 4 * EPS) * top / 448).all()
    unit = np.abs(want) / scales[:, None]
    step = np.maximum(unit * HALF["e4m3"], 2.0 ** -10) * (1 + 1e-5) + 448 * 2 * rel + unit * 8 * EPS
    assert (np.abs(y8.to_numpy() * scales[:, None] - want) <= step * scales[:, None]).all()


def test_rmsnorm_of_zeros_without_epsilon(dev, stream):
    """0 / 0, and only in its row."""
    say("rmsnorm zeros")
    for F in (96, 1001):
        x = np.ones((3, F), np.float32)
        x[1] = 0
        y = nn.Tensor(dev, (3, F))
        nn.RMSNorm(dev, F, 0.0).forward_residual(tensor(dev, x, "f32"), None, y, stream=stream)
        stream.sync(60000)
        y = y.to_numpy()
        assert np.isnan(y[1]).all() and (y[[0, 2]] == 1).all()


# ------------------------------------------------------------------ window step at far positions
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("H,KV,T,left,sinks,back", [(2, 2, 5, 30, 20, 0), (4, 2, 16, 900, 33, 0),
                                                    (1, 1, 9, 700, 65, 3)])
def test_window_step_farthest_positions(dev, stream, H, KV, T, left, sinks, back, dtype):
    """Several new tokens up to position 2^31 - 2, sinks in sight, the keys over one workgroup and split."""
    say(f"step farthest {T} tokens {left} back {sinks} sinks {dtype}")
    hd, slots, p = 48, sinks + left + T + 2, 2 ** 31 - 1 - T - back
    layer = nn.WindowAttention(dev, H, hd, KV, left, 0, sinks)
    rng = np.random.default_rng(T)
    w = KV * hd
    kc, vc = (rounded(rng.standard_normal((1, slots, w)), dtype) for _ in "kv")
    q = rounded(rng.standard_normal((1, T, H * hd)), dtype)
    k, v = (rounded(rng.standard_normal((1, T, w)), dtype) for _ in "kv")
    kt, vt = tensor(dev, kc, dtype), tensor(dev, vc, dtype)
    out = nn.Tensor(dev, q.shape, dtype=dtype)
    layer.step(tensor(dev, q, dtype), tensor(dev, k, dtype), tensor(dev, v, dtype),
               tensor(dev, np.array([p]), "i32"), kt, vt, out, stream=stream)
    stream.sync(60000)
    tokens = list(range(sinks)) + list(range(p - left, p))
    at = [slot_of(i, sinks, slots) for i in tokens]
    kk, vv = np.concatenate([kc[0, at], k[0]]), np.concatenate([vc[0, at], v[0]])
    key = np.array(tokens + list(range(p, p + T)))[None]
    mine = np.arange(p, p + T)[:, None]
    seen = (key <= mine) & ((key >= mine - left) | (key < sinks))
    want, spread, size = attend(q[0], kk, vv, seen, H, KV, hd ** -0.5)
    err = np.abs(out.to_numpy()[0] - want)
    assert (err <= attention_tolerance(spread, size, hd, left + 1 + sinks, dtype)).all()
    for i in range(T):
        kc[0, slot_of(p + i, sinks, slots)], vc[0, slot_of(p + i, sinks, slots)] = k[0, i], v[0, i]
    np.testing.assert_array_equal(kt.to_numpy(), kc)
    np.testing.assert_array_equal(vt.to_numpy(), vc)


# ------------------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize("hd,inter", [(64, False), (64, True), (6, False)])
@pytest.mark.parametrize("origin", [0, 900001])
def test_rotary_angles_keep_their_bits(dev, stream, hd, inter, origin):
    """Pairs (1, 0) turn into their cosine and sine: two roundings each (the function's, the remainder's
    term), about 0.42 half steps rms of values of all sizes or 2.5e-8, together 3.5e-8, and a fifth more
    for a function that is off by somewhat above half a step. An angle rounded to fp32 adds 4.1e-8."""
    say(f"rotary bits hd {hd} interleaved {inter} from {origin}")
    S, base = 4000, 3.0  # rates of all the pairs turn far
    x = np.zeros((S, hd), np.float32)
    x[:, 0::2] = 1 if inter else 0
    x[:, :hd // 2] = x[:, :hd // 2] if inter else 1
    pos = (origin + np.arange(S))[:, None]
    y = nn.Tensor(dev, (S, hd))
    nn.Rotary(dev, hd, [hd], base=base, interleaved=inter).forward(
        tensor(dev, x, "f32"), None, tensor(dev, pos, "i32"), y, stream=stream)
    stream.sync(60000)
    want = rotary(x[None], pos, 1, hd, [hd], base, inter)[0]
    off = np.linalg.norm(y.to_numpy() - want) / np.linalg.norm(want)
    print(f"distance {off:.3g}")
    assert off <= 4.2e-8


# -------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,S,H,KV,hd,left,right,sinks", [
    (2, 1345, 8, 8, 48, 168, 168, 4), (1, 700, 2, 1, 64, 300, 1, 129), (5, 1030, 8, 8, 48, 70, 0, 3),
    (3, 1025, 16, 16, 128, 64, 64, 2), (1, 2500, 2, 2, 48, 1000, 0, 5), (2, 130, 4, 2, 32, 16, 16, 4),
    (6, 901, 8, 2, 64, 200, 5, 70)])
def test_window_attention_distance(dev, stream, B, S, H, KV, hd, left, right, sinks, dtype):
    """The largest distance of a sequence from 64 bits, in every way that a call is cut."""
    say(f"window distance {B}x{S} heads {H}/{KV} hd {hd} {dtype}")
    rng = np.random.default_rng(S)
    q, k = (rounded(rng.standard_normal((B, S, n * hd)) * 1.3, dtype) for n in (H, KV))
    v = rounded(rng.standard_normal((B, S, KV * hd)), dtype)
    o = nn.Tensor(dev, q.shape, dtype=dtype)
    nn.WindowAttention(dev, H, hd, KV, left, right, sinks).forward(
        *(tensor(dev, x, dtype) for x in (q, k, v)), o, stream=stream)
    stream.sync(60000)
    got, seen = o.to_numpy(), window_seen(S, left, right, sinks)
    off = max(bits.distance(got[b], attend(q[b], k[b], v[b], seen, H, KV, hd ** -0.5)[0]) for b in range(B))
    print(f"distance {off:.3g}")
    assert off <= (bits.ATTENTION_F32 if dtype == "f32" else bits.ATTENTION_BF16)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,H,KV,hd,left,sinks", [(3, 1, 8, 8, 48, 511, 4), (1, 5, 8, 2, 64, 900, 4),
                                                    (2, 16, 4, 4, 128, 100, 33)])
def test_window_step_distance(dev, stream, B, T, H, KV, hd, left, sinks, dtype):
    """Steps keep their probabilities in fp32 whatever the tensors' type."""
    say(f"step distance {B}x{T} heads {H}/{KV} hd {hd} {dtype}")
    rng = np.random.default_rng(hd)
    slots, p = sinks + left + T, 3000
    kc, vc, k, v = (rounded(rng.standard_normal((B, n, KV * hd)) * s, dtype)
                    for n, s in ((slots, 1.3), (slots, 1), (T, 1.3), (T, 1)))
    q = rounded(rng.standard_normal((B, T, H * hd)) * 1.3, dtype)
    o = nn.Tensor(dev, q.shape, dtype=dtype)
    nn.WindowAttention(dev, H, hd, KV, left, 0, sinks).step(
        *(tensor(dev, x, dtype) for x in (q, k, v)), tensor(dev, np.full(B, p), "i32"),
        tensor(dev, kc, dtype), tensor(dev, vc, dtype), o, stream=stream)
    stream.sync(60000)
    tokens = list(range(sinks)) + list(range(p - left, p))
    at = [slot_of(i, sinks, slots) for i in tokens]
    key = np.array(tokens + list(range(p, p + T)))[None]
    mine = np.arange(p, p + T)[:, None]
    seen = (key <= mine) & ((key >= mine - left) | (key < sinks))
    got = o.to_numpy()
    off = max(bits.distance(got[b], attend(q[b], np.concatenate([kc[b, at], k[b]]),
                                           np.concatenate([vc[b, at], v[b]]), seen, H, KV, hd ** -0.5)[0])
              for b in range(B))
    print(f"distance {off:.3g}")
    assert off <= (bits.ATTENTION_F32 if dtype == "f32" else bits.STEP_BF16)


BAD = [("k", np.inf), ("k", -np.inf), ("k", 3e38), ("k", -3e38), ("v", np.inf), ("v", 3e38), ("v", np.nan)]


def sighted(got, want, tol, what):
    """Infinities and NaN where the formula has them, the rest within the tolerance."""
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=what)
    np.testing.assert_array_equal(got[np.isinf(want)], want[np.isinf(want)], err_msg=what)
    fine = np.isfinite(want)
    assert (np.abs(got[fine] - want[fine]) <= tol[fine]).all(), what


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("what,bad", BAD)
@pytest.mark.parametrize("B,H", [(1, 1), (6, 8)])  # one or four key groups a workgroup
def test_window_attention_of_a_value_in_sight(dev, stream, B, H, what, bad, dtype):
    """The queries that see a key (or value) with an infinite, NaN or huge entry: a score of -infinity
    has weight 0, one of +infinity or NaN leaves NaN, a huge one takes all or nothing. The queries' entry
    beside the huge one is below 1, so that no sum of products leaves fp32."""
    say(f"window in sight of {what} {bad} {dtype} {B} x {H}")
    S, hd, left, sinks, at = 700, 48, 150, 2, 301
    rng = np.random.default_rng(61)
    q = rng.standard_normal((B, S, H * hd))
    q[..., 5::hd] = rng.uniform(0.05, 0.9, (B, S, H)) * rng.choice([-1, 1], (B, S, H))
    q, k, v = (rounded(x, dtype) for x in (q, *(rng.standard_normal((2, B, S, H * hd)))))
    {"k": k, "v": v}[what][:, at, 5::hd] = rounded(np.float32(bad), dtype)
    o = nn.Tensor(dev, q.shape, dtype=dtype)
    nn.WindowAttention(dev, H, hd, window_left=left, sinks=sinks).forward(
        *(tensor(dev, x, dtype) for x in (q, k, v)), o, stream=stream)
    stream.sync(60000)
    got = o.to_numpy()
    rows = slice(at - 20, at + left + 20)
    seen = window_seen(S, left, 0, sinks)[rows]
    with np.errstate(invalid="ignore"):
        for b in (0, B - 1):
            want, spread, size = attend(q[b, rows], k[b], v[b], seen, H, H, hd ** -0.5)
            # a huge score takes all: its own size is no error of the others
            spread = np.where(np.isfinite(spread) & (spread < 1e3), spread, 0) + 10
            sighted(got[b, rows], want, attention_tolerance(spread, np.abs(size), hd, S, dtype), f"sequence {b}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("what,bad", BAD)
@pytest.mark.parametrize("left", [150, 1000])  # one workgroup a head, or its keys split
def test_window_step_of_a_value_in_sight(dev, stream, what, bad, left, dtype):
    say(f"step in sight of {what} {bad} {dtype} {left} back")
    hd, H, T, sinks = 48, 2, 6, 2
    slots, p = sinks + left + T, 5 * left
    at = p - left + 3  # seen by the first four of the six tokens
    rng = np.random.default_rng(62)
    q = rng.standard_normal((1, T, H * hd))
    q[..., 5::hd] = rng.uniform(0.05, 0.9, (1, T, H)) * rng.choice([-1, 1], (1, T, H))
    q = rounded(q, dtype)
    kc, vc, k, v = (rounded(rng.standard_normal((1, n, H * hd)), dtype) for n in (slots, slots, T, T))
    {"k": kc, "v": vc}[what][0, slot_of(at, sinks, slots), 5::hd] = rounded(np.float32(bad), dtype)
    o = nn.Tensor(dev, q.shape, dtype=dtype)
    nn.WindowAttention(dev, H, hd, window_left=left, sinks=sinks).step(
        *(tensor(dev, x, dtype) for x in (q, k, v)), tensor(dev, np.array([p]), "i32"),
        tensor(dev, kc, dtype), tensor(dev, vc, dtype), o, stream=stream)
    stream.sync(60000)
    tokens = list(range(sinks)) + list(range(p - left, p))
    slot = [slot_of(i, sinks, slots) for i in tokens]
    key = np.array(tokens + list(range(p, p + T)))[None]
    mine = np.arange(p, p + T)[:, None]
    seen = (key <= mine) & ((key >= mine - left) | (key < sinks))
    with np.errstate(invalid="ignore"):
        want, spread, size = attend(q[0], np.concatenate([kc[0, slot], k[0]]), np.concatenate([vc[0, slot], v[0]]),
                                    seen, H, H, hd ** -0.5)
    spread = np.where(np.isfinite(spread) & (spread < 1e3), spread, 0) + 10
    sighted(o.to_numpy()[0], want, attention_tolerance(spread, np.abs(size), hd, left + 3, dtype), "step")
