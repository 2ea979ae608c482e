"""The bits that the decoder's operators hold, through the C ABI against 64-bit references.
Tolerances count roundings (token_refs.py, decoder_refs.py) and were fixed before the first run."""
import numpy as np
import pytest

from metalaudio_amd import nn
from tests import token_bits as bits
from tests.decoder_refs import (blocks_of, held_rows, held_tolerance, linear_blocks, memory, quantise_blocks,
                                quantise_tiles, values_of)
from tests.test_gpu_tokens import check, tensor
from tests.token_refs import EPS, HALF, attend, rounded, slot_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return nn.AudioDevice(0)


@pytest.fixture(scope="module")
def stream(dev):
    return nn.Stream(dev)


def say(msg):
    print(f"[case] {msg}", flush=True)


# ------------------------------------------------------- probabilities of calls in bf16, few rows
def check_probabilities(got, want, spread, size, hd, keys, what):
    """The sums' bounds are those of f32 calls; the probabilities are two bf16 values, of which the second is off by
    a half step of what the first one leaves, 2^-8 of 2^-8; the result is rounded once. Values of both signs cancel,
    so that probabilities of one bf16 value (2^-8 of the sum of magnitudes) miss these bounds by far."""
    tol = held_tolerance(spread, size, hd, keys, "f32") + HALF["bf16"] ** 2 * size
    check(got, want, tol + HALF["bf16"] * (np.abs(want) + tol), what)


@pytest.mark.parametrize("B,T,H,KV,hd,left,sinks", [
    (3, 1, 8, 2, 64, 23, 2), (2, 16, 8, 2, 64, 1023, 4), (16, 1, 16, 4, 64, 2100, 4), (1, 1, 4, 4, 32, 700, 0),
    (2, 3, 6, 3, 96, 300, 1), (2, 1, 4, 1, 128, 90, 0), (1, 40, 2, 1, 48, 64, 3)])
def test_window_step_held_probabilities(dev, stream, B, T, H, KV, hd, left, sinks):
    say(f"8-bit step bits {B}x{T} heads {H}/{KV} hd {hd} left {left} sinks {sinks}")
    rng = np.random.default_rng(B + T + hd)
    slots, w, p0 = sinks + left + T, KV * hd, 3 * (sinks + left) + 5
    old = [held_rows(1.2 * rng.standard_normal((B, slots, w)), KV) for _ in "kv"]
    q = rounded(1.3 * rng.standard_normal((B, T, H * hd)), "bf16")
    new = [rounded(1.2 * rng.standard_normal((B, T, w)), "bf16") for _ in "kv"]
    out = nn.Tensor(dev, q.shape, dtype="bf16")
    nn.WindowAttention(dev, H, hd, KV, left, 0, sinks).step(
        tensor(dev, q, "bf16"), *(tensor(dev, x, "bf16") for x in new), tensor(dev, np.full(B, p0), "i32"),
        *(tensor(dev, x, "e4m3") for x, _ in old), out, None, stream, *(tensor(dev, s, "f32") for _, s in old))
    stream.sync(60000)
    got, wants = out.to_numpy(), np.empty(q.shape)
    told = list(range(sinks)) + list(range(p0 - left, p0 + T))
    at = [slot_of(p, sinks, slots) for p in told[:len(told) - T]]
    mine, key = np.arange(p0, p0 + T)[:, None], np.array(told)[None]
    seen = (key <= mine) & ((key >= mine - left) | (key < sinks))
    for b in range(B):
        k, v = (np.concatenate([values_of(x[b, at], s[b, at]), values_of(*held_rows(n[b], KV))])
                for (x, s), n in zip(old, new))
        wants[b], spread, size = attend(q[b], k, v, seen, H, KV, hd ** -0.5)
        check_probabilities(got[b], wants[b], spread, size, hd, len(told), f"stream {b}")
    assert bits.distance(got, wants) <= bits.STEP_BF16


@pytest.mark.parametrize("held", [False, True])
@pytest.mark.parametrize("B,T,S,H,KV,hd", [
    (2, 1, 31, 8, 8, 48), (64, 1, 700, 16, 4, 64), (1, 1, 4100, 4, 2, 64), (3, 4, 333, 8, 2, 128), (2, 16, 90, 5, 5, 32),
    (1, 61, 512, 8, 8, 96), (4, 5, 1000, 6, 2, 72)])
def test_memory_of_few_rows_probabilities(dev, stream, B, T, S, H, KV, hd, held):
    say(f"memory bits {B}x{T} on {S} heads {H}/{KV} hd {hd} held {held}")
    rng = np.random.default_rng(B + T + S)
    q = rounded(1.3 * rng.standard_normal((B, T, H * hd)), "bf16")
    kv = [rounded(1.2 * rng.standard_normal((B, S, KV * hd)), "bf16") for _ in "kv"]
    rows, scales = [tensor(dev, x, "bf16") for x in kv], [None, None]
    if held:
        h = [held_rows(x, KV) for x in kv]
        kv = [values_of(*x) for x in h]
        rows, scales = [tensor(dev, x, "e4m3") for x, _ in h], [tensor(dev, s, "f32") for _, s in h]
    out = nn.Tensor(dev, q.shape, dtype="bf16")
    nn.MemoryAttention(dev, H, hd, KV).forward(tensor(dev, q, "bf16"), *rows, out, None, None, *scales, stream=stream)
    stream.sync(60000)
    got, wants = out.to_numpy(), np.empty(q.shape)
    for b in range(B):
        wants[b], spread, size = memory(q[b], kv[0][b], kv[1][b], H, KV, hd ** -0.5)
        check_probabilities(got[b], wants[b], spread, size, hd, S + 8, f"sequence {b}")
    assert bits.distance(got, wants) <= bits.STEP_BF16


# ------------------------------------------------------------------ the linear layer, in blocks
# (rows, outputs) of each of the kernel's forms: few rows, few and more, tiles of 64 and 128 square, of 128 x 256
LINEARS = [(5, 96), (64, 320), (1000, 400), (2500, 1240), (4000, 4090)]


def linear_blocks_of(dev, stream, x, w, out="f32"):
    layer = nn.Linear(dev, w.shape[1], w.shape[0], use_bias=False, precision="e4m3_block")
    layer.load_weights(w)
    y = nn.Tensor(dev, (x.shape[0], w.shape[0]), dtype=out)
    layer.forward_scaled(tensor(dev, x, "f32"), None, y, stream=stream)
    stream.sync(60000)
    return y.to_numpy()


def check_linear(got, x, w, what):
    """As for ordinary sizes (1.5 half steps of the running sum an addition, a few a block for its scales), and half of
    fp32's smallest step a block where sums are that small."""
    K = x.shape[1]
    want, mass = linear_blocks(*quantise_blocks(x), *quantise_tiles(w), None)
    check(got, want, (1.5 * K + 4 * blocks_of(K) + 8) * EPS * mass + blocks_of(K) * 2.0 ** -150, what)


@pytest.mark.parametrize("xsize,wsize", [(1e-20, 1e-17), (2e-17, 1e-20), (1e-19, 1e-19), (1e-28, 1e-9), (1e-7, 1e-30),
                                         (1e18, 1e-18), (1e16, 1e15)])
@pytest.mark.parametrize("M,N", LINEARS)
def test_linear_blocks_scales_of_one_sign(dev, stream, M, N, xsize, wsize):
    """Rows and weights that are both small: their scales' product is no normal number, the results are. And both large."""
    say(f"linear blocks {M} rows {N} outputs sizes {xsize} {wsize}")
    rng = np.random.default_rng(M)
    x = (rng.standard_normal((M, 300)) * np.exp(rng.standard_normal((M, 1)))).astype(np.float32) * np.float32(xsize)
    x[1::3] /= np.float32(xsize)  # ordinary rows between them, whose scales' products are normal numbers
    w = rng.standard_normal((N, 300)).astype(np.float32) * np.float32(wsize)
    check_linear(linear_blocks_of(dev, stream, x, w), x, w, "both small or large")


@pytest.mark.parametrize("M,N", LINEARS)
def test_linear_blocks_beside_a_huge_weight(dev, stream, M, N):
    """One weight near fp32's largest: it takes the bits of its own 128 x 128 values and of no others, however small what they are
    multiplied by. A row of zeros gives zeros, also where the product of its weights' scale and the rows' is infinite."""
    say(f"linear blocks {M} rows {N} outputs, one weight of 1e38")
    rng = np.random.default_rng(M + 1)
    x = (rng.standard_normal((M, 400)) * 1e-6).astype(np.float32)
    w = (rng.standard_normal((N, 400)) / 20).astype(np.float32)
    w[N - 3, 140] = 1e38
    w[N - 2] = 0
    x[2] = 1e30
    x[2, 140] = 0
    got = linear_blocks_of(dev, stream, x, w)
    assert (got[:, N - 2] == 0).all()
    check_linear(got, x, w, "beside 1e38")


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("K", [128, 384])
@pytest.mark.parametrize("M,N", LINEARS)
def test_linear_blocks_sums_that_cancel_within_a_block(dev, stream, M, N, K, out):
    """Two products of 448 x 448 cancel beside small ones of the same block. All products are multiples of 1/16 and no sum of
    some of them reaches 2^19, so no block's sum is rounded; times the block's scale, within some half steps of 1, it is by a
    half step, and so is each addition of another block's, which is no larger than the sums of the magnitudes."""
    say(f"linear blocks that cancel in a block {M}x{K}x{N} {out}")
    rng = np.random.default_rng(M + K + N)
    for gap in (1, 7, 40, 100):
        x = rng.integers(-4, 5, (M, K)).astype(np.float32) / 4
        w = rng.integers(-4, 5, (N, K)).astype(np.float32) / 4
        at = int(rng.integers(0, K // 128)) * 128 + int(rng.integers(0, 128 - gap))
        w[::128, ::128] = 448  # every block's largest value
        x[:, ::128] = 0
        x[:, [at, at + gap]] = 448
        w[:, at], w[:, at + gap] = 448, -448
        wq, ws = quantise_tiles(w)
        np.testing.assert_array_equal(wq, w)
        assert (ws == ws[0, 0]).all()
        layer = nn.Linear(dev, K, N, use_bias=False, precision="e4m3_block")
        layer.load_weights(w)
        y = nn.Tensor(dev, (M, N), dtype=out)
        layer.forward_scaled(tensor(dev, x, "e4m3"), tensor(dev, np.ones((M, K // 128)), "f32"), y, stream=stream)
        stream.sync(60000)
        sums = [x[:, i:i + 128].astype(np.float64) @ w[:, i:i + 128].astype(np.float64).T for i in range(0, K, 128)]
        want = sum(sums) * float(ws[0, 0])
        tol = 2 * EPS * sum(np.abs(s) for s in sums) * (2 if K > 128 else 1)
        check(y.to_numpy(), want, tol + HALF[out] * (out == "bf16") * (np.abs(want) + tol), f"gap {gap}")
