"""The bits that the token operators hold, through the C ABI against 64-bit references: sums of products
that cancel, and distances in the 2-norm, which the bounds of single elements are too wide to see.
Tolerances count roundings (token_refs.py) and were fixed before the first run."""
import numpy as np
import pytest

from metalaudio_amd import nn
from tests.test_gpu_tokens import linear_case
from tests.token_refs import EPS, HALF, quantise, rounded

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
