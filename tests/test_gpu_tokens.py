"""The token operators through the C ABI against 64-bit references: RMS norm with residual and 8-bit
output, the 8-bit linear layer, rotary positions, window attention and its step on rolling caches.
Tolerances count roundings (token_refs.py) and were fixed before the first run."""
import ctypes as C

import numpy as np
import pytest

from metalaudio_amd import nn
from tests.token_refs import (EPS, HALF, TINY, attend, attention_tolerance, quantise, rmsnorm, rotary,
                              rounded, row_scales, slot_of, window_seen)

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


def check(got, want, tol, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    err = np.abs(got - want)
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(err / tol):.3g} times "
                           f"the tolerance, first at {np.argwhere(bad)[0]}: {got[bad][0]} for {want[bad][0]}")


def refuses(code, call):
    with pytest.raises(nn.MNNError) as e:
        call()
    assert e.value.name == code, e.value


# ------------------------------------------------------------------------------------- RMS norm
def norm_case(dev, stream, rows, F, dtype, residual, out, seed=0, alias=None, data=None):
    rng = np.random.default_rng(seed + rows * 7 + F)
    x = rng.standard_normal((rows, F)) * np.exp(rng.standard_normal((rows, 1)))
    r = rng.standard_normal((rows, F)) * 2 if residual else None
    if data is not None:
        x, r = data, None
    w = (1 + 0.2 * rng.standard_normal(F)).astype(np.float32)
    x = rounded(x, dtype)
    r = rounded(r, dtype) if r is not None else None
    layer = nn.RMSNorm(dev, F, 1e-5)
    layer.load_parameters(w)
    xt, rt = tensor(dev, x, dtype), tensor(dev, r, dtype) if r is not None else None
    yt = nn.Tensor(dev, (rows, F), dtype=out)
    st = nn.Tensor(dev, (rows,)) if out == "e4m3" else None
    ht = xt if alias == "x" else rt if alias == "r" else nn.Tensor(dev, (rows, F), dtype=dtype)
    layer.forward_residual(xt, rt, yt, sum=ht, scales=st, stream=stream)
    stream.sync(60000)
    h32 = x + r if r is not None else x  # one fp32 addition
    return x, w, h32, ht.to_numpy(), yt.to_numpy(), st.to_numpy() if st else None


@pytest.mark.parametrize("rows,F,dtype,residual,out", [
    (1, 8, "f32", True, "e4m3"), (8, 512, "f32", True, "e4m3"), (5, 384, "bf16", True, "e4m3"),
    (67, 257, "f32", True, "e4m3"), (3, 1000, "bf16", True, "bf16"), (130, 48, "bf16", False, "e4m3"),
    (33, 2048, "bf16", True, "e4m3"), (9, 4096, "f32", True, "f32"), (7, 5000, "bf16", True, "e4m3"),
    (4, 1, "f32", False, "e4m3"), (2, 20004, "f32", True, "e4m3"), (301, 384, "f32", False, "bf16"),
    (1001, 768, "bf16", True, "f32"), (2500, 384, "bf16", True, "e4m3"), (70, 1536, "f32", True, "e4m3"),
    (12, 3000, "bf16", True, "e4m3"), (5, 4104, "bf16", True, "e4m3")])
def test_rmsnorm_residual(dev, stream, rows, F, dtype, residual, out):
    say(f"rmsnorm {rows}x{F} {dtype} residual {residual} -> {out}")
    x, w, h, gh, gy, gs = norm_case(dev, stream, rows, F, dtype, residual, out)
    np.testing.assert_array_equal(gh, rounded(h, dtype))
    y = rmsnorm(h.astype(np.float64), w, 1e-5)
    # h one rounding, the sum of squares at most a half step an addition in each lane's F / 64 terms and
    # the tree, half of it in the root; division, root, two products
    rel = (F / 64 + 24) * EPS
    if out != "e4m3":
        return check(gy, y, (rel + HALF[out] * (out != "f32")) * np.abs(y) + 1e-37, "out")
    want, _ = row_scales(y.astype(np.float32))
    check(gs, np.maximum(np.abs(y).max(-1), TINY) / 448, (rel + 4 * EPS) * want, "scales")
    unit = np.abs(y) / want[:, None].astype(np.float64)
    step = np.maximum(unit * HALF["e4m3"], 2.0 ** -10)  # half a step; e4m3's smallest one is 2^-9
    check(gy * gs[:, None].astype(np.float64), y,
          (step * (1 + 1e-5) + unit * (rel + 8 * EPS) + 448 * 2 * rel) * want[:, None], "out")


@pytest.mark.parametrize("alias", ["x", "r"])
@pytest.mark.parametrize("rows,F,dtype", [(40, 384, "bf16"), (6, 1001, "f32"), (300, 512, "f32")])
def test_rmsnorm_sum_in_place(dev, stream, alias, rows, F, dtype):
    say(f"rmsnorm sum is {alias} {rows}x{F} {dtype}")
    plain = norm_case(dev, stream, rows, F, dtype, True, "e4m3")
    again = norm_case(dev, stream, rows, F, dtype, True, "e4m3", alias=alias)
    for a, b in zip(plain[3:], again[3:]):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("F", [384, 1001])
def test_rmsnorm_rows_of_zeros_and_not_finite(dev, stream, F):
    say(f"rmsnorm odd rows {F}")
    x = np.random.default_rng(3).standard_normal((6, F)).astype(np.float32)
    x[1] = 0
    x[2, 5] = np.nan
    x[3, F - 1] = np.inf
    x[4] *= 1e-30
    _, w, h, gh, gy, gs = norm_case(dev, stream, 6, F, "f32", False, "e4m3", data=x)
    assert (gy[1] == 0).all() and gs[1] == TINY * np.float32(1 / 448)
    assert not np.isfinite(gy[2] * gs[2]).any() and np.isnan(gy[3, F - 1] * gs[3])
    for i in (0, 4, 5):
        y = rmsnorm(h[i], w, 1e-5)
        assert np.abs(gy[i] * gs[i].astype(np.float64) - y).max() <= np.abs(y).max() * HALF["e4m3"] * 1.01


def test_rmsnorm_layer_forward_and_model(dev, stream):
    """The one-input forward (f32 and bf16 input, f32 output, also in place) and a model of RMSNorm and
    an 8-bit linear."""
    say("rmsnorm forward, sequential")
    rng = np.random.default_rng(4)
    x = rng.standard_normal((3, 21, 96)).astype(np.float32)
    w = (1 + 0.2 * rng.standard_normal(96)).astype(np.float32)
    norm = nn.RMSNorm(dev, 96)
    norm.load_parameters(w)
    for dtype in ("f32", "bf16"):
        y = rmsnorm(rounded(x, dtype), w, 1e-5)
        got = norm(tensor(dev, x, dtype), stream)
        stream.sync(60000)
        check(got.to_numpy(), y, 32 * EPS * np.abs(y) + 1e-37, dtype)
    xt = tensor(dev, x, "f32")
    norm.forward(xt, xt, stream)
    lin = nn.Linear(dev, 96, 40, precision="e4m3", activation="relu")
    W = rng.standard_normal((40, 96)).astype(np.float32) / 10
    lin.load_weights(W, np.zeros(40, np.float32))
    want = lin(xt, stream)
    seq = nn.Sequential(dev)
    seq.add(norm)
    seq.add(lin)
    seq.build()
    got = seq.forward(tensor(dev, x, "f32"), stream)
    stream.sync(60000)
    np.testing.assert_array_equal(got.to_numpy(), want.to_numpy())


def test_rmsnorm_refusals(dev, stream):
    say("rmsnorm refusals")
    layer = nn.RMSNorm(dev, 64)
    T = lambda shape, dtype="f32": nn.Tensor(dev, shape, dtype=dtype)  # noqa: E731
    x, r, y, q, s = T((4, 64)), T((4, 64)), T((4, 64)), T((4, 64), "e4m3"), T((4,))
    f = layer.forward_residual
    arg, size = "MNN_ERR_INVALID_ARGUMENT", "MNN_ERR_BUFFER_SIZE_MISMATCH"
    refuses("MNN_ERR_INVALID_CONFIGURATION", lambda: nn.RMSNorm(dev, 0))
    refuses("MNN_ERR_INVALID_CONFIGURATION", lambda: nn.RMSNorm(dev, 8, float("nan")))
    refuses("MNN_ERR_SHAPE_MISMATCH", lambda: f(T((4, 63)), None, T((4, 63))))
    refuses(arg, lambda: f(x, T((4, 64), "bf16"), y))
    refuses(arg, lambda: f(x, r, y, sum=T((4, 64), "bf16")))
    refuses(size, lambda: f(x, T((3, 64)), y))
    refuses(size, lambda: f(x, r, T((4, 65))))
    refuses(size, lambda: f(x, r, y, sum=T((1, 64))))
    refuses(arg, lambda: f(x, r, q))
    refuses(arg, lambda: f(x, r, y, scales=s))
    refuses(size, lambda: f(x, r, q, scales=T((3,))))
    refuses(arg, lambda: f(x, r, q, scales=T((4,), "i32")))
    refuses(arg, lambda: f(q, None, y))
    refuses(arg, lambda: f(x, r, T((4, 64), "i32")))
    refuses(arg, lambda: f(x, r, y, sum=y))
    x1, s1 = T((4, 1)), T((4, 1))
    one = nn.RMSNorm(dev, 1)
    refuses(arg, lambda: one.forward_residual(x1, None, T((4, 1), "e4m3"), scales=x1))
    refuses(arg, lambda: one.forward_residual(x1, None, T((4, 1), "e4m3"), sum=s1, scales=s1))
    refuses(arg, lambda: nn.Linear(dev, 64, 64).forward_scaled(x, None, y))
    refuses(arg, lambda: nn.RMSNorm.forward_residual(nn.LayerNorm(dev, 64), x, r, y))
    refuses(arg, lambda: layer.forward(T((4, 64), "i32"), y))
    empty = T((0, 64))
    f(empty, None, T((0, 64)), stream=stream)  # no rows: nothing to do


# -------------------------------------------------------------------------------- 8-bit linear
ACTS = {"none": lambda y: y, "relu": lambda y: np.maximum(y, 0),
        "leaky_relu": lambda y: np.where(y >= 0, y, 0.01 * y),
        "gelu": lambda y: y / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (y + 0.044715 * y ** 3))),
        "swish": lambda y: y / (1 + np.exp(-y)), "sigmoid": lambda y: 1 / (1 + np.exp(-y)),
        "tanh": np.tanh}


def linear_case(dev, stream, M, K, N, act="none", residual=False, inp="e4m3", out="f32", bias=True,
                in_place=False, seed=0):
    rng = np.random.default_rng(seed + M + 3 * K + 7 * N)
    x = (rng.standard_normal((M, K)) * np.exp(0.5 * rng.standard_normal((M, 1)))).astype(np.float32)
    w = (rng.standard_normal((N, K)) / np.sqrt(K)).astype(np.float32)
    b = (0.1 * rng.standard_normal(N)).astype(np.float32)
    r = rounded(rng.standard_normal((M, N)), out) if residual else None
    layer = nn.Linear(dev, K, N, use_bias=bias, activation=act, precision="e4m3")
    layer.load_weights(w, b if bias else None)
    if inp == "e4m3":
        xq, xs = quantise(x)
        xt, st = tensor(dev, xq, "e4m3"), tensor(dev, xs, "f32")
    else:
        xq, xs = quantise(rounded(x, inp))
        xt, st = tensor(dev, x, inp), None
    rt = tensor(dev, r, out) if residual else None
    yt = rt if in_place else nn.Tensor(dev, (M, N), dtype=out)
    layer.forward_scaled(xt, st, yt, residual=rt, stream=stream)
    stream.sync(60000)
    wq, ws = quantise(w)
    xd, wd = xq.astype(np.float64) * xs[:, None], wq.astype(np.float64) * ws[:, None]
    y = xd @ wd.T + (b if bias else 0)
    mass = np.abs(xd) @ np.abs(wd).T
    # each addition rounds by at most 1.5 * 2^-24 of the running sum (matrix instructions); scales, bias
    # and activation a few half steps; exp's argument up to 30 half steps
    tol = (1.5 * K + 4) * EPS * mass + 4 * EPS * (np.abs(y) + 0.2)
    want = ACTS[act](y)
    tol = 1.13 * tol + (0 if act in ("none", "relu", "leaky_relu") else 64 * EPS * (np.abs(want) + 1e-3))
    if residual:
        want = want + r
        tol = tol + EPS * np.abs(want)
    if out == "bf16":
        tol = tol + HALF["bf16"] * np.abs(want)
    check(yt.to_numpy(), want, tol + 1e-37, f"{M}x{K}x{N}")


@pytest.mark.parametrize("M,K,N,kw", [
    (1, 128, 16, {}), (1, 512, 2048, {"act": "gelu", "out": "bf16"}), (5, 512, 2048, {"out": "bf16"}),
    (3, 1, 1, {}), (2, 100, 7, {"residual": True}), (17, 320, 200, {"act": "relu"}),
    (16, 2048, 512, {"residual": True}), (33, 1000, 777, {"act": "swish", "out": "bf16"}),
    (64, 384, 384, {"residual": True, "out": "bf16"}), (67, 384, 1536, {"act": "gelu"}),
    (129, 1536, 384, {"residual": True}), (257, 512, 513, {"act": "tanh"}), (700, 384, 1152, {}),
    (1344, 384, 1536, {"act": "gelu", "out": "bf16"}), (2688, 1536, 384, {"residual": True}),
    (200, 2048, 2048, {"act": "leaky_relu", "residual": True}), (130, 640, 130, {"act": "sigmoid"}),
    (1000, 256, 260, {"bias": False, "residual": True, "out": "bf16"}), (511, 896, 1026, {"out": "bf16"}),
    (4099, 256, 4104, {"residual": True, "out": "bf16"}), (4097, 384, 4100, {"act": "relu"})])
def test_linear_e4m3(dev, stream, M, K, N, kw):
    say(f"linear e4m3 {M}x{K}x{N} {kw}")
    linear_case(dev, stream, M, K, N, **kw)


@pytest.mark.parametrize("M,K,N", [(3001, 256, 1240), (3007, 640, 1237), (2100, 256, 2056), (2099, 130, 2055)])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_linear_e4m3_middle_sizes(dev, stream, M, K, N, out):
    """Between the square tiles' sizes, rows and columns that no tile divides, the residual in place."""
    say(f"linear e4m3 middle {M}x{K}x{N} {out}")
    linear_case(dev, stream, M, K, N, act="swish", residual=True, out=out, in_place=True)


@pytest.mark.parametrize("M,K,N,inp,out", [(1, 384, 96, "f32", "f32"), (9, 257, 64, "bf16", "bf16"),
                                           (300, 512, 300, "bf16", "f32"), (45, 1000, 33, "f32", "bf16")])
def test_linear_e4m3_rounds_wider_input(dev, stream, M, K, N, inp, out):
    say(f"linear e4m3 from {inp} {M}x{K}x{N}")
    linear_case(dev, stream, M, K, N, inp=inp, out=out, residual=True)


@pytest.mark.parametrize("M,K,N,out", [(4, 256, 64, "f32"), (300, 384, 384, "bf16"), (50, 100, 77, "f32")])
def test_linear_e4m3_residual_in_place(dev, stream, M, K, N, out):
    say(f"linear e4m3 in place {M}x{K}x{N} {out}")
    linear_case(dev, stream, M, K, N, residual=True, out=out, in_place=True)


@pytest.mark.parametrize("M,K,N", [(3, 128, 48), (150, 256, 160), (40, 100, 40)])
def test_linear_e4m3_keeps_rows_apart(dev, stream, M, K, N):
    """A NaN value, or a scale that is not finite, stays in its row; each product is in its place."""
    say(f"linear e4m3 rows {M}x{K}x{N}")
    rng = np.random.default_rng(9)
    layer = nn.Linear(dev, K, N, use_bias=False, precision="e4m3")
    w = np.zeros((N, K), np.float32)
    for n in range(N):
        w[n, (n * 5 + 3) % K] = 1 + n % 7
    layer.load_weights(w)
    x = rounded(rng.standard_normal((M, K)) * 20, "e4m3")
    s = np.exp2(rng.integers(-3, 4, M)).astype(np.float32)
    x[1, K - 1], s[2] = np.nan, np.inf
    yt = nn.Tensor(dev, (M, N))
    layer.forward_scaled(tensor(dev, x, "e4m3"), tensor(dev, s, "f32"), yt, stream=stream)
    stream.sync(60000)
    y = yt.to_numpy()
    assert np.isnan(y[1]).all() and not np.isfinite(y[2]).any()
    wq, ws = quantise(w)
    ok = [m for m in range(M) if m not in (1, 2)]
    want = (x[ok].astype(np.float64) * s[ok, None]) @ (wq.astype(np.float64) * ws[:, None]).T
    check(y[ok], want, 4 * EPS * np.abs(want) + 1e-37, "one-hot")


def test_linear_e4m3_many_calls_share_the_layer(dev, stream):
    """A later, larger call and a smaller one after it (workspaces that grew)."""
    say("linear e4m3 workspace")
    rng = np.random.default_rng(10)
    layer = nn.Linear(dev, 100, 30, use_bias=False, precision="e4m3")
    w = rng.standard_normal((30, 100)).astype(np.float32)
    layer.load_weights(w)
    first = {}
    for M in (5, 400, 5, 400):
        x = np.random.default_rng(M).standard_normal((M, 100)).astype(np.float32)
        y = layer(tensor(dev, x, "f32"), stream)
        stream.sync(60000)
        y = y.to_numpy()
        np.testing.assert_array_equal(first.setdefault(M, y), y)


def test_linear_e4m3_refusals(dev, stream):
    say("linear e4m3 refusals")
    T = lambda shape, dtype="f32": nn.Tensor(dev, shape, dtype=dtype)  # noqa: E731
    layer = nn.Linear(dev, 64, 32, precision="e4m3")
    q, s, y = T((4, 64), "e4m3"), T((4,)), T((4, 32))
    f = layer.forward_scaled
    arg, size, conf = ("MNN_ERR_INVALID_ARGUMENT", "MNN_ERR_BUFFER_SIZE_MISMATCH",
                       "MNN_ERR_INVALID_CONFIGURATION")
    refuses(arg, lambda: f(q, None, y))
    refuses(arg, lambda: f(T((4, 64)), s, y))
    refuses(arg, lambda: f(q, T((4,), "i32"), y))
    refuses(size, lambda: f(q, T((5,)), y))
    refuses("MNN_ERR_SHAPE_MISMATCH", lambda: f(T((4, 63), "e4m3"), s, y))
    refuses(size, lambda: f(q, s, T((4, 33))))
    refuses(arg, lambda: f(q, s, T((4, 32), "e4m3")))
    refuses(arg, lambda: f(q, s, y, residual=T((4, 32), "bf16")))
    refuses(size, lambda: f(q, s, y, residual=T((3, 32))))
    sq = nn.Linear(dev, 8, 1, precision="e4m3")
    ss = T((4, 1))
    refuses(arg, lambda: sq.forward_scaled(T((4, 8), "e4m3"), ss, ss))
    refuses(size, lambda: layer.load_weights(np.zeros(63 * 32, np.float32)))
    refuses(conf, lambda: layer.load_weights(np.full(64 * 32, np.nan, np.float32)))
    refuses(conf, lambda: nn.Linear(dev, 0, 8, precision="e4m3"))
    for p in ("f32", "bf16"):
        refuses(arg, lambda: nn.Linear(dev, 64, 32, precision=p).forward_scaled(q, s, y))
    # layers that make no 8-bit products, and 8-bit or integer tensors in layers that take none
    refuses(conf, lambda: nn.MultiHeadAttention(dev, 64, 8, precision="e4m3"))
    refuses(conf, lambda: nn.FeedForward(dev, 64, 128, precision="e4m3"))
    refuses(conf, lambda: nn.Conv1D(dev, 2, 4, 3, precision="e4m3"))
    refuses(conf, lambda: nn.UNetEncoderBlock(dev, 2, 8, num_groups=1, precision="e4m3"))
    refuses(arg, lambda: layer.forward(q, y))
    refuses(arg, lambda: nn.Linear(dev, 64, 32).forward(q, y))
    refuses(arg, lambda: nn.LayerNorm(dev, 64).forward(q, T((4, 64))))
    seq = nn.Sequential(dev)
    seq.add(nn.LayerNorm(dev, 64))
    seq.build()
    refuses(arg, lambda: seq.forward(q, stream))
    f(T((0, 64), "e4m3"), T((0,)), T((0, 32)), stream=stream)


def test_rmsnorm_refuses_more_features_than_its_indices_hold(dev):
    say("rmsnorm features")
    for n in (2 ** 30 + 1, 2 ** 31 - 1, -1):
        refuses("MNN_ERR_INVALID_CONFIGURATION", lambda: nn.RMSNorm(dev, n))


# ------------------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize("B,S,H,KV,hd,dims,inter,dtype", [
    (1, 1, 1, 1, 2, (2,), False, "f32"), (8, 1, 8, 8, 64, (32, 16), False, "f32"),
    (2, 37, 8, 2, 48, (24, 24), False, "bf16"), (2, 37, 8, 2, 48, (24, 24), True, "bf16"),
    (1, 300, 6, 3, 72, (36, 36), True, "f32"), (3, 65, 5, 5, 33, (2, 6, 10), False, "f32"),
    (1, 129, 4, 1, 128, (128,), False, "bf16"), (1, 129, 4, 1, 128, (128,), True, "f32"),
    (2, 50, 3, 3, 96, (18, 30, 6, 12), True, "bf16"), (1, 1000, 8, 8, 64, (64,), False, "f32"),
    (4, 200, 8, 8, 48, (16, 32), False, "f32"), (1, 77, 1, 1, 7, (4,), False, "bf16")])
@pytest.mark.parametrize("in_place", [False, True])
def test_rotary(dev, stream, B, S, H, KV, hd, dims, inter, dtype, in_place):
    say(f"rotary {B}x{S} heads {H}/{KV} hd {hd} {dims} interleaved {inter} {dtype} in place {in_place}")
    rng = np.random.default_rng(B + S + hd)
    q = rounded(rng.standard_normal((B, S, H * hd)), dtype)
    k = rounded(rng.standard_normal((B, S, KV * hd)), dtype)
    shape = (B, S, len(dims)) if B % 2 == 0 else (S, len(dims))
    pos = rng.integers(-50, 5000, shape).astype(np.int32)
    pos.reshape(-1)[0] = 2 ** 31 - 1
    pos.reshape(-1)[-1] = -2 ** 31
    layer = nn.Rotary(dev, hd, dims, base=9000.0, interleaved=inter)
    qt, kt, pt = tensor(dev, q, dtype), tensor(dev, k, dtype), tensor(dev, pos, "i32")
    qo = qt if in_place else nn.Tensor(dev, q.shape, dtype=dtype)
    ko = kt if in_place else nn.Tensor(dev, k.shape, dtype=dtype)
    layer.forward(qt, kt, pt, qo, ko, stream)
    stream.sync(60000)
    for x, got, n in ((q, qo, H), (k, ko, KV)):
        want = rotary(x, pos, n, hd, dims, 9000.0, inter)
        # the fraction of a turn: 64-bit product (2^-53 of up to 2^31 / 2 pi turns, both here and in the
        # reference) and its rounding to fp32; sine and cosine 2 half steps, two products, a sum
        big = np.abs(x.reshape(B, S, n, hd)).max(-1, keepdims=True).repeat(hd, -1).reshape(x.shape)
        tol = big * (2 * np.pi * 2.0 ** 31 * 2.0 ** -52 + 16 * EPS) * 2
        check(got.to_numpy(), want, tol + HALF[dtype] * np.abs(want) * (dtype != "f32"), "turned")
        rest = sum(dims)  # passes unchanged
        np.testing.assert_array_equal(got.to_numpy().reshape(-1, hd)[:, rest:], x.reshape(-1, hd)[:, rest:])


@pytest.mark.parametrize("H,hd,dims,inter,dtype", [
    (9, 4096, (4096,), False, "f32"), (33, 4096, (2048, 2, 6), True, "bf16"), (1001, 6, (2, 2), False, "bf16"),
    (700, 64, (16, 48), False, "f32")])
def test_rotary_wide_tokens(dev, stream, H, hd, dims, inter, dtype):
    """More units a token than a workgroup takes at a time."""
    say(f"rotary {H} heads of {hd} {dims} {dtype}")
    rng = np.random.default_rng(H)
    q = rounded(rng.standard_normal((1, 5, H * hd)), dtype)
    pos = rng.integers(0, 900, (5, len(dims))).astype(np.int32)
    layer = nn.Rotary(dev, hd, dims, interleaved=inter)
    qo = nn.Tensor(dev, q.shape, dtype=dtype)
    layer.forward(tensor(dev, q, dtype), None, tensor(dev, pos, "i32"), qo, None, stream)
    stream.sync(60000)
    want = rotary(q, pos, H, hd, dims, 10000.0, inter)
    big = np.abs(q.reshape(1, 5, H, hd)).max(-1, keepdims=True).repeat(hd, -1).reshape(q.shape)
    check(qo.to_numpy(), want, big * 32 * EPS + HALF[dtype] * np.abs(want) * (dtype != "f32"), "turned")


def test_rotary_q_alone_and_scores_of_shifted_tokens(dev, stream):
    """q without k; the product of a turned query and key depends on the distance alone."""
    say("rotary shift")
    rng = np.random.default_rng(12)
    hd, S = 64, 40
    x = rng.standard_normal((S, hd)).astype(np.float32)
    layer = nn.Rotary(dev, hd, [hd])
    outs = []
    for shift in (0, 700001):
        y = nn.Tensor(dev, (S, hd))
        layer.forward(tensor(dev, x, "f32"), None, tensor(dev, np.arange(S)[:, None] + shift, "i32"), y,
                      stream=stream)
        stream.sync(60000)
        y = y.to_numpy().astype(np.float64)
        outs.append(y @ y.T)
    # entries off by 32 half steps of their norms' product at most
    check(outs[1], outs[0], 64 * EPS * np.outer(*[np.linalg.norm(x, axis=1)] * 2), "scores")


def test_rotary_refusals(dev, stream):
    say("rotary refusals")
    T = lambda shape, dtype="f32": nn.Tensor(dev, shape, dtype=dtype)  # noqa: E731
    conf, arg, size, shp = ("MNN_ERR_INVALID_CONFIGURATION", "MNN_ERR_INVALID_ARGUMENT",
                            "MNN_ERR_BUFFER_SIZE_MISMATCH", "MNN_ERR_SHAPE_MISMATCH")
    for dims in ([3], [0], [], [6, 4], [-2]):
        refuses(conf, lambda: nn.Rotary(dev, 8, dims))
    refuses(conf, lambda: nn.Rotary(dev, 8, [8], base=0.0))
    refuses(conf, lambda: nn.Rotary(dev, 0, [2]))
    layer = nn.Rotary(dev, 8, [4, 4])
    q, k, p, o, ko = T((2, 5, 16)), T((2, 5, 8)), T((5, 2), "i32"), T((2, 5, 16)), T((2, 5, 8))
    f = layer.forward
    refuses(arg, lambda: f(q, k, p, o))
    refuses(arg, lambda: f(q, T((2, 5, 8), "bf16"), p, o, ko))
    refuses(arg, lambda: f(q, k, T((5, 2)), o, ko))
    refuses(arg, lambda: f(q, k, p, T((2, 5, 16), "bf16"), ko))
    refuses(arg, lambda: f(q, T((2, 5, 16)), p, o, o))
    refuses(arg, lambda: f(T((2, 5, 16), "e4m3"), None, p, T((2, 5, 16), "e4m3")))
    refuses(size, lambda: f(q, k, p, T((2, 5, 8)), ko))
    refuses(size, lambda: f(q, k, T((4, 2), "i32"), o, ko))
    refuses(shp, lambda: f(q, k, T((10, 1), "i32"), o, ko))
    refuses(shp, lambda: f(q, T((2, 4, 8)), p, o, T((2, 4, 8))))
    refuses(shp, lambda: f(T((2, 5, 12)), None, p, o))
    refuses(conf, lambda: nn.Layer.forward(layer, q, o))
    f(T((0, 16)), None, T((0, 2), "i32"), T((0, 16)), stream=stream)


# ----------------------------------------------------------------------------- window attention
def window_case(dev, stream, B, S, H, KV, hd, left, right, sinks, dtype, lengths=None, scale=0.0, seed=0,
                q=None, k=None, v=None, std=1.3):
    rng = np.random.default_rng(seed + B + S + hd + left)
    q = rounded(rng.standard_normal((B, S, H * hd)) * std if q is None else q, dtype)
    k = rounded(rng.standard_normal((B, S, KV * hd)) * std if k is None else k, dtype)
    v = rounded(rng.standard_normal((B, S, KV * hd)) if v is None else v, dtype)
    layer = nn.WindowAttention(dev, H, hd, KV, left, right, sinks, scale)
    out = np.full((B, S, H * hd), -7.0, np.float32)
    ot = tensor(dev, out, dtype)
    lt = tensor(dev, np.asarray(lengths), "i32") if lengths is not None else None
    layer.forward(tensor(dev, q, dtype), tensor(dev, k, dtype), tensor(dev, v, dtype), ot, lt, stream)
    stream.sync(60000)
    got = ot.to_numpy()
    for b in range(B):
        n = S if lengths is None else min(max(lengths[b], 0), S)
        assert (got[b, n:] == -7).all(), f"rows behind sequence {b} were written"
        if n:
            want, spread, size = attend(q[b, :n], k[b, :n], v[b, :n], window_seen(n, left, right, sinks),
                                        H, KV, scale or 1 / np.sqrt(hd))
            check(got[b, :n], want, attention_tolerance(spread, size, hd, n, dtype), f"sequence {b}")
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,S,H,KV,hd,left,right,sinks", [
    (1, 1, 1, 1, 8, 0, 0, 0), (1, 2, 2, 1, 64, 0, 0, 1), (2, 33, 3, 3, 48, 5, 0, 2),
    (1, 64, 2, 1, 64, 63, 0, 0), (1, 65, 1, 1, 128, 1000, 1000, 70), (2, 130, 4, 2, 32, 16, 16, 4),
    (1, 257, 2, 2, 72, 100, 0, 33), (1, 300, 1, 1, 96, 0, 299, 3), (1, 200, 2, 1, 16, 7, 3, 0),
    (1, 400, 2, 2, 48, 168, 168, 4), (1, 513, 1, 1, 64, 64, 0, 65), (1, 700, 2, 1, 64, 300, 1, 129),
    (5, 1030, 8, 8, 48, 70, 0, 3), (6, 901, 8, 2, 64, 200, 5, 70), (3, 1025, 16, 16, 128, 64, 64, 2),
    (2, 1000, 8, 2, 64, 130, 0, 4), (2, 999, 8, 8, 80, 90, 33, 1), (1, 2500, 2, 2, 48, 1000, 0, 5),
    (1, 385, 1, 1, 128, 127, 0, 4), (3, 97, 5, 5, 24, 31, 31, 1), (1, 290, 1, 1, 104, 2 ** 30, 0, 2 ** 30)])
def test_window_attention(dev, stream, B, S, H, KV, hd, left, right, sinks, dtype):
    say(f"window {B}x{S} heads {H}/{KV} hd {hd} left {left} right {right} sinks {sinks} {dtype}")
    window_case(dev, stream, B, S, H, KV, hd, left, right, sinks, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lengths,S,left,right,sinks", [
    ([150, 1, 0, 64], 150, 40, 0, 4), ([-3, 200, 99, 1000], 130, 20, 20, 2), ([65, 128, 129, 127], 129, 500, 3, 0)])
def test_window_attention_padded_batch(dev, stream, lengths, S, left, right, sinks, dtype):
    """Keys and values behind a sequence's end hold NaN; rows behind it stay as they were."""
    say(f"window lengths {lengths} of {S} {dtype}")
    rng = np.random.default_rng(21)
    q, k, v = (rng.standard_normal((4, S, w * 48)).astype(np.float32) for w in (4, 2, 2))
    for b, n in enumerate(lengths):
        for x in (q, k, v):
            x[b, max(n, 0):] = np.nan
    window_case(dev, stream, 4, S, 4, 2, 48, left, right, sinks, dtype, lengths, q=q, k=k, v=v)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("S,H,KV,hd,left,right,sinks,lengths", [
    (1345, 8, 8, 48, 168, 168, 4, [1345, 700]), (1101, 10, 5, 32, 300, 0, 45, [33, 1100]),
    (1057, 8, 2, 64, 500, 2, 97, [1057, 961]), (1025, 9, 3, 40, 31, 64, 1, [1024, 0])])
def test_window_attention_groups_of_96(dev, stream, S, H, KV, hd, left, right, sinks, lengths, dtype):
    """Two ragged sequences whose workgroups of 96 queries just fit the compute units, NaN behind their ends."""
    say(f"window groups of 96 {S} heads {H}/{KV} hd {hd} {dtype}")
    rng = np.random.default_rng(25)
    q, k, v = (rng.standard_normal((2, S, w * hd)).astype(np.float32) for w in (H, KV, KV))
    for b, n in enumerate(lengths):
        for x in (q, k, v):
            x[b, n:] = np.nan
    window_case(dev, stream, 2, S, H, KV, hd, left, right, sinks, dtype, lengths, q=q, k=k, v=v)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, 3e38])
def test_window_attention_values_out_of_sight(dev, stream, what, bad, dtype):
    """One key (or value) holds a value that is not finite or overflows: the queries that do not see it
    are as without it, the others as the formula has them (not finite, or 0 weight on it)."""
    say(f"window {what} holds {bad} {dtype}")
    S, left, sinks, at = 260, 20, 2, 100
    rng = np.random.default_rng(22)
    q, k, v = (rounded(rng.standard_normal((1, S, 48)), dtype) for _ in range(3))
    out = []
    for b in (None, bad):
        x = {"k": k.copy(), "v": v.copy()}
        if b is not None:
            x[what][0, at, 5] = b
        ot = nn.Tensor(dev, (1, S, 48), dtype=dtype)
        layer = nn.WindowAttention(dev, 1, 48, window_left=left, sinks=sinks)
        layer.forward(tensor(dev, q, dtype), tensor(dev, x["k"], dtype), tensor(dev, x["v"], dtype), ot,
                      stream=stream)
        stream.sync(60000)
        out.append(ot.to_numpy()[0])
    sees = np.zeros(S, bool)
    sees[at:at + left + 1] = True
    want, spread, size = attend(q[0], k[0], v[0], window_seen(S, left, 0, sinks), 1, 1, 48 ** -0.5)
    tol = attention_tolerance(spread, size, 48, S, dtype)
    for o in out:
        check(o[~sees], want[~sees], tol[~sees], "out of sight")
    if np.isnan(bad):
        hit = out[1][sees] if what == "k" else out[1][sees][:, 5]
        assert np.isnan(hit).all()
    elif what == "v":
        assert (out[1][sees][:, 5] > 1e30).any() or np.isinf(out[1][sees][:, 5]).any()
    if what == "v":
        cols = [c for c in range(48) if c != 5]
        check(out[1][:, cols], want[:, cols], tol[:, cols], "other dimensions")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_window_attention_sizes_of_scores(dev, stream, dtype):
    """Scores in the hundreds (one key takes all), tiny values, a scale of the caller's, a negative one."""
    say(f"window scores {dtype}")
    window_case(dev, stream, 1, 150, 2, 1, 64, 60, 0, 2, dtype, std=12.0)
    window_case(dev, stream, 1, 150, 2, 1, 64, 60, 9, 2, dtype, scale=-0.3)
    rng = np.random.default_rng(23)
    q = np.full((1, 200, 48), 30.0) * np.sign(rng.standard_normal((1, 200, 1)))
    k = np.sort(rng.standard_normal((1, 200, 1)) * 30, axis=1) * np.ones((1, 200, 48)) / 7
    window_case(dev, stream, 1, 200, 1, 1, 48, 120, 0, 3, dtype, q=q, k=k)
    v = rng.standard_normal((1, 200, 48)) * 1e-35
    window_case(dev, stream, 1, 200, 1, 1, 48, 120, 0, 3, dtype, v=v)


def test_window_attention_refusals(dev, stream):
    say("window refusals")
    T = lambda shape, dtype="f32": nn.Tensor(dev, shape, dtype=dtype)  # noqa: E731
    conf, arg, size, shp = ("MNN_ERR_INVALID_CONFIGURATION", "MNN_ERR_INVALID_ARGUMENT",
                            "MNN_ERR_BUFFER_SIZE_MISMATCH", "MNN_ERR_SHAPE_MISMATCH")
    for kw in (dict(num_heads=3, head_dim=16, num_kv_heads=2), dict(num_heads=2, head_dim=12),
               dict(num_heads=2, head_dim=136), dict(num_heads=0, head_dim=16),
               dict(num_heads=2, head_dim=16, window_left=-1), dict(num_heads=2, head_dim=16, sinks=-1),
               dict(num_heads=2, head_dim=16, scale=float("nan"))):
        refuses(conf, lambda: nn.WindowAttention(dev, **kw))
    layer = nn.WindowAttention(dev, 4, 16, 2, window_left=3, sinks=1)
    q, k, v, o = T((2, 5, 64)), T((2, 5, 32)), T((2, 5, 32)), T((2, 5, 64))
    f = layer.forward
    refuses(shp, lambda: f(T((2, 5, 32)), k, v, o))
    refuses(shp, lambda: f(q, T((2, 4, 32)), v, o))
    refuses(shp, lambda: f(q, k, T((1, 5, 32)), o))
    refuses(arg, lambda: f(q, T((2, 5, 32), "bf16"), v, o))
    refuses(arg, lambda: f(q, k, v, T((2, 5, 64), "bf16")))
    refuses(size, lambda: f(q, k, v, T((2, 5, 32))))
    refuses(arg, lambda: f(q, k, v, q))
    refuses(arg, lambda: f(q, k, v, o, T((2,))))
    refuses(size, lambda: f(q, k, v, o, T((3,), "i32")))
    refuses(conf, lambda: nn.Layer.forward(layer, q, o))
    f(T((2, 0, 64)), T((2, 0, 32)), T((2, 0, 32)), T((2, 0, 64)), stream=stream)
    # the step
    pos, kc, vc = T((2,), "i32"), T((2, 9, 32)), T((2, 9, 32))
    g = layer.step
    refuses(conf, lambda: g(q, k, v, pos, T((2, 8, 32)), T((2, 8, 32)), o))
    refuses(shp, lambda: g(q, k, v, pos, kc, T((2, 10, 32)), o))
    refuses(shp, lambda: g(q, k, v, pos, T((1, 9, 32)), vc, o))
    refuses(arg, lambda: g(q, k, v, pos, T((2, 9, 32), "bf16"), vc, o))
    refuses(arg, lambda: g(q, k, v, T((2,)), kc, vc, o))
    refuses(size, lambda: g(q, k, v, T((3,), "i32"), kc, vc, o))
    refuses(size, lambda: g(q, k, v, pos, kc, vc, o, T((1,), "i32")))
    refuses(arg, lambda: g(q, k, v, pos, kc, kc, o))
    refuses(arg, lambda: g(q, k, v, pos, kc, vc, q))
    both = nn.WindowAttention(dev, 4, 16, 2, window_left=3, window_right=1)
    refuses(conf, lambda: both.step(q, k, v, pos, kc, vc, o))


# ----------------------------------------------------------------------- steps on rolling caches
class Streams:
    """Token histories of B streams, their caches on the GPU, and steps checked against the history."""

    def __init__(self, dev, B, H, KV, hd, left, sinks, slots, dtype, seed=0):
        self.dev, self.H, self.KV, self.hd, self.left, self.sinks = dev, H, KV, hd, left, sinks
        self.slots, self.dtype, self.rng = slots, dtype, np.random.default_rng(seed)
        self.hist = [([], []) for _ in range(B)]
        self.layer = nn.WindowAttention(dev, H, hd, KV, left, 0, sinks)
        # slots that no token has had yet hold NaN: nobody may read them
        nan = np.full((B, slots, KV * hd), np.nan, np.float32)
        self.kc, self.vc = tensor(dev, nan, dtype), tensor(dev, nan, dtype)

    def step(self, stream, T, steps=None, idle=()):
        B, w = len(self.hist), self.KV * self.hd
        pos = [(-1 - b) if b in idle else len(self.hist[b][0]) for b in range(B)]
        q = rounded(self.rng.standard_normal((B, T, self.H * self.hd)) * 1.3, self.dtype)
        k = rounded(self.rng.standard_normal((B, T, w)) * 1.3, self.dtype)
        v = rounded(self.rng.standard_normal((B, T, w)), self.dtype)
        n = [0 if b in idle else min(max(steps[b], 0), T) if steps else T for b in range(B)]
        for b in range(B):
            q[b, n[b]:] = k[b, n[b]:] = v[b, n[b]:] = np.nan
        before = self.kc.to_numpy(), self.vc.to_numpy()
        out = tensor(self.dev, np.full(q.shape, -7, np.float32), self.dtype)
        call = [tensor(self.dev, x, self.dtype) for x in (q, k, v)]
        pt = tensor(self.dev, np.array(pos), "i32")
        st = tensor(self.dev, np.array(steps), "i32") if steps else None
        for _ in range(2):  # the same call again changes nothing
            self.layer.step(*call, pt, self.kc, self.vc, out, st, stream)
        stream.sync(60000)
        got, after = out.to_numpy(), (self.kc.to_numpy(), self.vc.to_numpy())
        for b in range(B):
            assert (got[b, n[b]:] == -7).all(), f"rows behind stream {b}'s last were written"
            hk, hv = self.hist[b]
            hk.extend(k[b, :n[b]])
            hv.extend(v[b, :n[b]])
            for c in range(2):
                want = before[c][b].copy()
                for i in range(n[b]):
                    want[slot_of(pos[b] + i, self.sinks, self.slots)] = (k, v)[c][b, i]
                np.testing.assert_array_equal(after[c][b], want)
            if n[b]:
                p0 = pos[b]
                mine = np.arange(p0, p0 + n[b])[:, None]
                key = np.arange(p0 + n[b])[None]
                seen = (key <= mine) & ((key >= mine - self.left) | (key < self.sinks))
                want, spread, size = attend(q[b, :n[b]], np.array(hk), np.array(hv), seen, self.H, self.KV,
                                            self.hd ** -0.5)
                keys = min(self.left + 1 + self.sinks, p0 + n[b])
                check(got[b, :n[b]], want, attention_tolerance(spread, size, self.hd, keys, self.dtype),
                      f"stream {b} at {p0}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,H,KV,hd,left,sinks,spare,chunks", [
    (1, 1, 1, 8, 0, 0, 0, [1, 1, 1]), (1, 8, 8, 48, 11, 4, 0, [1] * 5 + [7, 1, 9, 1, 1, 1]),
    (3, 8, 2, 64, 100, 4, 3, [90, 1, 16, 1, 5, 1, 1]), (2, 4, 1, 128, 63, 0, 1, [64, 1, 1, 3, 1]),
    (2, 6, 3, 72, 5, 33, 0, [20, 1, 20, 1, 1]), (4, 5, 5, 32, 300, 1, 40, [257, 60, 1, 2]),
    (1, 2, 1, 96, 1000, 2, 0, [1200, 1, 1]),
    (2, 4, 2, 64, 2500, 5, 3, [2600, 1, 3, 1]), (1, 3, 3, 128, 900, 0, 7, [950, 2, 1]), (2, 16, 1, 64, 40, 2, 0, [30, 1, 4, 1])])
def test_window_step(dev, stream, B, H, KV, hd, left, sinks, spare, chunks, dtype):
    say(f"step {B} streams heads {H}/{KV} hd {hd} left {left} sinks {sinks} chunks {chunks} {dtype}")
    s = Streams(dev, B, H, KV, hd, left, sinks, sinks + left + max(chunks) + spare, dtype)
    for T in chunks:
        s.step(stream, T)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_window_step_ragged_streams(dev, stream, dtype):
    """Streams that bring fewer rows than the others, none, or are left alone by their position."""
    say(f"step ragged {dtype}")
    s = Streams(dev, 5, 4, 2, 48, 20, 3, 3 + 20 + 9, dtype)
    s.step(stream, 9, [9, 4, 0, 1, 100])
    s.step(stream, 4, [-5, 4, 3, 4, 2], idle=(3,))
    s.step(stream, 1)
    s.step(stream, 9, [9, 9, 9, 9, 9], idle=(0,))
    s.step(stream, 9, [1, 9, 2, 9, 9])
    s.step(stream, 1, idle=(1, 2))


@pytest.mark.parametrize("dtype,hd,KV", [("f32", 48, 2), ("bf16", 64, 1)])
def test_window_step_far_positions(dev, stream, dtype, hd, KV):
    """Positions near the largest that a call takes; one beyond it leaves the stream alone."""
    say(f"step far {dtype}")
    left, sinks, slots = 30, 2, 40
    layer = nn.WindowAttention(dev, 2, hd, KV, left, 0, sinks)
    rng = np.random.default_rng(31)
    w = KV * hd
    kc, vc = (rounded(rng.standard_normal((2, slots, w)), dtype) for _ in "kv")
    q = rounded(rng.standard_normal((2, 1, 2 * hd)), dtype)
    k, v = (rounded(rng.standard_normal((2, 1, w)), dtype) for _ in "kv")
    p = 2 ** 31 - 2
    kt, vt = tensor(dev, kc, dtype), tensor(dev, vc, dtype)
    out = tensor(dev, np.full(q.shape, -7, np.float32), dtype)
    layer.step(tensor(dev, q, dtype), tensor(dev, k, dtype), tensor(dev, v, dtype),
               tensor(dev, np.array([p, p + 1]), "i32"), kt, vt, out, stream=stream)
    stream.sync(60000)
    got = out.to_numpy()
    at = list(range(sinks)) + [slot_of(i, sinks, slots) for i in range(p - left, p)]
    kk, vv = np.concatenate([kc[0, at], k[0]]), np.concatenate([vc[0, at], v[0]])
    want, spread, size = attend(q[0], kk, vv, np.ones((1, len(kk)), bool), 2, KV, hd ** -0.5)
    check(got[0], want, attention_tolerance(spread, size, hd, len(kk), dtype), "far")
    assert (got[1] == -7).all()
    np.testing.assert_array_equal(kt.to_numpy()[1], kc[1])


def test_window_step_equals_whole_sequence(dev, stream):
    """Steps of one token give what the whole sequence gives (fp32, the same formula)."""
    say("step against whole")
    S, H, KV, hd, left, sinks = 90, 4, 2, 48, 17, 3
    rng = np.random.default_rng(33)
    q, k, v = (rng.standard_normal((1, S, n * hd)).astype(np.float32) for n in (H, KV, KV))
    layer = nn.WindowAttention(dev, H, hd, KV, left, 0, sinks)
    whole = nn.Tensor(dev, q.shape)
    layer.forward(*(tensor(dev, x, "f32") for x in (q, k, v)), whole, stream=stream)
    kc, vc = (nn.Tensor(dev, (1, sinks + left + 1, KV * hd)) for _ in "kv")
    rows = []
    for i in range(S):
        o = nn.Tensor(dev, (1, 1, H * hd))
        layer.step(*(tensor(dev, x[:, i:i + 1], "f32") for x in (q, k, v)),
                   tensor(dev, np.array([i]), "i32"), kc, vc, o, stream=stream)
        stream.sync(60000)
        rows.append(o.to_numpy()[0, 0])
    stream.sync(60000)
    want, spread, size = attend(q[0], k[0], v[0], window_seen(S, left, 0, sinks), H, KV, hd ** -0.5)
    tol = attention_tolerance(spread, size, hd, S, "f32")
    check(whole.to_numpy()[0], want, tol, "whole")
    check(np.array(rows), want, tol, "steps")


def test_window_step_slots_beyond_32_bit_offsets(dev, stream):
    """A cache of 8.6 GB: the slots in use lie past 2^32 bytes and past 2^32 values."""
    say("step far slots")
    H, hd, left, slots = 32, 128, 6, (1 << 20) + 64
    layer = nn.WindowAttention(dev, H, hd, H, left)
    rng = np.random.default_rng(41)
    kc, vc = (nn.Tensor(dev, (1, slots, H * hd), dtype="bf16") for _ in "kv")
    hist, p0 = [], slots - 9
    for i in range(12):  # runs over the ring's end
        q, k, v = (rounded(rng.standard_normal((1, 1, H * hd)), "bf16") for _ in range(3))
        hist.append((k[0, 0], v[0, 0]))
        o = nn.Tensor(dev, q.shape, dtype="bf16")
        layer.step(tensor(dev, q, "bf16"), tensor(dev, k, "bf16"), tensor(dev, v, "bf16"),
                   tensor(dev, np.array([p0 + i]), "i32"), kc, vc, o, stream=stream)
        if i < left:
            continue  # the window still holds the cache's zeros
        stream.sync(60000)
        kk, vv = (np.array([h[c] for h in hist[-left - 1:]]) for c in (0, 1))
        want, spread, size = attend(q[0], kk, vv, np.ones((1, left + 1), bool), H, H, hd ** -0.5)
        check(o.to_numpy()[0], want, attention_tolerance(spread, size, hd, left + 1, "bf16"), f"token {i}")


def test_rows_beyond_32_bit_offsets(dev, stream):
    """Rows past 2^32 values: an 8-bit linear fills them with its bias, the norm reads them and its sum."""
    say("far rows")
    rows, F = (1 << 20) + 5, 4096
    rng = np.random.default_rng(42)
    bias = rounded(rng.standard_normal(F), "bf16")
    lin = nn.Linear(dev, 8, F, precision="e4m3")
    lin.load_weights(np.zeros((F, 8), np.float32), bias)
    y = nn.Tensor(dev, (rows, F), dtype="bf16")
    lin.forward_scaled(nn.Tensor(dev, (rows, 8), dtype="e4m3"), nn.Tensor(dev, (rows,)), y, stream=stream)
    norm = nn.RMSNorm(dev, F)
    total, scales, q = nn.Tensor(dev, (rows, F), dtype="bf16"), nn.Tensor(dev, (rows,)), nn.Tensor(
        dev, (rows, F), dtype="e4m3")
    norm.forward_residual(y, None, q, sum=total, scales=scales, stream=stream)
    stream.sync(60000)
    want = np.abs(rmsnorm(bias, np.ones(F), 1e-5)).max() / 448
    first = scales.to_numpy()
    check(first, np.full(rows, want), (F / 64 + 28) * EPS * want, "scales")
    norm.forward_residual(total, None, q, scales=scales, stream=stream)
    stream.sync(60000)
    np.testing.assert_array_equal(scales.to_numpy(), first)


# ------------------------------------------------------------------------ together, and captured
class Block:
    """Attention of a pre-norm transformer block on streams: norm with residual to 8 bits, q, k and v
    in one product, rotary positions, the step on rolling caches, the output product with residual."""

    def __init__(self, dev, B, E, heads, left, sinks, dtype, seed=0):
        self.dev, self.B, self.E, self.H, self.hd, self.dtype = dev, B, E, heads, E // heads, dtype
        rng = np.random.default_rng(seed)
        self.w = {n: (rng.standard_normal((E, E)) / np.sqrt(E)).astype(np.float32) for n in "qkvo"}
        self.b = {n: (0.1 * rng.standard_normal(E)).astype(np.float32) for n in "qkvo"}
        self.g = (1 + 0.1 * rng.standard_normal(E)).astype(np.float32)
        self.norm = nn.RMSNorm(dev, E)
        self.norm.load_parameters(self.g)
        self.lin = {}
        for n in "qkvo":
            self.lin[n] = nn.Linear(dev, E, E, precision="e4m3")
            self.lin[n].load_weights(self.w[n], self.b[n])
        self.dims = [self.hd // 2, self.hd // 4 * 2 - self.hd // 4 % 2 * 2]
        self.rot = nn.Rotary(dev, self.hd, self.dims)
        self.left, self.sinks, self.slots = left, sinks, sinks + left + 1
        self.att = nn.WindowAttention(dev, heads, self.hd, window_left=left, sinks=sinks)
        T = lambda dt, *shape: nn.Tensor(dev, shape, dtype=dt)  # noqa: E731
        self.x, self.r = T(dtype, B, 1, E), T(dtype, B, 1, E)
        self.h, self.n8, self.s = T(dtype, B, 1, E), T("e4m3", B, 1, E), T("f32", B)
        self.t = {n: T(dtype, B, 1, E) for n in "qkvao"}
        self.kc, self.vc = T(dtype, B, self.slots, E), T(dtype, B, self.slots, E)
        self.pos, self.grid = T("i32", B), T("i32", B, 1, 2)

    def run(self, stream):
        t = self.t
        self.norm.forward_residual(self.x, self.r, self.n8, sum=self.h, scales=self.s, stream=stream)
        for n in "qkv":
            self.lin[n].forward_scaled(self.n8, self.s, t[n], stream=stream)
        self.rot.forward(t["q"], t["k"], self.grid, t["q"], t["k"], stream)
        self.att.step(t["q"], t["k"], t["v"], self.pos, self.kc, self.vc, t["a"], stream=stream)
        self.lin["o"].forward_scaled(t["a"], None, t["o"], residual=self.h, stream=stream)

    def feed(self, x, r, pos):
        self.x.copy_from(x)
        self.r.copy_from(r)
        self.pos.copy_from(np.array(pos))
        self.grid.copy_from(np.array([[[p, p // 7]] for p in pos]))


def linear_reference(x, xs, w, b, dtype):
    wq, ws = quantise(w)
    xd, wd = x.astype(np.float64) * xs[:, None], wq.astype(np.float64) * ws[:, None]
    y = xd @ wd.T + b
    mass = np.abs(xd) @ np.abs(wd).T
    return y, (1.5 * x.shape[1] + 8) * EPS * (mass + np.abs(y) + 0.5) + HALF[dtype] * np.abs(y) * (dtype != "f32")


@pytest.mark.parametrize("B,E,heads,dtype", [(3, 384, 8, "bf16"), (2, 96, 2, "f32")])
def test_block_on_streams(dev, stream, B, E, heads, dtype):
    """Every stage against its reference on what the GPU gave the stage before it."""
    say(f"block {B} streams E {E} {dtype}")
    m = Block(dev, B, E, heads, 9, 2, dtype)
    rng = np.random.default_rng(51)
    hist = [[] for _ in range(B)]
    pos = [0, 3, 40][:B]  # the later streams' windows hold the caches' zeros at first
    for b in range(B):
        hist[b] = [(np.zeros(E), np.zeros(E))] * pos[b]
    for _ in range(25):
        x, r = (rounded(rng.standard_normal((B, 1, E)), dtype) for _ in range(2))
        m.feed(x, r, pos)
        m.run(stream)
        stream.sync(60000)
        h = m.h.to_numpy()
        np.testing.assert_array_equal(h, rounded(x + r, dtype))
        n8, s = m.n8.to_numpy()[:, 0], m.s.to_numpy()
        y = rmsnorm((x + r)[:, 0], m.g, 1e-5)
        unit = np.abs(y) / s[:, None]
        check(n8 * s[:, None].astype(np.float64), y,
              (np.maximum(unit * HALF["e4m3"], 2.0 ** -10) * (1 + 1e-5) + 448 * 80 * EPS) * s[:, None], "norm")
        got = {n: t.to_numpy() for n, t in m.t.items()}
        want, tol = linear_reference(n8, s, m.w["v"], m.b["v"], dtype)
        check(got["v"][:, 0], want, tol, "v")
        for n in "qk":
            want, tol = linear_reference(n8, s, m.w[n], m.b[n], dtype)
            grid = np.array([[[p, p // 7]] for p in pos])
            turned = rotary(want[:, None], grid, heads, m.hd, m.dims)
            size = np.abs(want).reshape(B, heads, m.hd).max(-1, keepdims=True).repeat(m.hd, -1).reshape(B, E)
            slack = tol.reshape(B, heads, m.hd).max(-1, keepdims=True).repeat(m.hd, -1).reshape(B, E)
            # a pair's errors add up to sqrt(2) of the larger one's, and one more rounding
            check(got[n][:, 0], turned[:, 0], 1.5 * slack + size * (HALF[dtype] + 32 * EPS), n)
        for b in range(B):
            hist[b].append((got["k"][b, 0].astype(np.float64), got["v"][b, 0].astype(np.float64)))
            keys = [i for i in range(pos[b] + 1) if i >= pos[b] - m.left or i < m.sinks]
            kk, vv = (np.array([hist[b][i][c] for i in keys]) for c in (0, 1))
            want, spread, size = attend(got["q"][b], kk, vv, np.ones((1, len(keys)), bool), heads, heads,
                                        m.hd ** -0.5)
            check(got["a"][b], want, attention_tolerance(spread, size, m.hd, len(keys), dtype), "attention")
        aq, asc = quantise(got["a"][:, 0])
        want, tol = linear_reference(aq, asc, m.w["o"], m.b["o"], dtype)
        want = want + h[:, 0]
        check(got["o"][:, 0], want, tol + (HALF[dtype] if dtype != "f32" else EPS) * np.abs(want), "out")
        pos = [p + 1 for p in pos]


class Graph:
    """Calls on a stream, captured once and replayed."""

    def __init__(self, stream, calls):
        path = next(ln.split()[-1] for ln in open("/proc/self/maps") if "libamdhip64" in ln)
        self.hip = C.CDLL(path)
        self.s = C.c_void_p(C.cast(stream.handle, C.POINTER(C.c_void_p))[1])  # {device, hipStream_t, ..}
        graph, self.exec = C.c_void_p(), C.c_void_p()
        self.ok(self.hip.hipStreamBeginCapture(self.s, 2))
        calls()
        self.ok(self.hip.hipStreamEndCapture(self.s, C.byref(graph)))
        self.ok(self.hip.hipGraphInstantiate(C.byref(self.exec), graph, None, None, C.c_size_t(0)))

    def ok(self, status):
        assert status == 0, f"hip status {status}"

    def replay(self):
        self.ok(self.hip.hipGraphLaunch(self.exec, self.s))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_block_captured_and_replayed(dev, dtype):
    """The block in a graph, replayed with other inputs, positions and eager work of the same layers
    between the replays (also larger calls, which grow their workspaces), equals the eager block."""
    say(f"block captured {dtype}")
    s, other = nn.Stream(dev), nn.Stream(dev)
    B, E = 2, 192
    eager, taken = (Block(dev, B, E, 4, 700, 2, dtype) for _ in range(2))  # split keys: a workspace
    rng = np.random.default_rng(52)

    def inputs():
        return (rounded(rng.standard_normal((B, 1, E)), dtype) for _ in range(2))

    x, r = inputs()
    for m in (eager, taken):  # workspaces are made by a call outside the graph
        m.feed(x, r, [0, 5])
        m.run(s)
    s.sync(60000)
    graph = Graph(s, lambda: taken.run(s))
    for i in range(6):
        x, r = inputs()
        pos = [3 * i, 1000 + i]
        for m in (eager, taken):
            m.feed(x, r, pos)
        eager.run(other)
        graph.replay()
        s.sync(60000)
        other.sync(60000)
        for n in "qkvao":
            np.testing.assert_array_equal(taken.t[n].to_numpy(), eager.t[n].to_numpy())
        np.testing.assert_array_equal(taken.kc.to_numpy(), eager.kc.to_numpy())
        # other calls of the captured layers, on their stream, larger than any before
        big = tensor(dev, rng.standard_normal((40 + 30 * i, E)), dtype)
        taken.lin["o"].forward_scaled(big, None, nn.Tensor(dev, (40 + 30 * i, E), dtype=dtype), stream=s)
        n = 30 + 10 * i
        qkv = [tensor(dev, rng.standard_normal((3, n, E)), dtype) for _ in range(3)]
        caches = [nn.Tensor(dev, (3, 702 + n, E), dtype=dtype) for _ in range(2)]
        taken.att.step(*qkv, tensor(dev, np.array([0, 9, 800]), "i32"), *caches,
                       nn.Tensor(dev, (3, n, E), dtype=dtype), stream=s)
        s.sync(60000)


def test_calls_on_many_streams(dev):
    """The same work on several streams at once, one layer a stream, and on the default stream."""
    say("streams")
    rng = np.random.default_rng(53)
    S, H, hd = 300, 4, 48
    x = [rng.standard_normal((1, S, H * hd)).astype(np.float32) for _ in range(3)]
    want = None
    jobs = []
    for stream in [None] + [nn.Stream(dev) for _ in range(4)]:
        layer = nn.WindowAttention(dev, H, hd, window_left=40, window_right=7, sinks=3)
        out = nn.Tensor(dev, x[0].shape)
        layer.forward(*(tensor(dev, v, "f32") for v in x), out, stream=stream)
        jobs.append((layer, out))
    dev.synchronize()
    for _, out in jobs:
        got = out.to_numpy()
        want = got if want is None else want
        np.testing.assert_array_equal(got, want)
