"""The decoder's operators through the C ABI against 64-bit references: the linear layer with scales for
blocks of 128, rolling caches in 8 bits and the window step on them, attention to an encoder's states.
Tolerances count roundings (token_refs.py, decoder_refs.py) and were fixed before the first run."""
import numpy as np
import pytest

from metalaudio_amd import nn
from tests.decoder_refs import (blocks_of, held_rows, held_tolerance, linear_blocks, memory, quantise_blocks,
                                quantise_tiles, split_tolerance, spread_scales, values_of)
from tests.test_gpu_tokens import ACTS, Graph, check, refuses, tensor
from tests.token_refs import EPS, HALF, TINY, attend, rmsnorm, rounded, slot_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return nn.AudioDevice(0)


@pytest.fixture(scope="module")
def stream(dev):
    return nn.Stream(dev)


def say(msg):
    print(f"[case] {msg}", flush=True)


def empty(dev, shape, dtype="f32", fill=None):
    t = nn.Tensor(dev, shape, dtype=dtype)
    if fill is not None:
        t.copy_from(np.full(shape, fill, np.float32))
    return t


# ------------------------------------------------------------------ the linear layer, in blocks
def outliers(rng, m, k):
    """Activations with a few channels far above the others, which a scale a row would not hold."""
    x = rng.standard_normal((m, k)) * np.exp(0.5 * rng.standard_normal((m, 1)))
    x[:, 5::61] *= 300
    return x.astype(np.float32)


def blocks_case(dev, stream, M, K, N, act="none", residual=False, inp="e4m3", out="f32", bias=True,
                in_place=False, seed=0):
    rng = np.random.default_rng(seed + M * 5 + K * 3 + N)
    x = outliers(rng, M, K)
    w = (rng.standard_normal((N, K)) / np.sqrt(K)).astype(np.float32)
    w[:, 3::200] *= 30
    b = (0.1 * rng.standard_normal(N)).astype(np.float32)
    r = rounded(rng.standard_normal((M, N)), out) if residual else None
    layer = nn.Linear(dev, K, N, use_bias=bias, activation=act, precision="e4m3_block")
    layer.load_weights(w, b if bias else None)
    if inp == "e4m3":
        xq, xs = quantise_blocks(x)
        xt, st = tensor(dev, xq, "e4m3"), tensor(dev, xs, "f32")
    else:
        xq, xs = quantise_blocks(rounded(x, inp))
        xt, st = tensor(dev, x, inp), None
    rt = tensor(dev, r, out) if residual else None
    yt = rt if in_place else nn.Tensor(dev, (M, N), dtype=out)
    layer.forward_scaled(xt, st, yt, residual=rt, stream=stream)
    stream.sync(60000)
    y, mass = linear_blocks(xq, xs, *quantise_tiles(w), b if bias else None)
    # each addition rounds by at most 1.5 * 2^-24 of the running sum (matrix instructions), each block's sum
    # by its scales' product and its addition; bias and activation a few half steps
    tol = (1.5 * K + 3 * blocks_of(K) + 4) * EPS * mass + 4 * EPS * (np.abs(y) + 0.2)
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
    (3, 1, 1, {}), (2, 100, 7, {"residual": True}), (17, 320, 200, {"act": "relu"}), (32, 129, 129, {}),
    (16, 2048, 512, {"residual": True}), (33, 1000, 777, {"act": "swish", "out": "bf16"}),
    (64, 384, 384, {"residual": True, "out": "bf16"}), (67, 384, 1536, {"act": "gelu"}),
    (129, 1536, 384, {"residual": True}), (257, 512, 513, {"act": "tanh"}), (700, 384, 1152, {}),
    (1344, 384, 1536, {"act": "gelu", "out": "bf16"}), (2688, 1536, 384, {"residual": True}),
    (200, 2048, 2048, {"act": "leaky_relu", "residual": True}), (130, 640, 130, {"act": "sigmoid"}),
    (1000, 256, 260, {"bias": False, "residual": True, "out": "bf16"}), (511, 896, 1026, {"out": "bf16"}),
    (4099, 256, 4104, {"residual": True, "out": "bf16"}), (4097, 384, 4100, {"act": "relu"}),
    (3001, 256, 1240, {"in_place": True, "residual": True}), (2099, 130, 2055, {"act": "swish"})])
def test_linear_blocks(dev, stream, M, K, N, kw):
    say(f"linear blocks {M}x{K}x{N} {kw}")
    blocks_case(dev, stream, M, K, N, **kw)


@pytest.mark.parametrize("M,K,N,kw", [
    (4000, 100, 4090, {"out": "bf16"}), (4096, 300, 3842, {"residual": True}), (3841, 640, 4096, {"act": "gelu", "out": "bf16"}),
    (3900, 256, 3970, {"residual": True, "out": "bf16"})])
def test_linear_blocks_tiles_of_128_by_256(dev, stream, M, K, N, kw):
    """One, two, three and five depth steps."""
    say(f"linear blocks 128 x 256 {M}x{K}x{N} {kw}")
    blocks_case(dev, stream, M, K, N, **kw)


@pytest.mark.parametrize("M,K,N,kw", [
    (600, 130, 500, {"out": "bf16"}), (900, 100, 300, {"residual": True}), (513, 1536, 520, {"act": "relu"}),
    (33, 2048, 512, {"out": "bf16"}), (500, 129, 511, {"residual": True, "in_place": True}), (512, 2048, 512, {"act": "gelu"}),
    (64, 100, 4096, {"out": "bf16"}), (257, 384, 900, {"residual": True, "out": "bf16"})])
def test_linear_blocks_between_few_and_many_rows(dev, stream, M, K, N, kw):
    """Tiles of 64 square, and 32 rows a workgroup where those are few."""
    say(f"linear blocks {M}x{K}x{N} {kw}")
    blocks_case(dev, stream, M, K, N, **kw)


@pytest.mark.parametrize("M,K,N,inp,out", [(1, 384, 96, "f32", "f32"), (9, 257, 64, "bf16", "bf16"),
                                           (300, 512, 300, "bf16", "f32"), (45, 1000, 33, "f32", "bf16"),
                                           (2, 20000, 24, "bf16", "f32"), (700, 136, 60, "bf16", "f32"),
                                           (40, 2052, 50, "f32", "f32")])
def test_linear_blocks_round_wider_input(dev, stream, M, K, N, inp, out):
    say(f"linear blocks from {inp} {M}x{K}x{N}")
    blocks_case(dev, stream, M, K, N, inp=inp, out=out, residual=True)


@pytest.mark.parametrize("M,K,N", [(3, 256, 48), (150, 256, 160), (40, 200, 40), (2500, 384, 1300)])
def test_linear_blocks_keep_rows_and_blocks_apart(dev, stream, M, K, N):
    """A NaN value, or a scale that is not finite, stays in its row; each product is in its place, times the
    scales of its own blocks, which differ by powers of two."""
    say(f"linear blocks rows {M}x{K}x{N}")
    rng = np.random.default_rng(9)
    layer = nn.Linear(dev, K, N, use_bias=False, precision="e4m3_block")
    w = np.zeros((N, K), np.float32)
    for n in range(N):
        w[n, (n * 131 + 3) % K] = (1 + n % 7) * 2.0 ** (n // 128 % 5) * 8.0 ** ((n * 131 + 3) % K // 128)
    layer.load_weights(w)
    x = rounded(rng.standard_normal((M, K)) * 20, "e4m3")
    s = np.exp2(rng.integers(-20, 20, (M, blocks_of(K)))).astype(np.float32)
    x[1, K - 1], s[2, 0] = np.nan, np.inf
    yt = nn.Tensor(dev, (M, N))
    layer.forward_scaled(tensor(dev, x, "e4m3"), tensor(dev, s, "f32"), yt, stream=stream)
    stream.sync(60000)
    y = yt.to_numpy()
    assert np.isnan(y[1]).all() and not np.isfinite(y[2]).any()
    wq, ws = quantise_tiles(w)
    ok = [m for m in range(M) if m not in (1, 2)]
    want, mass = linear_blocks(x[ok], s[ok], wq, ws, None)
    check(y[ok], want, 4 * EPS * mass + 1e-37, "one-hot")


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,K,N", [(5, 256, 96), (200, 384, 320), (2500, 256, 1400), (3001, 384, 1240),
                                   (4000, 256, 4090)])
def test_linear_blocks_sums_that_cancel(dev, stream, M, K, N, out):
    """Two products of 448 x 448 cancel beside small ones, within a block or over two: all partial sums are
    multiples of 1/16 below 2^19, so no fp32 sum is rounded; the weights' scales are one power of two."""
    say(f"linear blocks that cancel {M}x{K}x{N} {out}")
    rng = np.random.default_rng(M + K + N)
    for gap in (1, 5, 40, 130):
        x = rng.integers(-4, 5, (M, K)).astype(np.float32) / 4
        w = rng.integers(-4, 5, (N, K)).astype(np.float32) / 4
        at = int(rng.integers(0, K - gap))
        x[:, [at, at + gap]] = 448
        w[:, at], w[:, at + gap] = 448, -448
        w[::64, ::64] = 448  # every block's largest value
        x[:, ::64] = np.where(np.isin(np.arange(0, K, 64), [at, at + gap]), 448, 0)
        wq, ws = quantise_tiles(w)
        np.testing.assert_array_equal(wq, w)
        want = (x.astype(np.float64) @ w.astype(np.float64).T) * float(ws[0, 0])
        layer = nn.Linear(dev, K, N, use_bias=False, precision="e4m3_block")
        layer.load_weights(w)
        y = nn.Tensor(dev, (M, N), dtype=out)
        layer.forward_scaled(tensor(dev, x, "e4m3"), tensor(dev, np.ones((M, blocks_of(K))), "f32"), y,
                             stream=stream)
        stream.sync(60000)
        # the scale's product, and the additions of blocks that it has made inexact
        tol = 4 * EPS * np.abs(want) + HALF[out] * (out == "bf16") * np.abs(want)
        tol = tol + (EPS * 2 ** 19 * float(ws[0, 0]) * 2 * blocks_of(K) if gap == 130 or K > 128 else 0)
        check(y.to_numpy(), want, tol, f"gap {gap}")


@pytest.mark.parametrize("scale", [1e-28, 1e-15, 1e18, 1e33])
def test_linear_blocks_far_scales(dev, stream, scale):
    """Rows and weights whose scales multiply to little or much more than either, results in range."""
    say(f"linear blocks scale {scale}")
    rng = np.random.default_rng(3)
    for M in (4, 90):
        x = (outliers(rng, M, 300) * scale).astype(np.float32)
        w = (rng.standard_normal((70, 300)) / np.float32(scale)).astype(np.float32)
        layer = nn.Linear(dev, 300, 70, use_bias=False, precision="e4m3_block")
        layer.load_weights(w)
        y = nn.Tensor(dev, (M, 70))
        layer.forward_scaled(tensor(dev, x, "f32"), None, y, stream=stream)
        stream.sync(60000)
        want, mass = linear_blocks(*quantise_blocks(x), *quantise_tiles(w), None)
        check(y.to_numpy(), want, (1.5 * 300 + 16) * EPS * mass, f"{M} rows")


def test_linear_blocks_many_calls_share_the_layer(dev, stream):
    say("linear blocks workspace")
    layer = nn.Linear(dev, 300, 30, use_bias=False, precision="e4m3_block")
    layer.load_weights(np.random.default_rng(10).standard_normal((30, 300)))
    first = {}
    for M in (5, 400, 5, 400):
        x = np.random.default_rng(M).standard_normal((M, 300)).astype(np.float32)
        y = layer(tensor(dev, x, "f32"), stream)
        stream.sync(60000)
        y = y.to_numpy()
        np.testing.assert_array_equal(first.setdefault(M, y), y)


def test_linear_blocks_weights_loaded_under_a_graph(dev):
    """A captured call sees weights that are loaded between its replays, whatever their size."""
    say("linear blocks loaded under a graph")
    s = nn.Stream(dev)
    rng = np.random.default_rng(17)
    for M in (3, 200):
        K, N = 256, 300
        layer, fresh = (nn.Linear(dev, K, N, precision="e4m3_block") for _ in range(2))
        w, b = rng.standard_normal((N, K)), rng.standard_normal(N)
        x, y, z = tensor(dev, rng.standard_normal((M, K)), "f32"), nn.Tensor(dev, (M, N)), nn.Tensor(dev, (M, N))
        layer.load_weights(w, b)
        layer.forward_scaled(x, None, y, stream=s)
        s.sync(60000)
        graph = Graph(s, lambda: layer.forward_scaled(x, None, y, stream=s))
        for size in (1.0, 5000.0, 1e30, 2.0):
            for m in (layer, fresh):
                m.load_weights(w * size, b)
            graph.replay()
            fresh.forward_scaled(x, None, z, stream=s)
            s.sync(60000)
            np.testing.assert_array_equal(y.to_numpy(), z.to_numpy())


def test_linear_blocks_hold_outliers_that_rows_do_not(dev, stream):
    """What blocks are for: one value of 10^6 costs a row's other blocks nothing."""
    say("linear blocks outlier")
    rng = np.random.default_rng(12)
    x = rng.standard_normal((50, 512)).astype(np.float32)
    x[:, 400] = 1e6
    w = rng.standard_normal((64, 512)).astype(np.float32)
    w[:, 400] = 0
    err = {}
    for precision in ("e4m3", "e4m3_block"):
        layer = nn.Linear(dev, 512, 64, use_bias=False, precision=precision)
        layer.load_weights(w)
        y = layer(tensor(dev, x, "f32"), stream)
        stream.sync(60000)
        want = x.astype(np.float64) @ w.astype(np.float64).T
        err[precision] = np.linalg.norm(y.to_numpy() - want) / np.linalg.norm(want)
    # three quarters of the sum's squares are held to a rounding of e4m3 (at most 2^-4) on both sides
    assert err["e4m3_block"] < 0.55 and err["e4m3"] > 0.9, err


def test_linear_blocks_refusals(dev, stream):
    say("linear blocks refusals")
    T = lambda shape, dtype="f32": nn.Tensor(dev, shape, dtype=dtype)  # noqa: E731
    layer = nn.Linear(dev, 200, 32, precision="e4m3_block")
    q, s, y = T((4, 200), "e4m3"), T((4, 2)), T((4, 32))
    f = layer.forward_scaled
    arg, size, conf = ("MNN_ERR_INVALID_ARGUMENT", "MNN_ERR_BUFFER_SIZE_MISMATCH",
                       "MNN_ERR_INVALID_CONFIGURATION")
    f(q, s, y, stream=stream)
    refuses(arg, lambda: f(q, None, y))
    refuses(arg, lambda: f(T((4, 200)), s, y))
    refuses(size, lambda: f(q, T((4,)), y))
    refuses(size, lambda: f(q, T((4, 3)), y))
    refuses(size, lambda: nn.Linear(dev, 200, 32, precision="e4m3").forward_scaled(q, s, y))
    refuses("MNN_ERR_SHAPE_MISMATCH", lambda: f(T((4, 199), "e4m3"), s, y))
    refuses(size, lambda: f(q, s, T((4, 33))))
    refuses(arg, lambda: f(q, s, T((4, 32), "e4m3")))
    refuses(arg, lambda: f(q, s, y, residual=T((4, 32), "bf16")))
    refuses(conf, lambda: layer.load_weights(np.full(200 * 32, np.inf, np.float32)))
    refuses(conf, lambda: nn.MultiHeadAttention(dev, 64, 8, precision="e4m3_block"))
    refuses(conf, lambda: nn.Conv1D(dev, 2, 4, 3, precision="e4m3_block"))
    norm = nn.RMSNorm(dev, 300)
    refuses(size, lambda: norm.forward_residual(T((4, 300)), None, T((4, 300), "e4m3"), scales=T((4, 2))))


@pytest.mark.parametrize("rows,F,dtype,residual", [
    (1, 8, "f32", True), (8, 512, "f32", True), (5, 384, "bf16", True), (67, 257, "f32", True),
    (3, 1000, "bf16", True), (130, 48, "bf16", False), (33, 2048, "bf16", True), (9, 4096, "f32", True),
    (7, 5000, "bf16", True), (2, 20004, "f32", True), (301, 384, "f32", False), (1001, 768, "bf16", True),
    (2500, 384, "bf16", True), (300, 136, "bf16", False), (70, 1536, "f32", True), (5, 129, "bf16", True)])
def test_rmsnorm_blocks(dev, stream, rows, F, dtype, residual):
    say(f"rmsnorm blocks {rows}x{F} {dtype} residual {residual}")
    rng = np.random.default_rng(rows * 7 + F)
    x = rounded(outliers(rng, rows, F), dtype)
    r = rounded(rng.standard_normal((rows, F)) * 2, dtype) if residual else None
    w = (1 + 0.2 * rng.standard_normal(F)).astype(np.float32)
    layer = nn.RMSNorm(dev, F, 1e-5)
    layer.load_parameters(w)
    nb = blocks_of(F)
    ht, yt, st = nn.Tensor(dev, (rows, F), dtype=dtype), nn.Tensor(dev, (rows, F), dtype="e4m3"), nn.Tensor(
        dev, (rows, nb))
    layer.forward_residual(tensor(dev, x, dtype), tensor(dev, r, dtype) if residual else None, yt, sum=ht,
                           scales=st, stream=stream)
    stream.sync(60000)
    h = x + r if residual else x
    np.testing.assert_array_equal(ht.to_numpy(), rounded(h, dtype))
    y = rmsnorm(h.astype(np.float64), w, 1e-5)
    rel = (F / 64 + 24) * EPS  # as of the norm's other outputs
    gy, gs = yt.to_numpy(), st.to_numpy()
    top = np.stack([np.abs(y[:, j * 128:(j + 1) * 128]).max(-1) for j in range(nb)], -1)
    want = np.maximum(top, TINY) / 448
    check(gs, want, (rel + 4 * EPS) * want, "scales")
    each = spread_scales(gs, y.shape)
    unit = np.abs(y) / each
    step = np.maximum(unit * HALF["e4m3"], 2.0 ** -10)
    check(gy * each, y, (step * (1 + 1e-5) + unit * (rel + 8 * EPS) + 448 * 2 * rel) * each, "out")


def test_rmsnorm_blocks_of_zeros_and_not_finite(dev, stream):
    say("rmsnorm odd blocks")
    for F in (384, 389):
        x = np.random.default_rng(3).standard_normal((4, F)).astype(np.float32)
        x[1] = 0
        x[2, 5] = np.nan
        yt, st = nn.Tensor(dev, (4, F), dtype="e4m3"), nn.Tensor(dev, (4, blocks_of(F)))
        nn.RMSNorm(dev, F).forward_residual(tensor(dev, x, "f32"), None, yt, scales=st, stream=stream)
        stream.sync(60000)
        y, s = yt.to_numpy(), st.to_numpy()
        assert (y[1] == 0).all() and (s[1] == TINY * np.float32(1 / 448)).all()
        assert np.isnan(y[2] * spread_scales(s, y.shape)[2]).all()
        assert np.isfinite(y[[0, 3]]).all() and np.isfinite(s[[0, 3]]).all()


# ------------------------------------------------------------------------- rolling caches
def cache_case(dev, stream, B, T, KV, hd, sinks, slots, dtype, held, pos, steps=None, seed=0):
    rng = np.random.default_rng(seed + B + T * 3 + slots)
    w = KV * hd
    x = [rounded(rng.standard_normal((B, T, w)) * np.exp(rng.standard_normal((B, T, 1))), dtype) for _ in "kv"]
    n = [0 if p < 0 or p > 2 ** 31 - 1 - T else T if steps is None else min(max(steps[b], 0), T)
         for b, p in enumerate(pos)]
    for b in range(B):
        x[0][b, n[b]:] = np.nan  # rows that are no tokens
    layer = nn.KVCache(dev, KV, hd, sinks)
    kind = "e4m3" if held else dtype
    old = [rounded(rng.standard_normal((B, slots, w)), kind) for _ in "kv"]
    olds = [np.exp(rng.standard_normal((B, slots, KV))).astype(np.float32) for _ in "kv"]
    xt, ct = [tensor(dev, v, dtype) for v in x], [tensor(dev, v, kind) for v in old]
    st = [tensor(dev, v, "f32") for v in olds] if held else [None, None]
    pt = tensor(dev, np.array(pos), "i32")
    nt = tensor(dev, np.array(steps), "i32") if steps is not None else None
    for _ in range(2):
        layer.write(*xt, pt, *ct, *st, steps=nt, stream=stream)
    stream.sync(60000)
    for c in range(2):
        want, wants = old[c].copy(), olds[c].copy()
        for b in range(B):
            for i in range(n[b]):  # in order: the last of those that share a slot stays
                at = slot_of(pos[b] + i, sinks, slots)
                if held:
                    want[b, at], wants[b, at] = (r[0] for r in held_rows(x[c][b, i:i + 1], KV))
                else:
                    want[b, at] = x[c][b, i]
        np.testing.assert_array_equal(ct[c].to_numpy(), want)
        if held:
            np.testing.assert_array_equal(st[c].to_numpy(), wants)
        old[c], olds[c] = want, wants
    out = [empty(dev, (B, T, w), dtype, -7) for _ in "kv"]
    layer.read(*ct, pt, *out, *st, steps=nt, stream=stream)
    stream.sync(60000)
    for c in range(2):
        got = out[c].to_numpy()
        for b in range(B):
            assert (got[b, n[b]:] == -7).all()
            at = [slot_of(pos[b] + i, sinks, slots) for i in range(n[b])]
            if not held:
                np.testing.assert_array_equal(got[b, :n[b]], old[c][b, at])
                continue
            want = old[c][b, at].reshape(n[b], KV, hd) * olds[c][b, at][..., None]  # one fp32 product
            np.testing.assert_array_equal(got[b, :n[b]], rounded(want.reshape(n[b], w), dtype))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("held", [True, False])
@pytest.mark.parametrize("B,T,KV,hd,sinks,slots,pos,steps", [
    (1, 1, 1, 8, 0, 1, [0], None), (1, 7, 8, 48, 4, 11, [0], None), (2, 30, 2, 64, 4, 12, [3, 100], None),
    (3, 9, 3, 72, 1, 40, [0, 39, 7], [9, 0, 4]), (2, 5, 1, 128, 33, 35, [30, 31], [100, -3]),
    (4, 3, 5, 32, 0, 3, [-1, 2 ** 31 - 4, 2 ** 31 - 3, 8], None), (1, 300, 2, 96, 2, 301, [5], [257]),
    (2, 64, 4, 16, 10, 64, [2, 9], None), (1, 40, 1, 120, 0, 16, [1000], None)])
def test_cache_write_and_read(dev, stream, B, T, KV, hd, sinks, slots, pos, steps, held, dtype):
    say(f"cache {B}x{T} heads {KV} hd {hd} sinks {sinks} slots {slots} at {pos} steps {steps} {dtype} {held}")
    cache_case(dev, stream, B, T, KV, hd, sinks, slots, dtype, held, pos, steps)


def test_cache_rows_that_are_odd(dev, stream):
    """Rows of zeros, tiny and large ones, infinities and NaN: each row by itself, by the rule."""
    say("cache odd rows")
    rng = np.random.default_rng(5)
    for hd in (8, 48, 128):
        x = rng.standard_normal((1, 6, 2 * hd)).astype(np.float32)
        x[0, 1] = 0
        x[0, 2] *= 1e-36
        x[0, 3] *= 1e37
        x[0, 4, 3], x[0, 5, hd - 1] = np.nan, np.inf
        c, s = [nn.Tensor(dev, (1, 6, 2 * hd), dtype="e4m3") for _ in "kv"], [nn.Tensor(dev, (1, 6, 2)) for _ in "kv"]
        layer, pos = nn.KVCache(dev, 2, hd), tensor(dev, np.zeros(1), "i32")
        xt = [tensor(dev, x, "f32") for _ in "kv"]
        layer.write(*xt, pos, *c, *s, stream=stream)
        back = [nn.Tensor(dev, x.shape) for _ in "kv"]
        layer.read(*c, pos, *back, *s, stream=stream)
        stream.sync(60000)
        got, scales = back[0].to_numpy().reshape(6, 2, hd), s[0].to_numpy()[0]
        rows = x.reshape(6, 2, hd)
        assert (got[1] == 0).all() and (scales[1] == TINY * np.float32(1 / 448)).all()
        assert not np.isfinite(got[4, 0]).any() and not np.isfinite(got[5, 0]).any()
        for i, j in [(0, 0), (3, 1), (4, 1), (5, 1)]:
            err = np.abs(got[i, j].astype(np.float64) - rows[i, j])
            size = np.abs(rows[i, j]).max()
            assert (err <= np.maximum(np.abs(rows[i, j]) * HALF["e4m3"], size / 448 * 2.0 ** -10) * 1.0001).all()
        top = np.abs(rows[2]).max(-1, keepdims=True)  # below 2^-100: the steps are those of 2^-100
        assert (np.abs(got[2].astype(np.float64) - rows[2]) <= TINY / 448 * 2.0 ** -4 + top * HALF["e4m3"]).all()


def test_cache_slots_beyond_32_bit_offsets(dev, stream):
    """Caches of 4.4 GB: rows past 2^32 bytes."""
    say("cache far slots")
    KV, hd, slots = 32, 128, (1 << 20) + 64
    layer = nn.KVCache(dev, KV, hd)
    c = [nn.Tensor(dev, (1, slots, KV * hd), dtype="e4m3") for _ in "kv"]
    s = [nn.Tensor(dev, (1, slots, KV)) for _ in "kv"]
    x = [np.random.default_rng(i).standard_normal((1, 20, KV * hd)).astype(np.float32) for i in (1, 2)]
    pos = tensor(dev, np.array([slots - 12]), "i32")  # runs over the ring's end
    layer.write(*(tensor(dev, v, "f32") for v in x), pos, *c, *s, stream=stream)
    out = [nn.Tensor(dev, (1, 20, KV * hd)) for _ in "kv"]
    layer.read(*c, pos, *out, *s, stream=stream)
    stream.sync(60000)
    for v, o in zip(x, out):
        q, scale = held_rows(v, KV)
        want = q.reshape(1, 20, KV, hd) * scale[..., None]
        np.testing.assert_array_equal(o.to_numpy(), want.reshape(v.shape))


def test_cache_of_more_rows_than_24_bits(dev, stream):
    """2^24 + 70 rows of one head: each is found again, unrounded."""
    T, hd = (1 << 24) + 70, 8
    say(f"cache rows {T}")
    step = rounded(np.random.default_rng(5).standard_normal((4099, hd)), "bf16")
    k = np.tile(step.astype(np.float32), (-(-T // 4099), 1))[:T].reshape(1, T, hd)
    k[0, :, 0] = np.arange(T) % 251  # whole numbers that bf16 holds; 251 and 4099 share no factor
    layer, pos = nn.KVCache(dev, 1, hd, 3), tensor(dev, np.array([0]), "i32")
    rows, kc, vc = tensor(dev, k, "bf16"), *(nn.Tensor(dev, (1, T + 1, hd), dtype="bf16") for _ in "kv")
    layer.write(rows, rows, pos, kc, vc, stream=stream)
    outs = [nn.Tensor(dev, k.shape, dtype="bf16") for _ in "kv"]
    layer.read(kc, vc, pos, *outs, stream=stream)
    stream.sync(60000)
    for out in outs:
        np.testing.assert_array_equal(out.to_numpy(), k)
    for c in (kc, vc):
        np.testing.assert_array_equal(c.to_numpy()[:, :T], k)


def test_cache_refusals(dev, stream):
    say("cache refusals")
    T = lambda shape, dtype="f32": nn.Tensor(dev, shape, dtype=dtype)  # noqa: E731
    conf, arg, size, shp = ("MNN_ERR_INVALID_CONFIGURATION", "MNN_ERR_INVALID_ARGUMENT",
                            "MNN_ERR_BUFFER_SIZE_MISMATCH", "MNN_ERR_SHAPE_MISMATCH")
    for args in ((0, 16), (2, 12), (2, 136), (2, 16, -1)):
        refuses(conf, lambda: nn.KVCache(dev, *args))
    layer = nn.KVCache(dev, 2, 16, 3)
    k, v, pos = T((2, 5, 32)), T((2, 5, 32)), T((2,), "i32")
    c = lambda *s: (T(s or (2, 9, 32), "e4m3"), T(s or (2, 9, 32), "e4m3"))  # noqa: E731
    s = lambda: (T((2, 9, 2)), T((2, 9, 2)))  # noqa: E731
    kc, vc = c()
    ks, vs = s()
    for f in (lambda kc, vc, ks, vs, k=k, v=v, pos=pos, n=None: layer.write(k, v, pos, kc, vc, ks, vs, n),
              lambda kc, vc, ks, vs, k=k, v=v, pos=pos, n=None: layer.read(kc, vc, pos, k, v, ks, vs, n)):
        f(kc, vc, ks, vs)
        refuses(arg, lambda: f(kc, vc, None, None))
        refuses(arg, lambda: f(kc, vc, ks, None))
        refuses(arg, lambda: f(T((2, 9, 32)), T((2, 9, 32)), ks, vs))
        refuses(arg, lambda: f(T((2, 9, 32), "bf16"), T((2, 9, 32), "bf16"), None, None))
        refuses(arg, lambda: f(kc, T((2, 9, 32)), ks, vs))
        refuses(shp, lambda: f(*c(2, 9, 48), ks, vs))
        refuses(shp, lambda: f(*c(1, 9, 32), ks, vs))
        refuses(shp, lambda: f(kc, T((2, 10, 32), "e4m3"), ks, vs))
        refuses(conf, lambda: f(*c(2, 3, 32), ks, vs))
        refuses(shp, lambda: f(kc, vc, T((2, 9)), vs))
        refuses(arg, lambda: f(kc, vc, T((2, 9, 2), "i32"), vs))
        refuses(shp, lambda: f(kc, vc, ks, vs, k=T((2, 4, 32))))
        refuses(arg, lambda: f(kc, vc, ks, vs, k=T((2, 5, 32), "i32"), v=T((2, 5, 32), "i32")))
        refuses(arg, lambda: f(kc, vc, ks, vs, pos=T((2,))))
        refuses(size, lambda: f(kc, vc, ks, vs, pos=T((3,), "i32")))
        refuses(size, lambda: f(kc, vc, ks, vs, n=T((1,), "i32")))
        refuses(arg, lambda: f(kc, vc, ks, vs, n=T((2,))))
    refuses(arg, lambda: layer.write(k, v, pos, kc, kc, ks, vs))
    refuses(arg, lambda: layer.write(k, v, pos, kc, vc, ks, ks))
    refuses(arg, lambda: layer.read(kc, vc, pos, k, k, ks, vs))
    plain = T((2, 9, 32)), T((2, 9, 32))
    refuses(arg, lambda: layer.write(plain[0], plain[1], pos, *plain))
    layer.write(T((2, 0, 32)), T((2, 0, 32)), pos, kc, vc, ks, vs)
    refuses(arg, lambda: nn.KVCache.write(nn.GELU(dev, (4,)), k, v, pos, kc, vc, ks, vs))
    stream.sync(60000)


# ------------------------------------------------------------- steps on rolling caches in 8 bits
class HeldStreams:
    """Token histories of B streams, their 8-bit caches on the GPU, and steps checked against the history as
    such a cache holds it."""

    def __init__(self, dev, B, H, KV, hd, left, sinks, slots, dtype, seed=0, scale=0.0):
        self.dev, self.H, self.KV, self.hd, self.left, self.sinks = dev, H, KV, hd, left, sinks
        self.slots, self.dtype, self.rng, self.scale = slots, dtype, np.random.default_rng(seed), scale
        self.hist = [([], []) for _ in range(B)]
        self.layer = nn.WindowAttention(dev, H, hd, KV, left, 0, sinks, scale)
        # slots that no token has had yet hold NaN, values and scales: nobody may read them
        nan = np.full((B, slots, KV * hd), np.nan, np.float32)
        self.c = [tensor(dev, nan, "e4m3") for _ in "kv"]
        self.s = [tensor(dev, nan[..., :KV], "f32") for _ in "kv"]

    def rows(self, B, T):
        x = self.rng.standard_normal((B, T, self.KV * self.hd)) * np.exp(0.3 * self.rng.standard_normal((B, T, 1)))
        return rounded(1.2 * x, self.dtype)

    def step(self, stream, T, steps=None, idle=()):
        B = len(self.hist)
        pos = [(-1 - b) if b in idle else len(self.hist[b][0]) for b in range(B)]
        q = rounded(self.rng.standard_normal((B, T, self.H * self.hd)) * 1.3, self.dtype)
        k, v = self.rows(B, T), self.rows(B, T)
        n = [0 if b in idle else min(max(steps[b], 0), T) if steps else T for b in range(B)]
        for b in range(B):
            q[b, n[b]:] = k[b, n[b]:] = v[b, n[b]:] = np.nan
        before = [t.to_numpy() for t in (*self.c, *self.s)]
        out = tensor(self.dev, np.full(q.shape, -7, np.float32), self.dtype)
        call = [tensor(self.dev, x, self.dtype) for x in (q, k, v)]
        pt = tensor(self.dev, np.array(pos), "i32")
        st = tensor(self.dev, np.array(steps), "i32") if steps else None
        for _ in range(2):  # the same call again changes nothing
            self.layer.step(*call, pt, *self.c, out, st, stream, *self.s)
        stream.sync(60000)
        got, after = out.to_numpy(), [t.to_numpy() for t in (*self.c, *self.s)]
        for b in range(B):
            assert (got[b, n[b]:] == -7).all(), f"rows behind stream {b}'s last were written"
            for c, x in enumerate((k, v)):
                want, wants = before[c][b].copy(), before[2 + c][b].copy()
                if n[b]:
                    xq, xs = held_rows(x[b, :n[b]], self.KV)
                    self.hist[b][c].extend(values_of(xq, xs))
                    for i in range(n[b]):
                        at = slot_of(pos[b] + i, self.sinks, self.slots)
                        want[at], wants[at] = xq[i], xs[i]
                np.testing.assert_array_equal(after[c][b], want)
                np.testing.assert_array_equal(after[2 + c][b], wants)
            if n[b]:
                p0 = pos[b]
                mine = np.arange(p0, p0 + n[b])[:, None]
                key = np.arange(p0 + n[b])[None]
                seen = (key <= mine) & ((key >= mine - self.left) | (key < self.sinks))
                hk, hv = (np.array(h) for h in self.hist[b])
                want, spread, size = attend(q[b, :n[b]], hk, hv, seen, self.H, self.KV, self.scale or self.hd ** -0.5)
                keys = min(self.left + 1 + self.sinks, p0 + n[b])
                check(got[b, :n[b]], want, held_tolerance(spread, size, self.hd, keys, self.dtype),
                      f"stream {b} at {p0}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,H,KV,hd,left,sinks,spare,chunks", [
    (1, 1, 1, 8, 0, 0, 0, [1, 1, 1]), (1, 8, 8, 48, 11, 4, 0, [1] * 5 + [7, 1, 9, 1, 1, 1]),
    (3, 8, 2, 64, 100, 4, 3, [90, 1, 16, 1, 5, 1, 1]), (2, 4, 1, 128, 63, 0, 1, [64, 1, 1, 3, 1]),
    (2, 6, 3, 72, 5, 33, 0, [20, 1, 20, 1, 1]), (4, 5, 5, 32, 300, 1, 40, [257, 60, 1, 2]),
    (1, 2, 1, 96, 1000, 2, 0, [1200, 1, 1]), (1, 2, 2, 56, 30, 1, 2, [40, 3, 1]), (2, 3, 1, 120, 17, 0, 0, [9, 30, 1]),
    (2, 4, 2, 64, 2500, 5, 3, [2600, 1, 3, 1]), (1, 3, 3, 128, 900, 0, 7, [950, 2, 1]),
    (2, 16, 1, 64, 40, 2, 0, [30, 1, 4, 1]), (1, 64, 1, 40, 70, 0, 0, [3, 1, 80, 1]), (3, 4, 4, 24, 64, 0, 5, [33, 31, 32, 1])])
def test_window_step_held(dev, stream, B, H, KV, hd, left, sinks, spare, chunks, dtype):
    say(f"8-bit step {B} streams heads {H}/{KV} hd {hd} left {left} sinks {sinks} chunks {chunks} {dtype}")
    s = HeldStreams(dev, B, H, KV, hd, left, sinks, sinks + left + max(chunks) + spare, dtype)
    for T in chunks:
        s.step(stream, T)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_window_step_held_ragged_streams(dev, stream, dtype):
    say(f"8-bit step ragged {dtype}")
    s = HeldStreams(dev, 5, 4, 2, 48, 20, 3, 3 + 20 + 9, dtype, scale=-0.3)
    s.step(stream, 9, [9, 4, 0, 1, 100])
    s.step(stream, 4, [-5, 4, 3, 4, 2], idle=(3,))
    s.step(stream, 1)
    s.step(stream, 9, [9, 9, 9, 9, 9], idle=(0,))
    s.step(stream, 9, [1, 9, 2, 9, 9])
    s.step(stream, 1, idle=(1, 2))


@pytest.mark.parametrize("dtype,hd,KV,T", [("f32", 48, 2, 1), ("bf16", 64, 1, 1), ("bf16", 64, 2, 16)])
def test_window_step_held_far_positions(dev, stream, dtype, hd, KV, T):
    """Positions near the largest that a call takes; one beyond it leaves the stream alone."""
    say(f"8-bit step far {dtype} {T}")
    left, sinks, slots = 30, 2, 60
    layer = nn.WindowAttention(dev, 2, hd, KV, left, 0, sinks)
    rng = np.random.default_rng(31)
    w = KV * hd
    c, s = zip(*(held_rows(rng.standard_normal((2, slots, w)), KV) for _ in "kv"))
    q = rounded(rng.standard_normal((2, T, 2 * hd)), dtype)
    new = [rounded(rng.standard_normal((2, T, w)), dtype) for _ in "kv"]
    p = 2 ** 31 - 1 - T
    ct, st = [tensor(dev, x, "e4m3") for x in c], [tensor(dev, x, "f32") for x in s]
    out = empty(dev, q.shape, dtype, -7)
    layer.step(tensor(dev, q, dtype), *(tensor(dev, x, dtype) for x in new),
               tensor(dev, np.array([p, p + 1]), "i32"), *ct, out, None, stream, *st)
    stream.sync(60000)
    got = out.to_numpy()
    for t in range(T):
        old = list(range(sinks)) + [slot_of(i, sinks, slots) for i in range(p + t - left, p)]
        kk, vv = (np.concatenate([values_of(c[i][0, old], s[i][0, old]),
                                  values_of(*held_rows(new[i][0, :t + 1], KV))]) for i in (0, 1))
        want, spread, size = attend(q[0, t:t + 1], kk, vv, np.ones((1, len(kk)), bool), 2, KV, hd ** -0.5)
        check(got[0, t:t + 1], want, held_tolerance(spread, size, hd, len(kk), dtype), "far")
    assert (got[1] == -7).all()
    np.testing.assert_array_equal(ct[0].to_numpy()[1], c[0][1])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_window_step_held_blocks_equal_single_tokens(dev, stream, dtype):
    """T tokens in one call see what they see one after the other: the caches end up the same, the
    outputs within their roundings."""
    say(f"8-bit step blocks {dtype}")
    a, b = (HeldStreams(dev, 2, 4, 2, 48, 13, 2, 2 + 13 + 8, dtype, seed=9) for _ in range(2))
    rng = np.random.default_rng(9)
    q, k, v = (rounded(rng.standard_normal((2, 24, n * 48)), dtype) for n in (4, 2, 2))

    def run(m, size):
        outs = []
        for i in range(0, 24, size):
            o = nn.Tensor(dev, (2, size, 4 * 48), dtype=dtype)
            m.layer.step(*(tensor(dev, x[:, i:i + size], dtype) for x in (q, k, v)),
                         tensor(dev, np.full(2, i), "i32"), *m.c, o, None, stream, *m.s)
            stream.sync(60000)
            outs.append(o.to_numpy())
        return np.concatenate(outs, 1)

    one, eight = run(a, 1), run(b, 8)
    for x, y in zip((*a.c, *a.s), (*b.c, *b.s)):
        np.testing.assert_array_equal(x.to_numpy(), y.to_numpy())
    hk, hv = (values_of(*held_rows(x, 2)) for x in (k, v))
    i = np.arange(24)
    seen = (i[None] <= i[:, None]) & ((i[None] >= i[:, None] - 13) | (i[None] < 2))
    for s in range(2):
        want, spread, size = attend(q[s], hk[s], hv[s], seen, 4, 2, 48 ** -0.5)
        tol = held_tolerance(spread, size, 48, 16, dtype)
        check(one[s], want, tol, "one by one")
        check(eight[s], want, tol, "by eights")


def test_window_step_held_after_a_prompt(dev, stream):
    """A prompt through the cache's write and whole-sequence attention, then steps that read it."""
    say("8-bit step after a prompt")
    H, KV, hd, left, sinks, S = 4, 2, 64, 50, 3, 333
    m = HeldStreams(dev, 1, H, KV, hd, left, sinks, sinks + left + 4, "bf16", seed=2)
    k, v = m.rows(1, S), m.rows(1, S)
    nn.KVCache(dev, KV, hd, sinks).write(*(tensor(dev, x, "bf16") for x in (k, v)), tensor(dev, np.zeros(1), "i32"),
                                         *m.c, *m.s, stream=stream)
    for c, x in enumerate((k, v)):
        m.hist[0][c].extend(values_of(*held_rows(x[0], KV)))
    for T in (1, 4, 1):
        m.step(stream, T)


def test_window_step_held_refusals(dev, stream):
    say("8-bit step refusals")
    T = lambda shape, dtype="f32": nn.Tensor(dev, shape, dtype=dtype)  # noqa: E731
    conf, arg, shp = "MNN_ERR_INVALID_CONFIGURATION", "MNN_ERR_INVALID_ARGUMENT", "MNN_ERR_SHAPE_MISMATCH"
    layer = nn.WindowAttention(dev, 4, 16, 2, window_left=3, sinks=1)
    q, k, v, o, pos = T((2, 5, 64)), T((2, 5, 32)), T((2, 5, 32)), T((2, 5, 64)), T((2,), "i32")
    c, s = [T((2, 9, 32), "e4m3") for _ in "kv"], [T((2, 9, 2)) for _ in "kv"]

    def f(c=c, s=s, o=o, pos=pos, steps=None):
        layer.step(q, k, v, pos, *c, o, steps, stream, *s)

    f()
    refuses(arg, lambda: f(c=[T((2, 9, 32)) for _ in "kv"]))
    refuses(arg, lambda: f(s=[s[0], None]))
    refuses(arg, lambda: f(s=[None, s[1]]))
    refuses(arg, lambda: layer.step(q, k, v, pos, *c, o))
    refuses(arg, lambda: f(s=[s[0], s[0]]))
    refuses(arg, lambda: f(s=[T((2, 9, 2), "bf16"), s[1]]))
    refuses(shp, lambda: f(s=[T((2, 9, 4)), s[1]]))
    refuses(shp, lambda: f(s=[T((2, 8, 2)), s[1]]))
    refuses(conf, lambda: f(c=[T((2, 8, 32), "e4m3") for _ in "kv"], s=[T((2, 8, 2)) for _ in "kv"]))
    refuses(arg, lambda: f(o=q))
    refuses(arg, lambda: f(pos=T((2,))))
    both = nn.WindowAttention(dev, 4, 16, 2, window_left=3, window_right=1)
    refuses(conf, lambda: both.step(q, k, v, pos, *c, o, None, stream, *s))
    stream.sync(60000)


# -------------------------------------------------------------- attention to an encoder's states
def memory_case(dev, stream, B, T, S, H, KV, hd, dtype, held, lengths=None, queries=None, scale=0.0, q=None, k=None,
                v=None, tight=True, seed=0):
    rng = np.random.default_rng(seed + B * 11 + T * 5 + S)
    draw = lambda n, w, std: rng.standard_normal((B, n, w)) * std * np.exp(0.3 * rng.standard_normal((B, n, 1)))  # noqa: E731
    q = rounded(draw(T, H * hd, 1.3) if q is None else q, dtype)
    k, v = (rounded(draw(S, KV * hd, 1.2) if x is None else x, dtype) for x in (k, v))
    scales, kind = [None, None], dtype
    if held:
        (k, ks), (v, vs) = held_rows(k, KV), held_rows(v, KV)
        scales, kind = [ks, vs], "e4m3"
    n = [S if lengths is None else min(max(lengths[b], 0), S) for b in range(B)]
    m = [T if queries is None else min(max(queries[b], 0), T) for b in range(B)]
    for b in range(B):  # what stands behind the ends is nobody's
        k[b, n[b]:] = v[b, n[b]:] = np.nan
        q[b, m[b]:] = np.nan
        if held:
            ks[b, n[b]:] = vs[b, n[b]:] = np.nan
    layer = nn.MemoryAttention(dev, H, hd, KV, scale)
    out = empty(dev, q.shape, dtype, -7)
    i32 = lambda x: None if x is None else tensor(dev, np.array(x), "i32")  # noqa: E731
    args = [tensor(dev, q, dtype), tensor(dev, k, kind), tensor(dev, v, kind), out, i32(queries), i32(lengths)]
    args += [None if x is None else tensor(dev, x, "f32") for x in scales]
    layer.forward(*args, stream=stream)
    stream.sync(60000)
    got = out.to_numpy()
    for b in range(B):
        assert (got[b, m[b]:] == -7).all(), f"rows behind sequence {b}'s last were written"
        kk, vv = ((values_of(x[b, :n[b]], s[b, :n[b]]) if held else x[b, :n[b]]) for x, s in zip((k, v), scales))
        want, spread, size = memory(q[b, :m[b]], kk, vv, H, KV, scale or hd ** -0.5)
        tol = (held_tolerance if held else split_tolerance)(spread, size, hd, n[b], dtype)
        check(got[b, :m[b]], want, tol, f"sequence {b}")
    return got


MEMORY = [
    (1, 1, 1, 1, 1, 8, {}), (1, 1, 33, 8, 8, 48, {}), (2, 3, 0, 2, 1, 16, {}), (1, 1, 1344, 8, 8, 48, {}),
    (3, 1, 700, 8, 2, 64, {"lengths": [700, 0, 1]}), (2, 5, 129, 6, 3, 72, {"lengths": [64, 129], "queries": [5, 2]}),
    (1, 31, 64, 4, 1, 128, {}), (1, 33, 65, 3, 3, 40, {}), (4, 16, 300, 16, 4, 64, {"lengths": [300, -4, 999, 31]}),
    (1, 61, 512, 8, 8, 48, {"scale": 0.4}), (2, 130, 40, 5, 5, 32, {"queries": [0, 130]}),
    (1, 200, 1000, 4, 2, 96, {}), (2, 257, 515, 8, 2, 64, {"lengths": [515, 200], "queries": [257, 100]}),
    (1, 700, 640, 2, 2, 120, {"scale": -0.05}), (1, 1344, 333, 8, 8, 48, {}), (1, 40, 2000, 64, 1, 24, {}),
    (2, 1, 5000, 2, 1, 56, {"lengths": [5000, 37]}), (1, 7, 96, 7, 7, 80, {}), (1, 515, 1030, 1, 1, 128, {}),
    (70, 1, 90, 4, 4, 64, {}), (1, 2000, 31, 3, 1, 104, {})]


@pytest.mark.parametrize("held", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,S,H,KV,hd,kw", MEMORY)
def test_memory_attention(dev, stream, B, T, S, H, KV, hd, kw, dtype, held):
    say(f"memory {B}x{T} on {S} heads {H}/{KV} hd {hd} {kw} {dtype} held {held}")
    memory_case(dev, stream, B, T, S, H, KV, hd, dtype, held, **kw)


@pytest.mark.parametrize("held", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,S,kw", [
    (3, 150, 700, {"lengths": [700, 1, 513]}), (6, 70, 100, {"queries": [70, 69, 0, 1, 33, 64]}),
    (8, 900, 90, {"lengths": [90, 0, 64, 65, 1, 31, 33, 90], "queries": [900, 769, 768, 513, 900, 1, 0, 257]}),
    (8, 800, 520, {"lengths": [520, 300, 520, 257, 10, 512, 511, 260]})])
@pytest.mark.parametrize("hd", [16, 40, 48, 64, 72, 96, 128])
def test_memory_attention_many_rows(dev, stream, B, T, S, kw, hd, dtype, held):
    say(f"memory rows {B}x{T} on {S} hd {hd} {kw} {dtype} held {held}")
    KV = 4 if B < 8 else 8
    memory_case(dev, stream, B, T, S, KV, KV, hd, dtype, held, **kw)


@pytest.mark.parametrize("held", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,S", [(1, 900), (40, 333), (300, 200), (600, 200)])
def test_memory_attention_sizes(dev, stream, T, S, dtype, held):
    """Scores from tiny to hundreds, rising along the keys, and values of all sizes."""
    say(f"memory sizes {T} on {S} {dtype} held {held}")
    rng = np.random.default_rng(7)
    H, hd = 2, 64
    ramp = np.sort(rng.standard_normal((1, S, 1)) * 30, axis=1) * np.ones((1, S, H * hd)) / 7
    sign = np.full((1, T, H * hd), 30.0) * np.sign(rng.standard_normal((1, T, 1)))
    memory_case(dev, stream, 1, T, S, H, H, hd, dtype, held, q=sign, k=ramp)
    memory_case(dev, stream, 1, T, S, H, H, hd, dtype, held, q=1e-3 * sign, k=1e-5 * ramp)
    for size in (1e-30, 1e30):
        memory_case(dev, stream, 1, T, S, H, H, hd, dtype, held, v=rng.standard_normal((1, S, H * hd)) * size)


@pytest.mark.parametrize("T", [1, 50, 300, 8192])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_memory_attention_not_finite(dev, stream, T, dtype):
    """A NaN or an infinity among the values reaches its head and dimension, a NaN key its head; other
    heads and sequences keep their results."""
    say(f"memory not finite {T} {dtype}")
    rng = np.random.default_rng(8)
    B, S, H, KV, hd = 2, 150, 4, 2, 48
    q, k, v = (rounded(rng.standard_normal((B, n, w * hd)), dtype) for n, w in ((T, H), (S, KV), (S, KV)))
    layer = nn.MemoryAttention(dev, H, hd, KV)

    def run(k, v):
        out = nn.Tensor(dev, q.shape, dtype=dtype)
        layer.forward(*(tensor(dev, x, dtype) for x in (q, k, v)), out, stream=stream)
        stream.sync(60000)
        return out.to_numpy().reshape(B, T, KV, H // KV, hd)

    clean = run(k, v)
    want, spread, size = memory(q[1], k[1], v[1], H, KV, hd ** -0.5)
    tol = split_tolerance(spread, size, hd, S, dtype)
    head = np.s_[:, 1, :, np.arange(hd) != 5]
    want, tol = (x.reshape(T, KV, H // KV, hd)[head] for x in (want, tol))
    for bad in (np.nan, np.inf, -np.inf):
        v2 = v.copy()
        v2[1, 77, hd + 5] = bad
        got = run(k, v2)
        np.testing.assert_array_equal(got[0], clean[0])
        np.testing.assert_array_equal(got[1, :, 0], clean[1, :, 0])
        np.testing.assert_array_equal(got[1, :, 1, :, 5], np.full((T, H // KV), bad))
        check(got[1][head], want, tol, f"beside {bad}")
    k2 = k.copy()
    k2[0, 149, 3] = np.nan
    got = run(k2, v)
    assert np.isnan(got[0, :, 0]).all()
    np.testing.assert_array_equal(got[0, :, 1], clean[0, :, 1])
    np.testing.assert_array_equal(got[1], clean[1])
    # scores of -infinity count for nothing beside finite ones
    k2 = k.copy()
    k2[0, 20, :hd] = np.where(np.arange(hd) == 3, np.inf, 0)
    q2 = q.copy()
    q2[0, :, 3::hd] = -1
    out = nn.Tensor(dev, q.shape, dtype=dtype)
    layer.forward(tensor(dev, q2, dtype), tensor(dev, k2, dtype), tensor(dev, v, dtype), out, stream=stream)
    stream.sync(60000)
    keep = np.arange(S) != 20
    want, spread, size = memory(q2[0], k2[0, keep], v[0, keep], H, KV, hd ** -0.5)
    got = out.to_numpy()[0].reshape(T, KV, H // KV, hd)[:, 0]
    first = slice(0, H // KV * hd)
    check(got.reshape(T, -1), want[:, first], split_tolerance(spread, size, hd, S, dtype)[:, first], "-inf")


def test_memory_attention_states_beyond_32_bit_offsets(dev, stream):
    """8-bit states of 4.4 GB, of which the last sequence's lie past 2^32 bytes."""
    say("memory far states")
    B, S, H, hd = 40, 1 << 15, 32, 128
    k, v = (nn.Tensor(dev, (B, S, H * hd), dtype="e4m3") for _ in "kv")
    ks, vs = (nn.Tensor(dev, (B, S, H)) for _ in "kv")
    rng = np.random.default_rng(13)
    n = 300
    rows = [rounded(rng.standard_normal((B, n, H * hd)), "bf16") for _ in "kv"]
    nn.KVCache(dev, H, hd).write(*(tensor(dev, r, "bf16") for r in rows), tensor(dev, np.zeros(B), "i32"), k, v, ks, vs,
                                 stream=stream)
    q = rounded(rng.standard_normal((B, 2, H * hd)), "bf16")
    out = nn.Tensor(dev, q.shape, dtype="bf16")
    nn.MemoryAttention(dev, H, hd).forward(tensor(dev, q, "bf16"), k, v, out, lengths=tensor(dev, np.full(B, n), "i32"),
                                           k_scales=ks, v_scales=vs, stream=stream)
    stream.sync(60000)
    got = out.to_numpy()
    for b in (0, B - 1):
        want, spread, size = memory(q[b], *(values_of(*held_rows(r[b], H)) for r in rows), H, H, hd ** -0.5)
        check(got[b], want, held_tolerance(spread, size, hd, n, "bf16"), f"sequence {b}")


def test_memory_attention_refusals(dev, stream):
    say("memory refusals")
    T = lambda shape, dtype="f32": nn.Tensor(dev, shape, dtype=dtype)  # noqa: E731
    conf, arg, size, shp = ("MNN_ERR_INVALID_CONFIGURATION", "MNN_ERR_INVALID_ARGUMENT",
                            "MNN_ERR_BUFFER_SIZE_MISMATCH", "MNN_ERR_SHAPE_MISMATCH")
    for kw in (dict(num_heads=3, head_dim=16, num_kv_heads=2), dict(num_heads=2, head_dim=12),
               dict(num_heads=2, head_dim=136), dict(num_heads=0, head_dim=16),
               dict(num_heads=2, head_dim=16, scale=float("nan"))):
        refuses(conf, lambda: nn.MemoryAttention(dev, **kw))
    layer = nn.MemoryAttention(dev, 4, 16, 2)
    q, k, v, o = T((2, 5, 64)), T((2, 9, 32)), T((2, 9, 32)), T((2, 5, 64))
    f = layer.forward
    f(q, k, v, o, stream=stream)
    f(T((5, 64)), T((9, 32)), T((9, 32)), T((5, 64)), stream=stream)
    refuses(shp, lambda: f(T((2, 5, 32)), k, v, o))
    refuses(shp, lambda: f(q, T((2, 8, 32)), v, o))
    refuses(shp, lambda: f(q, T((1, 9, 32)), T((1, 9, 32)), o))
    refuses(shp, lambda: f(q, T((2, 9, 64)), T((2, 9, 64)), o))
    refuses(arg, lambda: f(q, T((2, 9, 32), "bf16"), T((2, 9, 32), "bf16"), o))
    refuses(arg, lambda: f(q, T((2, 9, 32), "e4m3"), T((2, 9, 32), "e4m3"), o))
    refuses(arg, lambda: f(q, k, v, T((2, 5, 64), "bf16")))
    refuses(size, lambda: f(q, k, v, T((2, 4, 64))))
    refuses(arg, lambda: f(q, k, v, q))
    refuses(arg, lambda: f(q, k, v, o, T((2,))))
    refuses(size, lambda: f(q, k, v, o, T((3,), "i32")))
    refuses(size, lambda: f(q, k, v, o, lengths=T((1,), "i32")))
    refuses(arg, lambda: f(q, k, v, o, k_scales=T((2, 9, 2)), v_scales=T((2, 9, 2))))
    e = T((2, 9, 32), "e4m3")
    refuses(arg, lambda: f(q, e, e, o, k_scales=T((2, 9, 2))))
    refuses(shp, lambda: f(q, e, e, o, k_scales=T((2, 9, 2)), v_scales=T((2, 9, 1))))
    one = nn.MemoryAttention(dev, 1, 8)
    x = T((1, 1, 8))
    refuses(arg, lambda: one.forward(T((1, 1, 8)), x, T((1, 1, 8)), x))
    refuses(conf, lambda: nn.Layer.forward(layer, q, o))
    refuses(arg, lambda: nn.MemoryAttention.forward(nn.GELU(dev, (4,)), q, k, v, o))
    f(T((2, 0, 64)), k, v, T((2, 0, 64)), stream=stream)
    stream.sync(60000)


# ------------------------------------------------------------------------ together, and captured
class Decoder:
    """A decoder block on live streams: norm to 8 bits in blocks, q, k and v, the step on 8-bit rolling caches,
    the output product with the residual; norm, q, attention to the encoder's states in 8 bits, output product."""

    def __init__(self, dev, B, E, heads, left, sinks, S, dtype, seed=0):
        self.dev, self.B, self.E, self.H, self.hd, self.dtype = dev, B, E, heads, E // heads, dtype
        rng = np.random.default_rng(seed)
        names = ("q", "k", "v", "o", "mq", "mo")
        self.w = {n: (rng.standard_normal((E, E)) / np.sqrt(E)).astype(np.float32) for n in names}
        self.b = {n: (0.1 * rng.standard_normal(E)).astype(np.float32) for n in names}
        self.lin = {}
        for n in names:
            self.lin[n] = nn.Linear(dev, E, E, precision="e4m3_block")
            self.lin[n].load_weights(self.w[n], self.b[n])
        self.norm = nn.RMSNorm(dev, E)
        self.left, self.sinks, self.slots, self.S = left, sinks, sinks + left + 1, S
        self.att = nn.WindowAttention(dev, heads, self.hd, window_left=left, sinks=sinks)
        self.mem = nn.MemoryAttention(dev, heads, self.hd)
        T = lambda dt, *shape: nn.Tensor(dev, shape, dtype=dt)  # noqa: E731
        nb = blocks_of(E)
        self.x = T(dtype, B, 1, E)
        self.n8, self.s = T("e4m3", B, 1, E), T("f32", B, nb)
        self.m8, self.ms = T("e4m3", B, 1, E), T("f32", B, nb)
        self.t = {n: T(dtype, B, 1, E) for n in (*names, "a", "ma")}
        self.c, self.cs = [T("e4m3", B, self.slots, E) for _ in "kv"], [T("f32", B, self.slots, heads) for _ in "kv"]
        self.states = [T("e4m3", B, S, E) for _ in "kv"]
        self.state_scales = [T("f32", B, S, heads) for _ in "kv"]
        self.lengths, self.pos, self.zero = T("i32", B), T("i32", B), T("i32", B)
        self.cache = nn.KVCache(dev, heads, self.hd)

    def encode(self, k, v, lengths, stream):
        """The encoder's states, once."""
        self.lengths.copy_from(np.array(lengths))
        self.cache.write(*(tensor(self.dev, x, self.dtype) for x in (k, v)), self.zero, *self.states, *self.state_scales,
                         steps=self.lengths, stream=stream)
        stream.sync(60000)

    def run(self, stream):
        t = self.t
        self.norm.forward_residual(self.x, None, self.n8, scales=self.s, stream=stream)
        for n in "qkv":
            self.lin[n].forward_scaled(self.n8, self.s, t[n], stream=stream)
        self.att.step(t["q"], t["k"], t["v"], self.pos, *self.c, t["a"], None, stream, *self.cs)
        self.lin["o"].forward_scaled(t["a"], None, t["o"], residual=self.x, stream=stream)
        self.norm.forward_residual(t["o"], None, self.m8, scales=self.ms, stream=stream)
        self.lin["mq"].forward_scaled(self.m8, self.ms, t["mq"], stream=stream)
        self.mem.forward(t["mq"], *self.states, t["ma"], lengths=self.lengths, k_scales=self.state_scales[0],
                         v_scales=self.state_scales[1], stream=stream)
        self.lin["mo"].forward_scaled(t["ma"], None, t["mo"], residual=t["o"], stream=stream)


def blocks_reference(xq, xs, w, b, dtype):
    y, mass = linear_blocks(xq, xs, *quantise_tiles(w), b)
    K = xq.shape[-1]
    return y, ((1.5 * K + 3 * blocks_of(K) + 8) * EPS * (mass + np.abs(y) + 0.5)
               + HALF[dtype] * np.abs(y) * (dtype != "f32"))


@pytest.mark.parametrize("B,E,heads,S,dtype", [(4, 384, 8, 100, "bf16"), (2, 96, 2, 1400, "f32")])
def test_decoder_on_streams(dev, stream, B, E, heads, S, dtype):
    """Every stage against its reference on what the GPU gave the stage before it."""
    say(f"decoder {B} streams E {E} on {S} states {dtype}")
    m = Decoder(dev, B, E, heads, 9, 2, S, dtype)
    rng = np.random.default_rng(61)
    ek, ev = (rounded(rng.standard_normal((B, S, E)), dtype) for _ in "kv")
    lengths = [S, 0, S // 2, 1][:B]
    m.encode(ek, ev, lengths, stream)
    ek, ev = (values_of(*held_rows(x, heads)) for x in (ek, ev))
    hist = [([], []) for _ in range(B)]
    for p in range(14):
        x = rounded(rng.standard_normal((B, 1, E)), dtype)
        m.x.copy_from(x)
        m.pos.copy_from(np.full(B, p))
        m.run(stream)
        stream.sync(60000)
        got = {n: t.to_numpy() for n, t in m.t.items()}
        for n8, s, source in ((m.n8, m.s, x), (m.m8, m.ms, got["o"])):
            y = rmsnorm(source[:, 0].astype(np.float64), np.ones(E), 1e-5)
            each = spread_scales(s.to_numpy(), y.shape)
            step = np.maximum(np.abs(y) / each * HALF["e4m3"], 2.0 ** -10) * (1 + 1e-5) + 448 * 80 * EPS
            check(n8.to_numpy()[:, 0] * each, y, step * each, "norm")
        for n in "qkv":
            want, tol = blocks_reference(m.n8.to_numpy()[:, 0], m.s.to_numpy(), m.w[n], m.b[n], dtype)
            check(got[n][:, 0], want, tol, n)
        want, tol = blocks_reference(m.m8.to_numpy()[:, 0], m.ms.to_numpy(), m.w["mq"], m.b["mq"], dtype)
        check(got["mq"][:, 0], want, tol, "mq")
        for b in range(B):
            for c, n in enumerate("kv"):
                hist[b][c].extend(values_of(*held_rows(got[n][b], heads)))
            keys = [i for i in range(p + 1) if i >= p - m.left or i < m.sinks]
            kk, vv = (np.array(h)[keys] for h in hist[b])
            want, spread, size = memory(got["q"][b], kk, vv, heads, heads, m.hd ** -0.5)
            check(got["a"][b], want, held_tolerance(spread, size, m.hd, len(keys), dtype), "step")
            n = lengths[b]
            want, spread, size = memory(got["mq"][b], ek[b, :n], ev[b, :n], heads, heads, m.hd ** -0.5)
            check(got["ma"][b], want, held_tolerance(spread, size, m.hd, n, dtype), "memory")
        for a, o, r in (("a", "o", x), ("ma", "mo", got["o"])):
            want, tol = blocks_reference(*quantise_blocks(got[a][:, 0]), m.w[o], m.b[o], dtype)
            want = want + r[:, 0]
            check(got[o][:, 0], want, tol + (HALF[dtype] if dtype != "f32" else EPS) * np.abs(want), o)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decoder_captured_and_replayed(dev, dtype):
    """The block in a graph, replayed with other inputs and positions and eager work of the same layers between
    the replays (also larger calls, which grow their workspaces), equals the eager block."""
    say(f"decoder captured {dtype}")
    s, other = nn.Stream(dev), nn.Stream(dev)
    B, E, S = 2, 192, 2000
    eager, taken = (Decoder(dev, B, E, 4, 1500, 2, S, dtype) for _ in range(2))  # split keys: workspaces
    rng = np.random.default_rng(62)
    ek, ev = (rounded(rng.standard_normal((B, S, E)), dtype) for _ in "kv")
    for m in (eager, taken):  # workspaces are made by a call outside the graph
        m.encode(ek, ev, [S, 700], s)
        m.run(s)
    s.sync(60000)
    graph = Graph(s, lambda: taken.run(s))
    for i in range(6):
        x = rounded(rng.standard_normal((B, 1, E)), dtype)
        for m in (eager, taken):
            m.x.copy_from(x)
            m.pos.copy_from(np.array([3 * i, 3000 + i]))
            m.lengths.copy_from(np.array([S - i, 300 * i]))
        eager.run(other)
        graph.replay()
        s.sync(60000)
        other.sync(60000)
        for n in eager.t:
            np.testing.assert_array_equal(taken.t[n].to_numpy(), eager.t[n].to_numpy())
        for a, b in zip(taken.c, eager.c):
            np.testing.assert_array_equal(a.to_numpy(), b.to_numpy())
        # other calls of the captured layers, on their stream, larger than any before
        big = tensor(dev, rng.standard_normal((40 + 30 * i, E)), dtype)
        taken.lin["o"].forward_scaled(big, None, nn.Tensor(dev, (40 + 30 * i, E), dtype=dtype), stream=s)
        n = 20 + 10 * i
        qkv = [tensor(dev, rng.standard_normal((3, n, E)), dtype) for _ in range(3)]
        caches = [nn.Tensor(dev, (3, 1502 + n, E), dtype="e4m3") for _ in "kv"]
        scales = [nn.Tensor(dev, (3, 1502 + n, 4)) for _ in "kv"]
        taken.att.step(*qkv, tensor(dev, np.array([0, 9, 800]), "i32"), *caches,
                       nn.Tensor(dev, (3, n, E), dtype=dtype), None, s, *scales)
        taken.mem.forward(qkv[0], *caches, nn.Tensor(dev, (3, n, E), dtype=dtype), k_scales=scales[0],
                          v_scales=scales[1], stream=s)
        s.sync(60000)


def test_decoder_calls_on_many_streams(dev):
    """The same work on several streams at once, one layer a stream, and on the default stream: the same bits."""
    say("decoder streams")
    rng = np.random.default_rng(63)
    H, hd, dtype = 4, 48, "f32"
    for T, S in ((3, 1500), (200, 700)):
        x = [rng.standard_normal((2, n, H * hd)).astype(np.float32) for n in (T, S, S)]
        jobs = []
        for stream in [None] + [nn.Stream(dev) for _ in range(4)]:
            layer, out = nn.MemoryAttention(dev, H, hd), nn.Tensor(dev, x[0].shape)
            args = [tensor(dev, v, dtype) for v in x]
            layer.forward(*args, out, stream=stream)
            jobs.append((layer, out, args, stream))
        dev.synchronize()
        for _, out, _, _ in jobs:
            np.testing.assert_array_equal(out.to_numpy(), jobs[0][1].to_numpy())
