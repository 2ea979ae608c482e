"""What the decoder's layers hold of the device and keep from call to call, and calls near the ends of what they take, through
the C ABI. Tolerances count roundings (token_refs.py, decoder_refs.py) and were fixed before the first run."""
import ctypes as C

import numpy as np
import pytest

from metalaudio_amd import nn
from metalaudio_amd._lib import check as ok
from metalaudio_amd._lib import lib
from tests.decoder_refs import (blocks_of, held_rows, held_tolerance, linear_blocks, memory, quantise_blocks,
                                quantise_tiles, values_of)
from tests.test_gpu_tokens import Graph, check, tensor
from tests.token_refs import EPS, rounded, slot_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return nn.AudioDevice(0)


def say(msg):
    print(f"[case] {msg}", flush=True)


def allocations():
    n = C.c_int64()
    ok(lib().mnn_debug_device_allocations(C.byref(n)))
    return n.value


def hip():
    path = next(ln.split()[-1] for ln in open("/proc/self/maps") if "libamdhip64" in ln)
    return C.CDLL(path)


def test_attention_layers_are_made_without_the_device(dev):
    """Making one neither allocates nor waits, so that it can be made while a stream is being captured."""
    say("attention layers without the device")
    s, graph = nn.Stream(dev), C.c_void_p()
    handle = C.c_void_p(C.cast(s.handle, C.POINTER(C.c_void_p))[1])
    before = allocations()
    assert hip().hipStreamBeginCapture(handle, 0) == 0
    try:
        layers = [nn.WindowAttention(dev, 4, 48, 2, window_left=9, sinks=1), nn.MemoryAttention(dev, 4, 48, 2),
                  nn.KVCache(dev, 2, 48, 1)]
    finally:
        ended = hip().hipStreamEndCapture(handle, C.byref(graph))
    assert ended == 0 and allocations() == before and len(layers) == 3


class MemoryCall:
    """A call on keys that several workgroups share out."""

    def __init__(self, dev, B, T, S, H, hd, dtype, seed):
        rng = np.random.default_rng(seed)
        self.args = [tensor(dev, rng.standard_normal((B, n, H * hd)), dtype) for n in (T, S, S)]
        self.out = nn.Tensor(dev, (B, T, H * hd), dtype=dtype)

    def run(self, layer, stream):
        layer.forward(*self.args, self.out, stream=stream)

    def result(self, layer, stream):
        self.out.copy_from(np.full(self.out.shape, -7, np.float32))
        self.run(layer, stream)
        stream.sync(60000)
        return self.out.to_numpy()


@pytest.mark.parametrize("kind", ["calls", "graphs"])
def test_calls_that_overlapped_spoil_no_later_ones(dev, kind):
    """A layer's workspace serves one call at a time: two that overlap all the same may have wrong results, but once they
    are done the layer's calls, the captured ones as well, have the bits of a layer that is new."""
    say(f"memory overlapped {kind}")
    H, hd, dtype = 2, 64, "bf16"
    streams = [nn.Stream(dev) for _ in "ab"]
    sizes = ((1, 1, 16000), (1, 2, 1400), (1, 300, 4000))  # joins of 64, of a few and of 15 ranges
    calls = [[MemoryCall(dev, *size, H, hd, dtype, i) for i, size in enumerate(sizes)] for _ in streams]
    want = [c.result(nn.MemoryAttention(dev, H, hd), streams[0]) for c in calls[0]]
    layer = nn.MemoryAttention(dev, H, hd)
    for c in calls[0]:
        c.run(layer, streams[0])  # the workspace's size
    streams[0].sync(60000)

    def all_of(i):
        for c in calls[i][i:] + calls[i][:i]:
            c.run(layer, streams[i])

    graphs = [Graph(s, lambda i=i: all_of(i)) for i, s in enumerate(streams)] if kind == "graphs" else []
    for _ in range(50):
        for i in (0, 1):
            graphs[i].replay() if graphs else all_of(i)
    for s in streams:
        s.sync(60000)
    for i, s in enumerate(streams):
        if graphs:
            for c in calls[i]:
                c.out.copy_from(np.full(c.out.shape, -7, np.float32))
            graphs[i].replay()
            s.sync(60000)
            for c, w in zip(calls[i], want):
                np.testing.assert_array_equal(c.out.to_numpy(), w)
        for c, w in zip(calls[i], want):
            np.testing.assert_array_equal(c.result(layer, s), w)


def test_more_captured_calls_than_counts(dev):
    """Each captured call keeps counts of its own while there are any left; those that come later clear the ones that they
    share before they use them."""
    say("memory captured often")
    H, hd, dtype = 2, 64, "f32"
    s = nn.Stream(dev)
    calls = [MemoryCall(dev, 1, T, S, H, hd, dtype, T) for T, S in ((1, 3000), (130, 1100))]
    layer = nn.MemoryAttention(dev, H, hd)
    want = [c.result(layer, s) for c in calls]
    graphs = [Graph(s, lambda: [c.run(layer, s) for c in calls for _ in range(1000)] and None) for _ in range(3)]
    for g in graphs + graphs[::-1]:
        for c in calls:
            c.out.copy_from(np.full(c.out.shape, -7, np.float32))
        g.replay()
        s.sync(60000)
        for c, w in zip(calls, want):
            np.testing.assert_array_equal(c.out.to_numpy(), w)
            np.testing.assert_array_equal(c.result(layer, s), w)


def test_calls_captured_before_any_other(dev):
    """Where the capture's mode lets a call allocate, a layer's first call may be a captured one."""
    say("memory captured first")
    H, hd, dtype = 2, 64, "bf16"
    s = nn.Stream(dev)
    calls = [MemoryCall(dev, 1, T, S, H, hd, dtype, T) for T, S in ((1, 3000), (300, 1100))]
    want = [c.result(nn.MemoryAttention(dev, H, hd), s) for c in calls]
    layer = nn.MemoryAttention(dev, H, hd)
    graph = Graph(s, lambda: [c.run(layer, s) for c in calls] and None)
    for i in range(4):
        for c in calls:
            c.out.copy_from(np.full(c.out.shape, -7, np.float32))
        graph.replay()
        s.sync(60000)
        for c, w in zip(calls, want):
            np.testing.assert_array_equal(c.out.to_numpy(), w)
            if i > 1:
                np.testing.assert_array_equal(c.result(layer, s), w)


def test_first_call_while_another_stream_is_captured(dev):
    say("memory first call beside a capture")
    a, b, graph = nn.Stream(dev), nn.Stream(dev), C.c_void_p()
    call = MemoryCall(dev, 1, 1, 3000, 2, 64, "bf16", 9)
    want = call.result(nn.MemoryAttention(dev, 2, 64), b)
    layer = nn.MemoryAttention(dev, 2, 64)
    handle = C.c_void_p(C.cast(a.handle, C.POINTER(C.c_void_p))[1])
    assert hip().hipStreamBeginCapture(handle, 2) == 0
    try:
        call.run(layer, b)
    finally:
        ended = hip().hipStreamEndCapture(handle, C.byref(graph))
    b.sync(60000)
    assert ended == 0
    np.testing.assert_array_equal(call.out.to_numpy(), want)
    np.testing.assert_array_equal(call.result(layer, a), want)


# ----------------------------------------------------------------- sizes near the ends of what calls take
def rows_of(rng, n, heads, hd):
    return rounded(rng.standard_normal((n, heads * hd)), "bf16")


@pytest.mark.parametrize("B,T,S,H,KV,hd", [(60001, 1, 3, 8, 8, 8), (1, 1, 5, 60003, 60003, 8), (65535, 1, 1, 1, 1, 16),
                                           (1, 300007, 5, 1, 1, 8), (7, 9001, 70, 16, 16, 8), (1, 1, 200003, 1, 1, 8)])
@pytest.mark.parametrize("held", [False, True])
def test_memory_attention_of_many_rows_heads_and_sequences(dev, B, T, S, H, KV, hd, held):
    say(f"memory many {B}x{T} on {S} heads {H}/{KV} hd {hd} held {held}")
    rng = np.random.default_rng(T)
    s = nn.Stream(dev)
    q, k, v = (rows_of(rng, B * n, w, hd).reshape(B, n, w * hd) for n, w in ((T, H), (S, KV), (S, KV)))
    kv, scales = [tensor(dev, x, "bf16") for x in (k, v)], [None, None]
    if held:
        (k8, ks), (v8, vs) = held_rows(k, KV), held_rows(v, KV)
        kv, scales = [tensor(dev, x, "e4m3") for x in (k8, v8)], [tensor(dev, x, "f32") for x in (ks, vs)]
        k, v = values_of(k8, ks), values_of(v8, vs)
    out = nn.Tensor(dev, q.shape, dtype="bf16")
    nn.MemoryAttention(dev, H, hd, KV).forward(tensor(dev, q, "bf16"), *kv, out, None, None, *scales, stream=s)
    s.sync(60000)
    got = out.to_numpy()
    for b in sorted({0, 1, B // 2, B - 2, B - 1} & set(range(B))):
        t = np.unique(np.r_[0:min(T, 40), T // 2:min(T, T // 2 + 40), max(0, T - 40):T])
        h = np.unique(np.r_[0:min(H, 3), H // 2:min(H, H // 2 + 3), H - min(H, 3):H])
        cols = (h[:, None] * hd + np.arange(hd)).ravel()
        want, spread, size = memory(q[b][t][:, cols], k[b][:, cols], v[b][:, cols], len(h), len(h), hd ** -0.5)
        check(got[b][t][:, cols], want, held_tolerance(spread, size, hd, S, "bf16"), f"sequence {b}")


@pytest.mark.parametrize("B,T,KV,hd,left,sinks", [(1, 65535, 1, 8, 10, 2), (30001, 1, 4, 8, 3, 1), (1, 2, 40009, 8, 3, 0)])
def test_window_step_held_of_many_rows_heads_and_streams(dev, B, T, KV, hd, left, sinks):
    say(f"8-bit step many {B}x{T} heads {KV} hd {hd}")
    rng = np.random.default_rng(B)
    s = nn.Stream(dev)
    slots, p0 = sinks + left + T, 7 * left
    q, k, v = (rows_of(rng, B * T, KV, hd).reshape(B, T, KV * hd) for _ in range(3))
    old = [held_rows(rng.standard_normal((B, slots, KV * hd)), KV) for _ in "kv"]
    out = nn.Tensor(dev, q.shape, dtype="bf16")
    c, sc = [tensor(dev, x, "e4m3") for x, _ in old], [tensor(dev, x, "f32") for _, x in old]
    nn.WindowAttention(dev, KV, hd, KV, left, 0, sinks).step(
        *(tensor(dev, x, "bf16") for x in (q, k, v)), tensor(dev, np.full(B, p0), "i32"), *c, out, None, s, *sc)
    s.sync(60000)
    got, cache, scales = out.to_numpy(), [x.to_numpy() for x in c], [x.to_numpy() for x in sc]
    new = [held_rows(x, KV) for x in (k, v)]
    at = [slot_of(p0 + i, sinks, slots) for i in range(T)]
    for i in (0, 1):
        np.testing.assert_array_equal(cache[i][:, at], new[i][0])
        np.testing.assert_array_equal(scales[i][:, at], new[i][1])
    h = np.unique(np.r_[0:min(KV, 3), KV // 2, KV - 1])
    cols = (h[:, None] * hd + np.arange(hd)).ravel()
    for b in sorted({0, B // 2, B - 1}):
        for t in sorted({0, min(1, T - 1), T // 2, T - 1}):
            told = [p for p in range(p0 + t + 1) if p < sinks or p >= p0 + t - left]
            rows = [np.stack([values_of(n[0][b, p - p0], n[1][b, p - p0]) if p >= p0 else
                              values_of(o[0][b, slot_of(p, sinks, slots)], o[1][b, slot_of(p, sinks, slots)])
                              for p in told])[:, cols] for n, o in zip(new, old)]
            want, spread, size = memory(q[b, t:t + 1][:, cols], *rows, len(h), len(h), hd ** -0.5)
            check(got[b, t:t + 1][:, cols], want, held_tolerance(spread, size, hd, len(told), "bf16"), f"{b} {t}")


@pytest.mark.parametrize("M,K,N", [(300007, 100, 8), (2, 16, (1 << 20) + 200), (70001, 130, 33), (1, 100003, 5)])
def test_linear_blocks_of_many_rows_and_outputs(dev, M, K, N):
    say(f"linear blocks many {M}x{K}x{N}")
    rng = np.random.default_rng(N)
    s = nn.Stream(dev)
    x = rng.standard_normal((M, K)).astype(np.float32)
    w = (rng.standard_normal((N, K)) / np.sqrt(K)).astype(np.float32)
    layer = nn.Linear(dev, K, N, use_bias=False, precision="e4m3_block")
    layer.load_weights(w)
    y = nn.Tensor(dev, (M, N))
    layer.forward_scaled(tensor(dev, x, "f32"), None, y, stream=s)
    s.sync(60000)
    rows = np.unique(np.r_[0:min(M, 70), M // 2:min(M, M // 2 + 70), max(0, M - 70):M])
    want, mass = linear_blocks(*quantise_blocks(x[rows]), *quantise_tiles(w), None)
    check(y.to_numpy()[rows], want, (1.5 * K + 4 * blocks_of(K) + 8) * EPS * mass + 1e-37, "rows")
