"""What the decoder's layers hold of the device, and keep from call to call."""
import ctypes as C

import numpy as np
import pytest

from metalaudio_amd import nn
from metalaudio_amd._lib import check as ok
from metalaudio_amd._lib import lib
from tests.test_gpu_tokens import Graph, tensor

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
