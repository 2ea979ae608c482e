"""What the decoder's layers hold of the device, and keep from call to call."""
import ctypes as C

import pytest

from metalaudio_amd import nn
from metalaudio_amd._lib import check as ok
from metalaudio_amd._lib import lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return nn.AudioDevice(0)


@pytest.fixture(scope="module")
def stream(dev):
    return nn.Stream(dev)


def say(msg):
    print(f"[case] {msg}", flush=True)


# --------------------------------------------------------------- what layers keep
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
