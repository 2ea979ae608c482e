"""The bits that the decoder's operators hold, through the C ABI against 64-bit references.
Tolerances count roundings (token_refs.py, decoder_refs.py) and were fixed before the first run."""
import numpy as np
import pytest

from metalaudio_amd import nn
from tests import token_bits as bits
from tests.decoder_refs import held_rows, held_tolerance, memory, values_of
from tests.test_gpu_tokens import check, tensor
from tests.token_refs import HALF, attend, rounded, slot_of

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
