"""CPU checks of the decoder's entry points: null handles and descriptors are refused with a message, and
the references of their GPU tests hold their own definitions."""
import ctypes as C

import numpy as np
import pytest

from metalaudio_amd import _lib
from tests.decoder_refs import (blocks_of, held_rows, linear_blocks, memory, quantise_blocks, quantise_tiles,
                                spread_scales, values_of)


@pytest.mark.parametrize("name", ["mnn_window_attention_step_e4m3", "mnn_kv_cache_write", "mnn_kv_cache_read",
                                  "mnn_memory_attention_forward", "mnn_linear_forward_scaled"])
def test_null_handles_are_refused(name):
    lib = _lib.lib()
    args = [None] * len(_lib.SIGNATURES[name][1])
    assert getattr(lib, name)(*args) == 12 and b"null" in lib.mnn_last_error_message()


def test_null_devices_are_refused():
    lib = _lib.lib()
    out = C.c_void_p()
    assert lib.mnn_kv_cache_create(None, 2, 16, 0, C.byref(out)) == 12
    assert lib.mnn_memory_attention_create(None, None, C.byref(out)) == 12
    assert lib.mnn_linear_create(None, 8, 8, 1, 0, 3, C.byref(out)) == 12
    assert not out.value


@pytest.mark.parametrize("m,k", [(3, 1), (2, 128), (4, 129), (1, 500)])
def test_blocks_hold_their_values(m, k):
    x = np.random.default_rng(k).standard_normal((m, k)).astype(np.float32)
    x[:, ::7] *= 1000
    q, s = quantise_blocks(x)
    assert s.shape == (m, blocks_of(k)) and np.abs(q).max() <= 448
    each = spread_scales(s, x.shape)
    step = np.maximum(np.abs(x) * 2.0 ** -4, each * 2.0 ** -10)
    assert (np.abs(q * each - x) <= step * (1 + 1e-5)).all()


def test_tiles_and_products():
    rng = np.random.default_rng(1)
    w = rng.standard_normal((200, 300)).astype(np.float32)
    q, s = quantise_tiles(w)
    assert s.shape == (2, 3)
    each = spread_scales(s, w.shape, 128)
    assert each.shape == w.shape and each[130, 260] == np.float64(s[1, 2])
    assert (np.abs(q * each - w) <= np.maximum(np.abs(w) * 2.0 ** -4, each * 2.0 ** -10) * (1 + 1e-5)).all()
    x = rng.standard_normal((5, 300)).astype(np.float32)
    xq, xs = quantise_blocks(x)
    y, mass = linear_blocks(xq, xs, q, s, None)
    slow = sum(np.outer(xs[:, j].astype(np.float64), s[np.arange(200) // 128, j])
               * (xq[:, 128 * j:128 * (j + 1)].astype(np.float64) @ q[:, 128 * j:128 * (j + 1)].T) for j in range(3))
    np.testing.assert_allclose(y, slow, rtol=0, atol=1e-12 * mass.max())


def test_held_rows_and_attention():
    rng = np.random.default_rng(2)
    x = rng.standard_normal((7, 6 * 16)).astype(np.float32)
    q, s = held_rows(x, 6)
    assert s.shape == (7, 6)
    np.testing.assert_allclose(values_of(q, s), x, atol=np.abs(x).max() * 2.0 ** -4)
    out, _, _ = memory(x[:, :64], x[:5, :32], x[:5, 32:64], 4, 2, 0.25)
    p = np.exp(x[2, 16:32].astype(np.float64) @ x[:5, :16].astype(np.float64).T * 0.25)
    np.testing.assert_allclose(out[2, 16:32], p / p.sum() @ x[:5, 32:48], rtol=1e-12)
    assert (memory(x[:, :64], x[:0, :32], x[:0, :32], 4, 2, 0.25)[0] == 0).all()
