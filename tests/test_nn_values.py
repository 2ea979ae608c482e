"""Host values of the tensors of positions and of 8 bits (no GPU)."""
import numpy as np
import pytest
import torch

from metalaudio_amd import nn


@pytest.mark.parametrize("x", [[0, -5, 2 ** 31 - 1, -2 ** 31], np.arange(6).reshape(2, 3), np.array([3.0, -2.0]),
                               np.array([], np.int64), 7])
def test_positions_are_kept(x):
    got = nn.i32_values(x)
    assert got.dtype == np.int32 and got.flags.c_contiguous and np.array_equal(got, np.asarray(x))


@pytest.mark.parametrize("x", [[2 ** 31], np.array([1, -2 ** 31 - 1]), np.array([2 ** 32 + 4]), [0.5], [np.nan], [np.inf],
                               np.array([2 ** 63], np.uint64)])
def test_positions_that_do_not_fit_are_refused(x):
    """They would come out as other positions, and a stream at one of them be left alone without a word."""
    with pytest.raises(ValueError):
        nn.i32_values(x)


def test_e4m3_patterns():
    bits = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(bits).view(torch.float8_e4m3fn).float().numpy()
    np.testing.assert_array_equal(nn.E4M3_VALUES, want)
    fine = ~np.isnan(want)
    np.testing.assert_array_equal(nn.e4m3_bits(want)[fine], bits[fine])
    x = np.concatenate([np.random.default_rng(0).standard_normal(4000) * s for s in (1e-3, 1, 100)]).astype(np.float32)
    half = (want[fine][:-1] + want[fine][1:]) / 2  # ties go to even
    x = np.concatenate([x[np.abs(x) < 448], half, [448, 464, -464, 0.0, -0.0]]).astype(np.float32)
    np.testing.assert_array_equal(nn.e4m3_bits(x), torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert (nn.e4m3_bits([465, np.inf, -np.inf, np.nan]) & 0x7F == 0x7F).all()
