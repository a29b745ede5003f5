"""Host parts of the 4-bit linears and of the block-sparse attention."""
import numpy as np
import pytest

import esm_gfx950 as eg
from conftest import rng
from esm_gfx950 import synthetic as syn


@pytest.mark.parametrize("lengths,block,want", [
    ([1], 16, [0, 1]),
    ([0], 64, [0, 0]),
    ([64, 0, 65, 1], 64, [0, 1, 1, 3, 4]),
    ([16, 17, 1023, 1024, 1025], 16, [0, 1, 3, 67, 131, 196]),
    ([2 ** 31 - 1], 1024, [0, 2 ** 21]),
])
def test_key_blocks(lengths, block, want):
    cu = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    np.testing.assert_array_equal(eg.key_blocks(cu, block), want)


@pytest.mark.parametrize("cu,block", [
    ([1, 5], 64), ([0, 5, 4], 64), ([0], 64), ([0, 5], 0), ([0, 5], 8), ([0, 5], 24), ([0, 5], 1040), ([0, 5], -16),
])
def test_key_blocks_refuses(cu, block):
    with pytest.raises(eg.Gfx950Error):
        eg.key_blocks(np.array(cu, np.int32), block)


@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (3, 33, 32), (16, 128, 64), (17, 131, 64), (5, 300, 128), (4, 77, 256)])
def test_quantize_weight_i4(n, k, group):
    """A weight is off by at most half a step of its group, the fp32 quotient's
    rounding (2^-24 of a quotient of at most 7, and of the scale) aside."""
    w = rng(n * 1000 + k).standard_normal((n, k)).astype(np.float32)
    w[0, :min(k, group)] = 0  # a group of zeros
    packed, scales = syn.quantize_weight_i4(w, group)
    assert packed.shape == (n, (k + 1) // 2) and packed.dtype == np.uint8
    assert scales.shape == (n, -(-k // group)) and scales.dtype == np.float32
    codes = np.stack([packed & 15, packed >> 4], axis=2).reshape(n, -1).astype(np.int64) - 8
    if k % 2:
        assert (codes[:, k] == 0).all()
    codes = codes[:, :k]
    step = np.repeat(scales.astype(np.float64), group, axis=1)[:, :k]
    assert (codes[0, :min(k, group)] == 0).all() and (scales[0, 0] == 0)
    assert (np.abs(codes * step - w) <= step * (0.5 + 7 * 2.0 ** -22)).all()
    big = np.abs(codes) == 7
    for g in range(scales.shape[1]):
        cols = slice(g * group, min((g + 1) * group, k))
        assert (big[:, cols].any(axis=1) | (scales[:, g] == 0)).all()
