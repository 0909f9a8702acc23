"""Matrices of more blocks than a launch has workgroups are refused before a launch."""

import pytest

from mojodgl import _lib

F32, BF16 = 0, 2
EINVAL = -1
P = 4096  # an aligned address that no refused call reads


@pytest.mark.parametrize("b1,b2", [(4095, 4097), (4096, 4096), (16777213, 1), (1, 16777209)])
@pytest.mark.parametrize("turned", [0, 1])
def test_too_many_blocks(b1, b2, turned):
    """A launch has (2^32 - 1) / 256 workgroups of 256 work-items, a multiple of 8 of them:
    16,777,208, seven fewer than 2^24 - 1."""
    assert b1 * b2 > ((2 ** 32 - 1) // 256) // 8 * 8
    call = _lib.lib().mdgl_quantize_blocks
    for d1, d2 in ((b1 * 128, b2 * 128), (b1 * 128 - 127, b2 * 128 - 127)):
        assert call(P, P, P, 1, d1, d2, turned, BF16, None) == EINVAL
        assert b"blocks a matrix" in _lib.lib().mdgl_last_error()
    assert call(P, P, P, 0, 4095 * 128, 4097 * 128, turned, F32, None) == EINVAL
