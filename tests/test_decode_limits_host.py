"""Limits of the decoder's attention that the library's C entries hold to, on the CPU: nothing is launched."""
import ctypes

from borch_amd import _lib

ARG, UNSUPPORTED = _lib.BQ_ERR_ARG, _lib.BQ_ERR_UNSUPPORTED


def test_rows_far_apart_are_the_16_bit_types_limit():
    far = (256, 64, 2 ** 23 + 8, 64, 2 ** 24, 64)

    def call(type, strides):  # refused for its workspace where nothing else is wrong
        return _lib.lib().bq_prompt_attention(16, 16, 16, type, 4000, 4, 2, 64, *strides, 16, 1, 1, 0.1, 16, None, 0, None)

    assert call(1, far) == UNSUPPORTED and call(2, far) == UNSUPPORTED
    assert call(0, far) == ARG and "workspace" in _lib.last_error()
    assert call(0, (256, 64, -64, 64, 128, 64)) == UNSUPPORTED
