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


def test_weights_that_overlap():
    """Rows of weights that share places (an expanded view's) would be added to by several workgroups."""
    d = _lib.Kv4Desc(16, 16, 16, 16, 8, 3, 32, 64)

    def call(w_seq, w_head, B=2, max_len=40, width=2):  # refused for its workspace where nothing else is wrong
        rc = _lib.lib().bq_kv4_attend(ctypes.byref(d), 16, 0, 1, 3, 256, 256, 64, 16, B, width, 16, max_len, 0.1, 16, 16,
                                      w_seq, w_head, None, 0, None)
        assert rc == ARG
        return "overlap" in _lib.last_error()

    assert not call(120, 40) and not call(40, 80) and not call(1000, 64) and not call(-120, 40)
    assert call(0, 40) and call(120, 0) and call(120, 39) and call(119, 40) and call(40, 79) and call(0, 0)
    assert not call(0, 40, B=1)
    assert not call(32, 64, width=1) and call(31, 64, width=1)  # 32 tokens are what a page has room for


def test_products_of_sizes_that_wrap():
    """Sequences, heads and blocks whose product passes 64 bits are too large, not a small grid."""
    lib = _lib.lib()
    d = _lib.Kv4Desc(16, 16, 16, 16, 8, 65535, 32, 64)
    most = 2 ** 31 - 8193
    for B in (2 ** 22, 2 ** 23 - 1):
        assert (B * 65535 * -(-most // 32) + 2 ** 63) % 2 ** 64 - 2 ** 63 < 2 ** 31  # as 64 bits have it
        assert lib.bq_kv4_read(ctypes.byref(d), 16, B, 1, 16, most, 16, 16, None) == ARG and "large" in _lib.last_error()
        keep = most // 2 // 32 * 32
        rc = lib.bq_kv4_evict(ctypes.byref(d), 16, 8, 8, 8, 16, B, 1, 16, 16, keep // 32 + 1, keep, 0, 16, 16, 16, None, 0, None)
        assert rc == ARG and "large" in _lib.last_error()
