"""Sizes that the 4-bit operators count in 32 bits are refused on the host, before any launch (no pointer is read)."""

import ctypes

import pytest

from mini_infra_b200 import _native as nat


@pytest.mark.parametrize("dtype,head_dim", [(nat.MI_BF16, 128), (nat.MI_F16, 64), (nat.MI_F32, 32)])
def test_decode_refuses_tables_of_more_tokens_than_32_bits_hold(dtype, head_dim):
    lib = nat.load()
    strides, there = nat.i64_array([0, 0, 0]), ctypes.c_void_p(256)

    def decode(width, batch=2, bs=16):
        return lib.mi_kv4_paged_decode(there, strides, None, None, None, None, there, there, 8, bs, 8, head_dim, there, width,
                                       width, there, batch, 16, ctypes.c_float(1.0), there, 0, there, 1 << 60, dtype, None)

    for width in (1 << 27, 1 << 28, 1 << 40, (1 << 63) - 1):
        assert decode(width) == nat.MI_ERR_UNSUPPORTED and "tokens a row" in nat.last_error()
        assert decode(width, batch=1) == nat.MI_ERR_UNSUPPORTED
        assert lib.mi_kv4_paged_decode_workspace_size(2, 16, 8, head_dim, width, 16, dtype) == 0
    assert decode(1 << 26, bs=32) == nat.MI_ERR_UNSUPPORTED
