"""Lengths of the attention's argument block whose products leave 64 bits are refused, not taken for small ones.  No GPU needed."""

import ctypes

import pytest

from nunchaku_amd import _native as nv


@pytest.fixture(scope="module")
def lib():
    if not nv.LIB_PATH.exists():
        nv.build()
    return nv.lib()


def test_lengths_whose_products_leave_64_bits(lib):
    i3 = ctypes.c_int64 * 3
    need = ctypes.c_int64()
    for q_len, heads in ((2**62 + 1, 4), (2**60 + 1, 16), (2**63 - 1, 2), (2**59 + 3, 32), (2**48, 65535), (2**31, 1), (2**62, 4)):
        args = nv.CrossAttentionArgs(q=16, k=16, v=16, out=16, batch=2, heads=heads, kv_heads=1, head_dim=64, q_len=q_len, k_len=5, q_stride=i3(768, 256, 64),
                                     k_stride=i3(640, 128, 64), v_stride=i3(640, 128, 64), out_stride=i3(768, 256, 64), scale=0.125)
        assert lib.svdq_cross_attention(ctypes.byref(args), None) == -1, (q_len, heads)
        assert b"q_len" in lib.svdq_last_error()
        assert lib.svdq_cross_attention_workspace(ctypes.byref(args), ctypes.byref(need)) == -1, (q_len, heads)
        assert b"q_len" in lib.svdq_last_error()
