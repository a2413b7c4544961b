"""Scales whose product with log2 e is no float are refused by both attention entry points, before any HIP call."""
import ctypes

import pytest

from crispybits_kernels import _C

P, I, L, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
lib = ctypes.CDLL(_C.LIB_PATH)
lib.cbk_kv4_attention.argtypes = [P, I, L, L, L, P, L, L, I, L, P, L, P, F, P, L, P, I, P]
lib.cbk_prompt_attention.argtypes = [P, P, P, I, L, L, L, I, L, L, L, L, L, L, P, L, L, F, I, P, I, P]
lib.cbk_last_error.restype = ctypes.c_char_p
A = 1 << 20          # a fake, 16-byte aligned "device" address: never dereferenced


@pytest.mark.parametrize("scale", [3e38, 2.0 ** 127 * 1.0001, float("inf"), float("nan"), 0.0, -1.0])
def test_scales(scale):
    assert lib.cbk_kv4_attention(A, 0, 2, 1, 4, A, 4, 2, 128, 64, A, 2, A, scale, A, 1 << 40, A, 0, None) == 1
    assert b"kv4_attention: scale must be" in lib.cbk_last_error()
    assert lib.cbk_prompt_attention(A, A, A, 0, 100, 4, 2, 128, 512, 128, 256, 128, 256, 128, A, 2, 80, scale, 1, A, 0, None) == 1
    assert b"prompt_attention: scale must be" in lib.cbk_last_error()
