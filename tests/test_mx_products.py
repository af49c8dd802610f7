"""The microscaled products' entry points without a GPU: which sums a caller may ask
for."""

from __future__ import annotations

import pytest

P = 1 << 20  # a 16-byte aligned address
SHORT = 16   # NVM_MX_SHORT_SUMS


def _lib():
    from nano_vllm_metal_amd import _lib

    return _lib.load()


def _matmul(fmt, K=0):
    return _lib().nvm_mx_matmul(P, P, 16, fmt, P, P, 16, 4, 64, K, 1, P, None)


def _swiglu(fmt, M=0):
    return _lib().nvm_mx_swiglu(P, P, 16, fmt, P, P, 16, P, P, 16, M, 64, 32, 1, P, P, 16, None)


@pytest.mark.parametrize("call", [_matmul, _swiglu])
def test_short_sums_are_a_flag_of_the_products(call):
    for fmt in (0, 1, SHORT, SHORT | 1):  # (nothing to compute: a no-op)
        assert call(fmt) == 0
    for fmt in (2, SHORT | 2, 2 * SHORT, 3 * SHORT | 1, -1, -SHORT):
        assert call(fmt) == -1 and b"a format" in _lib().nvm_last_error()


def test_other_entries_do_not_take_the_flag():
    lib = _lib()
    assert lib.nvm_mx_quantize(P, 0, 64, 64, 1, SHORT | 1, P, P, 16, None) == -1
    assert lib.nvm_mx_dequantize(P, P, 16, 0, 64, SHORT, 1, P, None) == -1
    assert lib.nvm_mx_embedding(P, 0, P, P, 16, 9, 64, SHORT | 1, 1, P, None) == -1
    assert lib.nvm_mx_swiglu(P, P, 16, 1, P, P, 16, P, P, 16, 0, 64, 32, SHORT | 1, P, P, 16,
                             None) == -1
