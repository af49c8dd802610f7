"""The microscaled products' entry points without a GPU: which sums a caller may ask
for, and which kernel runs for which sizes (as on 256 CUs)."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch

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


def _plan(gate_up, M, N, K, fmt):
    plan = (ctypes.c_int * 4)()
    rc = _lib().nvm_mx_product_plan(gate_up, M, N, K, fmt, plan)
    return tuple(plan) if rc == 0 else rc


def _ceil(a, b):
    return -(-a // b)


def _fits(gate_up, M, K, plan):
    """What a launch takes: 2^32 - 1 threads in x and 65535 blocks in y of the few-row
    kernel, 2^22 tiles of the others."""
    kernel, columns, rows, parts = plan
    x, y = _ceil(K * (2 if gate_up else 1), columns), _ceil(M, rows)
    if kernel == 0:
        return 256 * x < 2 ** 32 and y <= 65535
    return x * y <= 2 ** 22 and (kernel == 2 or parts == 0)


@pytest.mark.parametrize("fmt", [0, 1, SHORT | 1])
def test_many_rows_of_few_columns_get_a_kernel_that_can_be_launched(fmt):
    for gate_up, M, N, K in [(1, 4_200_000, 512, 32), (1, 4_200_000, 32, 32), (1, 2 ** 31 - 1, 64, 32),
                             (0, 4_200_000, 512, 32), (0, 2 ** 31 - 1, 32, 1), (0, 2 ** 29, 32, 64),
                             (0, 1_048_577, 32, 16), (0, 32, 32, 2 ** 30 - 1), (0, 1, 64, 2 ** 30)]:
        plan = _plan(gate_up, M, N, K, fmt)
        if isinstance(plan, tuple):
            assert _fits(gate_up, M, K, plan), (gate_up, M, N, K, plan)
        else:  # refused: the largest tile has too many
            assert plan == -2 and _ceil(M, 256) * _ceil(K * (1 + gate_up), 256) > 2 ** 22


@pytest.mark.parametrize("fmt", [0, 1, SHORT | 1])
def test_every_choice_can_be_launched(fmt):
    rng = random.Random(fmt)
    for _ in range(4000):
        gate_up, M = rng.randint(0, 1), int(2 ** rng.uniform(0, 31)) - 1
        N, K = 32 * int(2 ** rng.uniform(0, 15)), int(2 ** rng.uniform(0, 20))
        K = K if not gate_up else 32 * _ceil(K, 32)
        plan = _plan(gate_up, M, N, K, fmt)
        if M == 0:
            assert plan[0] == -1
        elif isinstance(plan, tuple):
            assert _fits(gate_up, M, K, plan), (gate_up, M, N, K, plan)
            assert plan[0] == 0 or M > 32
        else:
            assert plan == -2 and _ceil(M, 256) * _ceil(K * (1 + gate_up), 256) > 2 ** 22


def test_the_plan_refuses_what_the_products_refuse():
    lib, plan = _lib(), (ctypes.c_int * 4)()
    for args, rc, msg in [((0, 4, 64, 8, 1, None), -1, b"null"), ((0, 4, 48, 8, 1, plan), -1, b"of a"),
                          ((0, -1, 64, 8, 1, plan), -1, b"of a"), ((0, 4, 64, -8, 1, plan), -1, b"of w"),
                          ((0, 4, 64, 8, 2, plan), -1, b"a format"), ((1, 4, 64, 8, 1, plan), -1, b"output"),
                          ((0, 2 ** 31, 64, 8, 1, plan), -2, b"large")]:
        assert lib.nvm_mx_product_plan(*args) == rc and msg in lib.nvm_last_error()


def test_listed_sizes_reach_their_kernels():
    """(tests/mx_sizes.py, which the GPU tests go through: a new fit that sends them
    elsewhere shows here)"""
    from mx_sizes import REACH

    for gate_up, plan, fmt, sizes in REACH:
        for M, N, K in sizes:
            assert _plan(gate_up, M, N, K, fmt) == plan, (gate_up, M, N, K, fmt)
    assert len({(g, p, f) for g, p, f, _ in REACH}) == len(REACH) == REACHED


# every tile of every kernel for each of E2M1, E4M3 and E4M3 in short sums: seven
# blocks (E4M3 six) and four for gate/up, four tiles and three, 256 x 256 in whole
# tiles, halves and quarters
REACHED = 3 * (7 + 4 + 4 + 3 + 3 + 3) - 1


@pytest.mark.parametrize("fmt", [0, 1, SHORT | 1])
def test_no_other_kernel_is_chosen(fmt):
    from mx_sizes import REACH

    known = {(g, p, f) for g, p, f, _ in REACH}
    rng = random.Random(fmt + 1)
    for _ in range(20000):
        gate_up, M = rng.randint(0, 1), int(2 ** rng.uniform(0, 14))
        N, K = 32 * int(2 ** rng.uniform(0, 9)), 32 * int(2 ** rng.uniform(0, 10))
        assert (gate_up, _plan(gate_up, M, N, K, fmt), fmt) in known, (gate_up, M, N, K)


@pytest.mark.parametrize("shape,dtype", [((31,), torch.bfloat16), ((1, 32), torch.bfloat16),
                                         ((3, 32), torch.float32), ((3, 1), torch.float32),
                                         ((), torch.float32), ((1,), torch.float16),
                                         ((32,), torch.int32), ((32,), torch.float64)])
def test_linear_refuses_what_is_no_bias(shape, dtype):
    from nano_vllm_metal_amd import MxTensor, mx_linear

    def mx(rows, fmt):
        codes = torch.zeros(rows, 64 if fmt == "mxfp8" else 32, dtype=torch.uint8)
        return MxTensor(codes, torch.full((rows, 2), 127, dtype=torch.uint8), fmt)

    with pytest.raises(ValueError, match="bias must be"):
        mx_linear(mx(3, "mxfp8"), mx(32, "mxfp4"), bias=torch.zeros(shape, dtype=dtype))
    with pytest.raises(ValueError, match="GPU only"):  # (a good one: the next check)
        mx_linear(mx(3, "mxfp8"), mx(32, "mxfp4"), bias=torch.zeros(32))


def test_dequantize_refuses_what_is_no_mx_tensor():
    from nano_vllm_metal_amd import mx_dequantize

    for t in (torch.zeros(3, 64, dtype=torch.uint8), None):
        with pytest.raises(ValueError, match="must be an MxTensor"):
            mx_dequantize(t)
