"""Which kernel the microscaled products (include/nvm_mx.h) run for which sizes, and
that it is right there.  Oracle: float64 products of the decoded operands; bounds as
in test_gpu_mx_sums.py (float32 sums: N * 2^-23 * sum |a w|; short ones 7 * 2^-13 of
each eight's largest product more)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FMTS = ["mxfp4", "mxfp8"]
SHORT = 16  # NVM_MX_SHORT_SUMS


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _val(t):
    return O.decode(t.codes, t.scales, t.fmt)


def _random(g, rows, n, fmt, low=120, high=124):
    """Any finite codes under scales of a few sizes."""
    from nano_vllm_metal_amd import MxTensor

    c = torch.randint(0, 256, (rows, n // 2 if fmt == "mxfp4" else n), dtype=torch.uint8,
                      device=DEV, generator=g)
    if fmt == "mxfp8":
        c = torch.where((c & 127) == 127, c - 1, c)
    s = torch.randint(low, high, (rows, n // 32), dtype=torch.uint8, device=DEV, generator=g)
    return MxTensor(c, s, fmt)


def _plan(gate_up, M, N, K, fmt, short=False):
    from nano_vllm_metal_amd import _lib

    plan = (ctypes.c_int * 4)()
    code = FMTS.index(fmt) | (SHORT if short else 0)
    _lib.check(_lib.load().nvm_mx_product_plan(gate_up, M, N, K, code, plan))
    return tuple(plan)


def _sums(a, w, short):
    """The products of decoded operands and how far the sums may be off."""
    bound = a.shape[1] * 2.0 ** -23 * (a.abs() @ w.abs().t())
    if short:
        rows = max(1, 2 ** 27 // w.numel())
        for i in range(0, a.shape[0], rows):
            p = (a[i:i + rows, None, :] * w[None]).abs()
            bound[i:i + rows] += 7 * 2.0 ** -13 * p.unflatten(-1, (-1, 8)).amax(-1).sum(-1)
    return a @ w.t(), bound


def _silu_bound(g, eg, u, eu):
    s = g * torch.sigmoid(g)
    return s * u, 1.1 * eg * (u.abs() + eu) + s.abs() * eu + 2.0 ** -20 * (s * u).abs() + 2.0 ** -146


# ------------------------------------------------------ many rows, few columns


@pytest.mark.parametrize("fmt", FMTS)
def test_gate_and_up_of_four_million_rows_of_few_columns(fmt):
    """More rows than the few-row kernel's grid has: another one runs."""
    from nano_vllm_metal_amd import MxTensor, mx_swiglu

    M, N, K = 4_200_000, 512, 32
    g = _gen(1)
    a = MxTensor(*(torch.cat([x] * 42) for x in _two(_random(g, M // 42, N, fmt))), fmt)
    wg, wu = _random(g, K, N, "mxfp4", 116, 118), _random(g, K, N, "mxfp4", 116, 118)
    assert a.rows == M and _plan(1, M, N, K, fmt)[0] > 0
    y = mx_swiglu(a, wg, wu)
    i = torch.tensor([0, 1, 65535 * 64 - 1, 65535 * 64, M - 1], device=DEV)
    va = O.decode(a.codes[i], a.scales[i], fmt)
    (gate, eg), (up, eu) = _sums(va, _val(wg), False), _sums(va, _val(wu), False)
    O.check_quantized(y.codes[i], y.scales[i], "mxfp8", *_silu_bound(gate, eg, up, eu))
    # (the operand repeats itself, and so does the output)
    assert torch.equal(y.codes[-(M // 42):], y.codes[:M // 42])


def _two(t):
    return t.codes, t.scales


@pytest.mark.parametrize("fmt", FMTS)
def test_product_of_four_million_rows_of_few_columns(fmt):
    from nano_vllm_metal_amd import MxTensor, mx_linear

    M, N, K = 4_200_000, 64, 24
    g = _gen(2)
    a = MxTensor(*(torch.cat([x] * 42) for x in _two(_random(g, M // 42, N, fmt))), fmt)
    w = _random(g, K, N, "mxfp4")
    y = mx_linear(a, w, torch.float32)
    part = M // 42
    va = O.decode(a.codes[:part], a.scales[:part], fmt)
    want, bound = _sums(va, _val(w), False)
    assert ((y[:part].double() - want).abs() <= bound).all()
    assert torch.equal(y.view(42, part, K), y[:part].expand(42, part, K))
