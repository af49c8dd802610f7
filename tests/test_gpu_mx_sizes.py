"""Which kernel the microscaled products (include/nvm_mx.h) run for which sizes, and
that it is right there.  Oracle: float64 products of the decoded operands; bounds as
in test_gpu_mx_sums.py (float32 sums: N * 2^-23 * sum |a w|; short ones 7 * 2^-13 of
each eight's largest product more)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from mx_sizes import REACH
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


# ------------------------------------------------- every tile, every length of a row


def _hostile(t):
    """The tensor with NaN codes in the rows behind it, and NaN scales there and in
    the padding of its rows."""
    from nano_vllm_metal_amd import MxTensor

    rows, blocks = t.scales.shape
    codes = torch.full((rows + 3, t.codes.shape[1]), 0xFF, dtype=torch.uint8, device=DEV)
    scales = torch.full((rows + 3, t.pitch + 16), 255, dtype=torch.uint8, device=DEV)
    codes[:rows], scales[:rows, :blocks] = t.codes, t.scales
    return MxTensor(codes[:rows], scales[:rows, :blocks], t.fmt)


def _id(case):
    gate_up, plan, fmt, _ = case
    return f"{'gate_up' if gate_up else 'linear'}-{plan[0]}-{plan[1]}x{plan[2]}-{plan[3]}-{fmt}"


@pytest.mark.parametrize("case", [c for c in REACH if not c[0]], ids=_id)
def test_linear_on_every_tile(case):
    from nano_vllm_metal_amd import _lib

    _, plan, code, sizes = case
    fmt, short = FMTS[code & 1], code > SHORT
    for M, N, K in sizes:
        print("size", M, N, K, flush=True)
        assert _plan(0, M, N, K, fmt, short) == plan
        g = _gen(M + N + K)
        a, w = _random(g, M, N, fmt), _random(g, K, N, "mxfp4")
        want, bound = _sums(_val(a), _val(w), short)
        ah, wh = _hostile(a), _hostile(w)
        for dtype, dt in ((2, torch.float32), (M % 2, (torch.float16, torch.bfloat16)[M % 2])):
            out = torch.full((M + 2, K), 7.0, dtype=dt, device=DEV)
            _lib.check(_lib.load().nvm_mx_matmul(
                ah.codes.data_ptr(), ah.scales.data_ptr(), ah.pitch, code, wh.codes.data_ptr(),
                wh.scales.data_ptr(), wh.pitch, M, N, K, dtype, out.data_ptr(),
                _lib.stream_of(out.device)))
            tol = bound + torch.finfo(dt).eps / 2 * (want.abs() + bound) + torch.finfo(dt).tiny
            if dt == torch.float16:
                big = want.abs() + bound > 65504
                tol = torch.where(big, torch.full_like(tol, float("inf")), tol)
            off = (out[:M].double() - want).abs()
            assert (torch.nan_to_num(off, nan=float("inf"), posinf=1e300) <= tol).all()
            assert (out[M:] == 7).all()


@pytest.mark.parametrize("case", [c for c in REACH if c[0]], ids=_id)
def test_gate_and_up_on_every_tile(case):
    from nano_vllm_metal_amd import mx_swiglu

    _, plan, code, sizes = case
    fmt, short = FMTS[code & 1], code > SHORT
    for M, N, K in sizes:
        print("size", M, N, K, flush=True)
        assert _plan(1, M, N, K, fmt, short) == plan
        g = _gen(M + N + K)
        a = _random(g, M, N, fmt, 117, 121)
        wg, wu = _random(g, K, N, "mxfp4", 117, 121), _random(g, K, N, "mxfp4", 117, 121)
        ofmt = FMTS[N // 32 % 2]
        y = mx_swiglu(_hostile(a), _hostile(wg), _hostile(wu), ofmt, short)
        (gate, eg), (up, eu) = _sums(_val(a), _val(wg), short), _sums(_val(a), _val(wu), short)
        O.check_quantized(y.codes, y.scales, ofmt, *_silu_bound(gate, eg, up, eu))


@pytest.mark.parametrize("M", [3, 70, 300])
@pytest.mark.parametrize("fmt", FMTS)
def test_blocks_of_different_scales_add_up(M, fmt):
    """Bit for bit: a row has one value in each of four neighbouring blocks, whose
    scales are 2^0, 2^5, 2^10 and 2^15.  E2M1 by E2M1, and E4M3 elements of 1 to 7 in
    halves, are multiples of 1/4 up to 42: with the scales below 2^21 together."""
    from nano_vllm_metal_amd import MxTensor, mx_linear

    N, K = 672, 200
    g = _gen(M)
    w = _random(g, K, N, "mxfp4", 127, 128)
    m = torch.arange(M, device=DEV)
    grid = O.elements(fmt, DEV)
    ok = ((grid * 2 == (grid * 2).round()) & (grid <= 7)).nonzero()[:, 0]
    codes = torch.zeros(M, N, dtype=torch.int64, device=DEV)
    scales = torch.full((M, N // 32), 127, dtype=torch.uint8, device=DEV)
    for j in range(4):
        block = (4 * (m % 5) + j) % (N // 32)
        at = 32 * block + torch.randint(0, 32, (M,), device=DEV, generator=g)
        sign = torch.randint(0, 2, (M,), device=DEV, generator=g) * O.SIGN[fmt]
        codes[m, at] = ok[torch.randint(0, len(ok), (M,), device=DEV, generator=g)] + sign
        scales[m, block] = 127 + 5 * ((j + m) % 4).to(torch.uint8)
    a = MxTensor(O.pack(codes, fmt), scales, fmt)
    assert torch.equal(mx_linear(a, w, torch.float32).double(), _val(a) @ _val(w).t())
