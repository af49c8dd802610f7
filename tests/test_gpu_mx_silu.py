"""The function between the gate/up products and the quantisation of nvm_mx_swiglu
(include/nvm_mx.h), on gates and ups that are exact: a row of the activations has one
value for the gate and one for the up projection, a row of each weight one for it, so
both sums are single products.

Bound, for exp(-g) as 2^t (1 + d ln 2): 2^t 2^-23 (a unit in the last place), the
factor and the product 2^-24 each, so 2^-22 of exp(-g) and no more of 1 + exp(-g);
that sum 2^-24, its inverse 2^-23, and two products 2^-24 each: 2.25 * 2^-22 in all.
Where exp(-g) is beyond float32's range, g below -88.7, the result is zero, and a
result below float32's normal range is off by 2^-149 and the factor u more."""

from __future__ import annotations

import pytest
import torch

from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
REL = 2.25 * 2.0 ** -22


def _operands(a_codes, a_scale, gate_scale, up_scale):
    """Activations with the codes' two columns at k = 0 and 1, and weights of all
    pairs of E2M1 values, the gate's at 0 and the up projection's at 1."""
    from nano_vllm_metal_amd import MxTensor

    def tensor(codes, scale, fmt):
        s = torch.full((codes.shape[0], 1), scale, dtype=torch.uint8, device=DEV)
        return MxTensor(O.pack(codes, fmt), s, fmt)

    a = torch.zeros(a_codes.shape[0], 32, dtype=torch.int64, device=DEV)
    a[:, :2] = a_codes
    k = torch.arange(64, device=DEV)
    gate, up = (torch.zeros(64, 32, dtype=torch.int64, device=DEV) for _ in range(2))
    gate[:, 0], up[:, 1] = k % 8, k // 8 % 8
    return tensor(a, a_scale, "mxfp8"), tensor(gate, gate_scale, "mxfp4"), tensor(up, up_scale,
                                                                                  "mxfp4")


def _exact(a, gate, up):
    va = O.decode(a.codes, a.scales, "mxfp8")
    g = va @ O.decode(gate.codes, gate.scales, "mxfp4").t()
    u = va @ O.decode(up.codes, up.scales, "mxfp4").t()
    return g, u, g * torch.sigmoid(g) * u


@pytest.mark.parametrize("gate_scale", [115, 120, 122, 124, 125])
@pytest.mark.parametrize("short", [False, True])
def test_gates_of_all_sizes(gate_scale, short):
    """All pairs of E4M3 values by all pairs of E2M1: gates up to 2688 2^(s - 127),
    with many values close to a rounding border of the result."""
    from nano_vllm_metal_amd import mx_swiglu

    c = torch.arange(127, device=DEV)
    both = torch.cat((c, c + 128))
    codes = torch.cartesian_prod(both, c)
    a, gate, up = _operands(codes, 127, gate_scale, 127)
    y = mx_swiglu(a, gate, up, "mxfp8", short)
    g, u, h = _exact(a, gate, up)
    far = torch.where(g < -88.7, h.abs(), torch.zeros_like(h))  # (may be zero)
    O.check_quantized(y.codes, y.scales, "mxfp8", h, REL * h.abs() + far + 2.0 ** -148 * (1 + u.abs()))


@pytest.mark.parametrize("seed", range(4))
def test_gates_of_many_bits(seed):
    """Gates from -84 to -9 and ups that are sums of a large and a small product, 18
    bits in all, so exact: some of 26 million results lie within 2^-20 of a rounding
    border.  (A block's gates are alike but for the small product: of different ones
    the larger results' scale would leave the others nothing.)"""
    from nano_vllm_metal_amd import MxTensor, mx_swiglu

    g = torch.Generator(device=DEV).manual_seed(seed)

    def codes(rows, low, high):
        return torch.randint(low, high, (rows,), device=DEV, generator=g)

    M, K = 400_000, 64
    a = torch.zeros(M, 32, dtype=torch.int64, device=DEV)
    a[:, 0], a[:, 1] = 128 + codes(M, 0x4C, 0x5F), codes(M, 0x01, 0x38)  # -6 to -28, 2^-9 to 1
    a[:, 2], a[:, 3] = codes(M, 0x38, 0x40), codes(M, 0x01, 0x20)        # 1 to 2, up to 0.06
    w = torch.zeros(2, K, 32, dtype=torch.int64, device=DEV)
    for i in range(2):
        w[i, :, 2 * i], w[i, :, 2 * i + 1] = codes(K, 2, 6), codes(K, 1, 8)
    w[0, :32, 0], w[0, 32:, 0] = 5, 3  # 3 and 1.5
    w[0, :32, 1], w[0, 32:, 1] = 1 + seed, 7 - seed
    scale = lambda rows: torch.full((rows, 1), 127, dtype=torch.uint8, device=DEV)  # noqa: E731
    x = MxTensor(O.pack(a, "mxfp8"), scale(M), "mxfp8")
    gate, up = (MxTensor(O.pack(v, "mxfp4"), scale(K), "mxfp4") for v in w)
    gt, u, h = _exact(x, gate, up)
    assert gt.min() > -88.7 and ((gt * 2 ** 10).round() == gt * 2 ** 10).all()
    y = mx_swiglu(x, gate, up)
    O.check_quantized(y.codes, y.scales, "mxfp8", h, REL * h.abs())


def test_gates_just_above_where_exp_overflows():
    """-88.5 to -87: 1 / (1 + exp(-g)) is below float32's normal range."""
    from nano_vllm_metal_amd import mx_swiglu

    # 1.375 * 64 = 88, times E2M1 values at 2^0; ups of one size, so that a block is
    # of gates of -88 alone
    codes = torch.tensor([[128 + 0x6B, 0x38 + i] for i in range(8)], device=DEV)
    assert O.elements("mxfp8")[0x6B] == 88
    a, gate, up = _operands(codes, 127, 127, 140)
    gate.codes[:, 0] = 2  # (1.0)
    up.codes[:, 0] = 0x20
    y = mx_swiglu(a, gate, up)
    g, u, h = _exact(a, gate, up)
    assert (g == -88).all() and (h != 0).all()
    O.check_quantized(y.codes, y.scales, "mxfp8", h, REL * h.abs() + 2.0 ** -148 * u.abs())


def test_gates_near_the_end_of_float32():
    """Finite gates up to 3.2e38 with small ups: the product is finite, and so is its
    block; below -88.7 zeros, whatever the size."""
    from nano_vllm_metal_amd import mx_swiglu

    codes = torch.tensor([[0x38, 0x38], [0x38 + 2, 0x38], [0x80 + 0x38, 0x38], [0x80 + 0x3A, 0x40],
                          [0x30, 0x30]], device=DEV)
    a, gate, up = _operands(codes, 187, 127 + 65, 127 - 90)
    y = mx_swiglu(a, gate, up)
    g, u, h = _exact(a, gate, up)
    assert 3.1e38 < g.max() < 3.4e38 and g.min() < -3.1e38
    value = O.decode(y.codes, y.scales, "mxfp8")
    assert torch.isfinite(value).all() and (value[2:4] == 0).all()
    h = torch.where(g < -88.7, torch.zeros_like(h), h)
    O.check_quantized(y.codes, y.scales, "mxfp8", h, REL * h.abs())


def test_gates_that_are_not_finite():
    """g / (1 + exp(-g)): infinity stays, minus infinity and NaN are NaN; any of them
    takes its block along, and no other."""
    from nano_vllm_metal_amd import mx_swiglu

    codes = torch.tensor([[0x38, 0x38], [0x7E, 0x38], [0x80 + 0x7E, 0x38], [0x7F, 0x38]], device=DEV)
    a, gate, up = _operands(codes, 187, 127 + 65, 127 - 60)
    gate.codes[:32] = 0
    gate.codes[:32, 0] = 1  # 0.5: the first block's gates
    a.scales[0] = 60
    y = mx_swiglu(a, gate, up)
    value = O.decode(y.codes, y.scales, "mxfp8")
    assert torch.isfinite(value[0]).all()
    # 448 * 2^60 * 0.5 * 2^65 is past float32's range
    assert torch.isnan(value[1:, :32]).all()
