"""Sums of the microscaled products (include/nvm_mx.h): exact products and float32
sums whatever the sizes of neighbouring activations, and the shorter sums that a
caller may ask for.  Oracle: float64 products of the decoded operands.

Bounds: float32 sums of N products are off by at most N * 2^-23 * sum |a w| (each
addition by at most one unit in the last place), and not at all where every sum
of some of a row's products is a multiple of u and below 2^24 u.  E4M3 elements
are multiples of 2^-9 up to 448, E2M1 ones of 2^-1 up to 6: four products are
multiples of 2^-10 and below 2^14 together.
"""

from __future__ import annotations

import pytest
import torch

from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FMTS = ["mxfp4", "mxfp8"]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _val(t):
    return O.decode(t.codes, t.scales, t.fmt)


def _codes(g, rows, n, fmt):
    """Any finite codes."""
    c = torch.randint(0, 256, (rows, n // 2 if fmt == "mxfp4" else n), dtype=torch.uint8,
                      device=DEV, generator=g)
    return torch.where((c & 127) == 127, c - 1, c) if fmt == "mxfp8" else c


def _tensor(codes, scale, fmt):
    """All scales of a row alike: ``scale`` a number, or one a row."""
    from nano_vllm_metal_amd import MxTensor

    n = codes.shape[1] * (2 if fmt == "mxfp4" else 1)
    s = torch.as_tensor(scale, dtype=torch.uint8, device=DEV)
    return MxTensor(codes, s.reshape(-1, 1).expand(codes.shape[0], n // 32).contiguous(), fmt)


def _eight_apart(g, M, N):
    """E4M3 rows with four values, of all sizes, among eight neighbours: row m's in
    eight m % (N / 8)."""
    c = _codes(g, M, N, "mxfp8")
    k, m = torch.arange(N, device=DEV), torch.arange(M, device=DEV)[:, None]
    keep = (k // 8 == m % (N // 8)) & ((k + m // (N // 8)) % 2 == 0)
    return torch.where(keep, c, torch.zeros_like(c))


# one row to a few, some hundred and many, for every tile of every kernel (on 256
# CUs); rows of one step, of one run and a step, and cut short
SIZES = [(1, 32, 5), (16, 128, 16), (16, 2080, 4201), (11, 2080, 9001), (17, 160, 100),
         (33, 544, 257), (30, 2080, 4200), (48, 2592, 8003), (48, 448, 12200), (60, 2080, 8100),
         (90, 2080, 8100), (33, 992, 8008), (64, 512, 255), (127, 1024, 6100), (256, 2080, 5121),
         (510, 544, 5120), (512, 160, 5121), (390, 1184, 6001), (450, 640, 901), (300, 96, 1),
         (1000, 544, 1250), (1030, 96, 4000), (1030, 512, 8200), (1030, 672, 8193),
         (1100, 544, 15301), (1100, 160, 15200), (2600, 672, 8200), (3900, 160, 8100),
         (3900, 32, 8104), (3900, 672, 8100)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_small_activations_beside_large_ones_count(M, N, K):
    """Bit for bit: what a sum of sizes from 2^-10 to 2688 has, float32 holds."""
    from nano_vllm_metal_amd import mx_linear

    g = _gen(M + N + K)
    a = _tensor(_eight_apart(g, M, N), torch.randint(100, 150, (M,), device=DEV, generator=g),
                "mxfp8")
    w = _tensor(_codes(g, K, N, "mxfp4"), torch.randint(100, 150, (K,), device=DEV, generator=g),
                "mxfp4")
    y = mx_linear(a, w, torch.float32)
    assert torch.equal(y.double(), _val(a) @ _val(w).t())


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("fmt", FMTS)
def test_sums_are_float32(M, N, K, fmt):
    from nano_vllm_metal_amd import mx_linear

    g = _gen(M + N + K)
    a, w = _tensor(_codes(g, M, N, fmt), 127, fmt), _tensor(_codes(g, K, N, "mxfp4"), 120, "mxfp4")
    va, vw = _val(a), _val(w)
    off = (mx_linear(a, w, torch.float32).double() - va @ vw.t()).abs()
    assert (off <= N * 2.0 ** -23 * (va.abs() @ vw.abs().t())).all()


@pytest.mark.parametrize("M", [3, 70, 600])
def test_every_code_at_every_scale(M):
    """One value a row, so the product is exact: all E4M3 codes by all scales that
    keep it inside float32, times every E2M1 code; 255 is NaN in either operand."""
    from nano_vllm_metal_amd import MxTensor, mx_linear

    N, K = 160, 272
    g = _gen(M)
    w = _tensor(_codes(g, K, N, "mxfp4"), 127, "mxfp4")
    for first in range(0, 256, 64):
        b = torch.randint(first, first + 64, (M, 1), device=DEV, generator=g).clamp(3, 243)
        c = torch.zeros(M, N, dtype=torch.uint8, device=DEV)
        m = torch.arange(M, device=DEV)
        c[m, (m * 37 + first) % N] = _codes(g, M, 32, "mxfp8")[:, 0]
        a = MxTensor(c, b.to(torch.uint8).expand(M, N // 32).contiguous(), "mxfp8")
        y = mx_linear(a, w, torch.float32)
        want = (_val(a) @ _val(w).t()).float()
        assert torch.equal(y, want)
    bad = a.scales.clone()
    bad[M // 2, 1] = 255
    y = mx_linear(MxTensor(c, bad, "mxfp8"), w, torch.float32)
    assert torch.isnan(y[M // 2]).all() and torch.equal(y[:M // 2], want[:M // 2])


# gate and up of K columns each
PAIRS = [(1, 2048, 768), (30, 2080, 6144), (48, 2080, 6144), (60, 2080, 6144), (64, 2592, 768),
         (130, 2080, 4096), (300, 160, 800), (401, 640, 544), (1000, 544, 1056), (1030, 640, 4128),
         (1100, 672, 7616), (3900, 96, 4064), (3900, 672, 4064)]


@pytest.mark.parametrize("M,N,K", PAIRS)
@pytest.mark.parametrize("ofmt", FMTS)
def test_gate_and_up_sums_are_float32(M, N, K, ofmt):
    """The codes are such as a value gets that is as near as float32 sums and a few
    float32 operations on them leave it (2^-20 of it)."""
    from nano_vllm_metal_amd import mx_swiglu

    g = _gen(M + N + K)
    x = torch.randn(M, N, device=DEV, generator=g) * torch.exp(torch.randn(N, device=DEV, generator=g))
    ca, sa = O.quantize(x.double(), "mxfp8")
    from nano_vllm_metal_amd import MxTensor

    a = MxTensor(O.pack(ca, "mxfp8"), sa.to(torch.uint8), "mxfp8")
    wg, wu = (_tensor(_codes(g, K, N, "mxfp4"), 120, "mxfp4") for _ in range(2))
    y = mx_swiglu(a, wg, wu, ofmt)
    va, vg, vu = _val(a), _val(wg), _val(wu)
    gate, up = va @ vg.t(), va @ vu.t()
    eg = N * 2.0 ** -23 * (va.abs() @ vg.abs().t())
    eu = N * 2.0 ** -23 * (va.abs() @ vu.abs().t())
    s = gate * torch.sigmoid(gate)
    d = 1.1 * eg * (up.abs() + eu) + s.abs() * eu + 2.0 ** -20 * (s * up).abs() + 2.0 ** -146
    O.check_quantized(y.codes, y.scales, ofmt, s * up, d)
    # and hardly any differs from the exact one's (2^-20 of a value lies within
    # reach of a rounding border once in some 10^4 values)
    c, b = O.quantize(s * up, ofmt)
    got = O.unpack(y.codes, ofmt)
    same = ((got == c) | ((got | c) & (O.SIGN[ofmt] - 1) == 0)).double().mean()
    assert same > 0.999 and (y.scales.long() == b).double().mean() > 0.999


# ------------------------------------------------------- the sums of the instruction


def _short_bound(a, w):
    """Beside the float32 sums: what lies below 2^-13 of the largest of eight
    products is dropped, less than 7 * 2^-13 of it for each eight."""
    bound = a.shape[1] * 2.0 ** -23 * (a.abs() @ w.abs().t())
    rows = max(1, 2 ** 27 // w.numel())
    for i in range(0, a.shape[0], rows):
        p = (a[i:i + rows, None, :] * w[None]).abs()
        bound[i:i + rows] += 7 * 2.0 ** -13 * p.unflatten(-1, (-1, 8)).amax(-1).sum(-1)
    return bound


@pytest.mark.parametrize("M,N,K", [s for s in SIZES if s[0] * s[1] * s[2] < 3 * 10 ** 9])
def test_short_sums(M, N, K):
    from nano_vllm_metal_amd import mx_linear

    g = _gen(M + N + K)
    a, w = _tensor(_codes(g, M, N, "mxfp8"), 127, "mxfp8"), _tensor(_codes(g, K, N, "mxfp4"), 120,
                                                                     "mxfp4")
    y = mx_linear(a, w, torch.float32, short_sums=True)
    va, vw = _val(a), _val(w)
    assert ((y.double() - va @ vw.t()).abs() <= _short_bound(va, vw)).all()


@pytest.mark.parametrize("M,N,K", [(5, 544, 96), (300, 160, 800), (1030, 640, 4128)])
def test_short_sums_of_gate_and_up(M, N, K):
    from nano_vllm_metal_amd import mx_swiglu

    g = _gen(M)
    a = _tensor(_codes(g, M, N, "mxfp8"), 120, "mxfp8")
    wg, wu = (_tensor(_codes(g, K, N, "mxfp4"), 120, "mxfp4") for _ in range(2))
    y = mx_swiglu(a, wg, wu, short_sums=True)
    va, vg, vu = _val(a), _val(wg), _val(wu)
    gate, up, eg, eu = va @ vg.t(), va @ vu.t(), _short_bound(va, vg), _short_bound(va, vu)
    s = gate * torch.sigmoid(gate)
    d = 1.1 * eg * (up.abs() + eu) + s.abs() * eu + 2.0 ** -20 * (s * up).abs() + 2.0 ** -146
    O.check_quantized(y.codes, y.scales, "mxfp8", s * up, d)


@pytest.mark.parametrize("M", [5, 70, 1030])
def test_short_sums_change_nothing_for_four_bit_activations(M):
    from nano_vllm_metal_amd import mx_linear, mx_swiglu

    g = _gen(M)
    a, w = _tensor(_codes(g, M, 672, "mxfp4"), 127, "mxfp4"), _tensor(_codes(g, 4096, 672, "mxfp4"),
                                                                       120, "mxfp4")
    assert torch.equal(mx_linear(a, w), mx_linear(a, w, short_sums=True))
    x, y = mx_swiglu(a, w, w), mx_swiglu(a, w, w, short_sums=True)
    assert torch.equal(x.codes, y.codes) and torch.equal(x.scales, y.scales)


def test_a_model_in_short_sums():
    """The attribute reaches every product: layer by layer its step is that of the
    operators asked likewise, and not the float32 one."""
    from nano_vllm_metal_amd import (Qwen3Config, Qwen3Model, mx_embedding, mx_linear, mx_swiglu,
                                     residual_rms_norm_mx)
    from nano_vllm_metal_amd.fused import residual_rms_norm

    c = Qwen3Config(hidden_size=256, num_hidden_layers=1, num_attention_heads=4,
                    num_key_value_heads=2, head_dim=64, vocab_size=1024, intermediate_size=640,
                    max_position_embeddings=64)
    m = Qwen3Model.random(c, device=DEV, seed=3, std=0.06, mode="mxfp4")
    tokens = torch.randint(0, 1024, (1, 40), device=DEV, generator=_gen(1))
    got = {}
    for short in (False, True):
        m.short_sums = short
        cache = m.create_kv_cache(16, 16)
        cache.add(0)
        seen = []
        attention = m._attention
        m._attention = lambda *a: seen.append(attention(*a)) or seen[-1]
        got[short] = m.forward(tokens, cache, [0], last_only=False)
        del m._attention
        layer, eps, kw = m.layers[0], c.rms_norm_eps, dict(short_sums=short)
        h = mx_embedding(tokens, m.embed_w, m.dtype)
        h, x = residual_rms_norm_mx(h, seen[0], layer.post_norm, eps)
        y = mx_linear(mx_swiglu(x, layer.mlp.w_gate, layer.mlp.w_up, **kw), layer.mlp.w_down,
                      m.dtype, **kw)
        _, x = residual_rms_norm(h, y, m.norm, eps)
        assert torch.equal(got[short], mx_linear(x, m.lm_head, **kw))
    assert not torch.equal(got[False], got[True])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bias_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M", [1, 70])
def test_bias_of_any_type_leaves_the_output_type(M, dtype, bias_dtype):
    """The product's rounding and the sum's: eps / 2 of each, and of the bias, which the
    sum takes as it is, none."""
    from nano_vllm_metal_amd import mx_linear

    g = _gen(M)
    a, w = _tensor(_codes(g, M, 96, "mxfp8"), 122, "mxfp8"), _tensor(_codes(g, 40, 96, "mxfp4"), 124,
                                                                    "mxfp4")
    b = (100 * torch.randn(40, device=DEV, generator=g)).to(bias_dtype)
    plain, y = mx_linear(a, w, dtype), mx_linear(a, w, dtype, b)
    assert y.dtype == dtype and y.shape == (M, 40)
    want = plain.double() + b.double()
    # (float32's own rounding of the sum comes first)
    tol = (torch.finfo(dtype).eps / 2 + 2.0 ** -24) * want.abs() * (1 + 2.0 ** -7)
    assert ((y.double() - want).abs() <= tol + torch.finfo(dtype).tiny).all()
    row = mx_linear(type(a)(a.codes[0], a.scales[0], "mxfp8"), w, dtype, b)
    assert row.shape == (40,) and row.dtype == dtype
