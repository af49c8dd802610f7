"""GPU tests of the 4-bit cache where single results went wrong: weights that lost
bits.  Against the 64-bit results and bounds of ``oracle/mx_cache_oracle.py``, and
one rounding of the result.
"""

from __future__ import annotations

import pytest
import torch

from oracle import mx_cache_oracle as C

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _pages(t):
    from nano_vllm_metal_amd import MxPages

    return MxPages(t[0].to(DEV), t[1].to(DEV))


def _run(q, k, v, bt, lens, causal=False, scale=None):
    from nano_vllm_metal_amd import paged_attention_mx

    return paged_attention_mx(q.to(DEV), _pages(k), _pages(v), bt.to(DEV), lens.to(DEV), scale=scale,
                              mask="causal" if causal else None).cpu()


def _check(got, q, k, v, bt, lens, causal=False, scale=None):
    want, bound = C.attention(q, k, v, bt, lens, q.shape[-1] ** -0.5 if scale is None else scale,
                              causal)
    bound = bound + torch.finfo(q.dtype).eps / 2 * want.abs() + torch.finfo(q.dtype).tiny
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (f"{int((off > bound).sum())} of {off.numel()} off, "
                                  f"worst {float((off / bound).max()):.3g} of the bound")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L", [1, 2, 20])
def test_weights_of_values_that_cancel(L, D, dt):
    """Eight positions of nearly equal weights, values of 1 and -1: the result is some
    1/100 of the values, so its own rounding (2^-8 of that) hides no rounding of the
    weights to 2^-11."""
    g = torch.Generator().manual_seed(L + D)
    q = (0.02 * torch.randn(2, 8, L, D, generator=g)).to(dt)
    k, _ = (C.random_pages(g, 4, 2, 16, D) for _ in range(2))
    v = (torch.full((4, 2, 16, D // 2), 0x22, dtype=torch.uint8),
         torch.full((4, 2, 16, D // 32), 127, dtype=torch.uint8))
    v[0][:, :, 1::2] = 0xAA
    bt = torch.tensor([[2], [1]], dtype=torch.int32)
    lens = torch.tensor([8, 8], dtype=torch.int32)
    _check(_run(q, k, v, bt, lens), q, k, v, bt, lens)
