"""GPU tests of the 4-bit cache where results went wrong or no test could have told:
weights that lost bits, NaNs lost between splits, incomplete first tiles, storage
exchanged under the pages, indices of unusual types.  Against the 64-bit results and
bounds of ``oracle/mx_cache_oracle.py``, and one rounding of the result.
"""

from __future__ import annotations

import math

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


@pytest.mark.parametrize("nan,top", [(3, 1999), (1990, 5), (700, 701), (0, 1000)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L", [1, 2, 40])
def test_nan_value_far_below_the_largest_score(L, D, nan, top):
    """A value block of NaNs at a position whose weight is 2^-430 of the row's largest,
    which float32 holds as zero: it shows in its 32 dims of the rows that see it,
    however many splits lie between the two."""
    g = torch.Generator().manual_seed(nan)
    q = torch.ones(1, 4, L, D, dtype=torch.bfloat16)
    k = (torch.zeros(128, 2, 16, D // 2, dtype=torch.uint8),
         torch.full((128, 2, 16, D // 32), 127, dtype=torch.uint8))
    v = C.random_pages(g, 128, 2, 16, D)
    bt = torch.randperm(128, generator=g)[:125][None].int()
    lens = torch.tensor([2000], dtype=torch.int32)
    k[0][int(bt[0, top // 16]), :, top % 16] = 0x22  # ones
    scale = 300.0 / D
    _check(_run(q, k, v, bt, lens, False, scale), q, k, v, bt, lens, False, scale)
    clean = _run(q, k, v, bt, lens, False, scale)
    v[1][int(bt[0, nan // 16]), 1, nan % 16, 1] = 255
    got = _run(q, k, v, bt, lens, False, scale)
    assert got[:, 2:, :, 32:64].isnan().all()
    got[:, 2:, :, 32:64] = clean[:, 2:, :, 32:64]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("L", [1, 2])
def test_nan_key_far_from_the_largest_score(L):
    """A key block of NaNs: the whole row, wherever the largest score is."""
    g = torch.Generator().manual_seed(L)
    q = torch.ones(1, 2, L, 128, dtype=torch.float16)
    k, v = (C.random_pages(g, 128, 1, 16, 128) for _ in range(2))
    bt = torch.randperm(128, generator=g)[:125][None].int()
    lens = torch.tensor([2000], dtype=torch.int32)
    k[0][int(bt[0, 1999 // 16]), :, 1999 % 16], k[1][int(bt[0, 1999 // 16]), :, 1999 % 16] = 0x22, 132
    k[1][int(bt[0, 0]), 0, 7, 2] = 255
    assert _run(q, k, v, bt, lens).isnan().all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L", [2, 33])
@pytest.mark.parametrize("causal", [False, True])
def test_several_rows_first_tile_incomplete(causal, L, D, dt):
    """Several rows over contexts of 0, 1, 63, 64 and 65 positions, a negative length, one
    beyond the table, and one whose first page is not there; every column sees the first
    64 positions where there is no mask."""
    g = torch.Generator().manual_seed(L + D)
    lens = torch.tensor([1, 63, 64, 65, 200, 0, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32)
    q = torch.randn(len(lens), 4, L, D, generator=g).to(dt)
    k, v = (C.random_pages(g, 120, 2, 16, D) for _ in range(2))
    bt = torch.randperm(120, generator=g)[:13 * len(lens)].reshape(len(lens), 13).int()
    bt[4, 0] = -1
    _check(_run(q, k, v, bt, lens, causal), q, k, v, bt, lens, causal)


def test_store_into_the_pages_present_storage():
    """Codes and scales with another storage (as after moving a cache): the step writes
    there, and nothing into the storage before."""
    from nano_vllm_metal_amd import MxPages, paged_kv_read_mx, qk_norm_rope_store_mx

    T, D = 5, 64
    g = torch.Generator(device=DEV).manual_seed(1)
    qkv = torch.randn(T, 4 * D, device=DEV, generator=g).bfloat16()
    one, pos = torch.ones(D, device=DEV).bfloat16(), torch.arange(T, device=DEV).int()
    cos, sin = torch.ones(9, D // 2, device=DEV), torch.zeros(9, D // 2, device=DEV)

    def store(kp, vp):
        qk_norm_rope_store_mx(qkv, 2, 1, D, one, one, 1e-6, pos, cos, sin, pos % 3, pos, kp, vp)

    want = [MxPages.zeros(3, 1, 16, D, DEV) for _ in range(2)]
    store(*want)
    got = [MxPages.zeros(3, 1, 16, D, DEV) for _ in range(2)]
    before = []
    for p in got:
        for t in (p.codes, p.scales):
            before.append(t.detach().view(t.shape))
            t.data = torch.zeros_like(t)
    store(*got)
    for a, b in zip(got, want):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and b.codes.any()
    assert not any(t.any() for t in before)
    for x, y in zip(paged_kv_read_mx(*got, pos % 3, pos), paged_kv_read_mx(*want, pos % 3, pos)):
        assert torch.equal(x, y)


def test_unsigned_indices():
    """Page ids and lengths of 32 unsigned bits: those beyond 2^31 are no page, and a
    length beyond everything."""
    from nano_vllm_metal_amd import paged_attention_mx, paged_kv_read_mx

    g = torch.Generator().manual_seed(2)
    k, v = (C.random_pages(g, 4, 2, 16, 64) for _ in range(2))
    kp, vp = _pages(k), _pages(v)
    ids = torch.tensor([1, 2 ** 31 + 1, 2 ** 32 - 1, 3], dtype=torch.uint32, device=DEV)
    slots = torch.tensor([3, 3, 3, 3], dtype=torch.uint32, device=DEV)
    got = paged_kv_read_mx(kp, vp, ids, slots)[0]
    want = paged_kv_read_mx(kp, vp, torch.tensor([1, -1, -1, 3], device=DEV), slots.int())[0]
    assert torch.equal(got, want) and got[0].any() and not got[1:3].any()
    q = torch.randn(1, 4, 1, 64, generator=g).bfloat16()
    bt, lens = torch.tensor([[2, 0]], dtype=torch.int32), torch.tensor([2 ** 31 + 7], dtype=torch.uint32)
    got = paged_attention_mx(q.to(DEV), kp, vp, bt.to(DEV), lens.to(DEV)).cpu()
    _check(got, q, k, v, bt, torch.tensor([32]))


@pytest.mark.parametrize("dt", [torch.float64, torch.float32, torch.float16, torch.bfloat16])
def test_cache_write_rounds_once(dt):
    """Values next to a border of E2M1 (2.5 and 2.5 + 2^-10 in a block of 6: 2 and 3), which
    a rounding to bf16 before would put on it."""
    from nano_vllm_metal_amd import PagedKVCache
    from oracle import mx_oracle as MX

    cache = PagedKVCache(1, 2, 64, 3, 16, torch.bfloat16, DEV, kv_bits=4)
    x = torch.randn(1, 5, 2, 64, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
    x[..., ::4], x[..., 1::4] = 6.0, 2.5 + 2.0 ** -10
    x[0, 2:] *= 2.0 ** -5
    x = x.to(dt)
    ids, slots = torch.tensor([0, 0, 2, 1, 1]), torch.tensor([0, 1, 15, 3, 4])
    cache.write(0, x.to(DEV), -x.to(DEV), ids.to(DEV), slots.to(DEV))
    for pages, y in ((cache.key_pages[0], x), (cache.value_pages[0], -x)):
        c, b = MX.quantize(y.reshape(5, 2, 64).double(), "mxfp4")
        assert torch.equal(MX.pack(c, "mxfp4"), pages.codes.cpu()[ids, :, slots])
        assert torch.equal(b.to(torch.uint8), pages.scales.cpu()[ids, :, slots])
    if dt == torch.float32:
        assert (cache.read(0, ids.to(DEV), slots.to(DEV))[0][0, :, 1::4] == 3).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L", [1, 2])
@pytest.mark.parametrize("s,top", [(13, 100), (22, 2000), (27, 5), (40, 2999), (100, 1500)])
def test_small_weights_are_all_of_the_result(s, top, L, D, dt):
    """One position of a weight of 1 and a value of zero, 2999 of weights 2^-s and values
    of one size: the result is these alone, and is compared relative to itself.  With
    u = 2^-23 their exponents are off by u (|s| + |m|) log2 e and (D + 4) u |s| (2^-9 at
    s = 100), exp2 by 2 u, the parts of a weight by 2^-16, sums of n terms by
    2 n u; then one rounding."""
    n, u = 3000, 2.0 ** -23
    g = torch.Generator().manual_seed(s)
    q = torch.ones(1, 2, L, D).to(dt)
    k, v = ((torch.full((190, 1, 16, D // 2), 0x22, dtype=torch.uint8),
             torch.full((190, 1, 16, D // 32), 127, dtype=torch.uint8)) for _ in range(2))
    bt = torch.randperm(190, generator=g)[:188][None].int()
    lens = torch.tensor([n], dtype=torch.int32)
    at = int(bt[0, top // 16]), 0, top % 16
    k[1][at] = 128          # a score of D above the others
    v[1][:] = 127 + s - 11  # (results of about 1.5)
    v[0][at] = 0
    scale = s * math.log(2.0) / D
    got = _run(q, k, v, bt, lens, False, scale).double()
    w = 2.0 ** -s
    want = (n - 1) * w / (1 + (n - 1) * w) * 2.0 ** (s - 11)
    m = 2 * s * math.log(2.0)  # the largest score; the others' are half of it
    rel = (1.5 * m * 1.45 + (D + 4) * m + 2) * u + 2.0 ** -16 + 2 * n * u + torch.finfo(dt).eps / 2
    assert ((got - want).abs() <= rel * want).all()


@pytest.mark.parametrize("D", [32, 96, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths_next_to_the_least_integer(causal, D):
    """Other head dims, several rows: lengths from -2^31 on are empty contexts (the first
    rows' bounds lie below -2^31), those up to 2^31 - 1 all of the table."""
    g = torch.Generator().manual_seed(D)
    lens = torch.tensor([-2 ** 31, -2 ** 31 + 3, -1, 2 ** 31 - 1, 30], dtype=torch.int32)
    q = torch.randn(5, 4, 6, D, generator=g).bfloat16()
    k, v = (C.random_pages(g, 20, 2, 16, D) for _ in range(2))
    bt = torch.randperm(20, generator=g)[:15].reshape(5, 3).int()
    got = _run(q, k, v, bt, lens, causal)
    assert (got[:3] == 0).all()
    _check(got, q, k, v, bt, lens, causal)
