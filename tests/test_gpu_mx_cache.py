"""GPU tests of the 4-bit KV cache (include/nvm_mx_cache.h) against 64-bit
results.

Codes and scales of values are compared bit for bit; keys go through float64,
so their codes have to be those of a value within 2^-40 of the exact one (sums
of at most 256 float64 squares, and a few products).  q is float32: each of the
two products of a rotated value has a relative error below 2^-19 (D/2 + 8
additions and products of 2^-24 at D = 256: 2^-17 of the sum of squares, half of
that in its root), and one rounding to 16 bits.  Attention: the bound that
``oracle/mx_cache_oracle.py`` derives, and one rounding of the result
(finfo.eps / 2).
"""

from __future__ import annotations

import pytest
import torch

from oracle import mx_cache_oracle as C
from oracle import mx_oracle as MX

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-6
ACTS = [torch.bfloat16, torch.float16]


def _pages(t):
    from nano_vllm_metal_amd import MxPages

    return MxPages(t[0].to(DEV), t[1].to(DEV))


def _tables(D, n, theta=1e4):
    f = torch.outer(torch.arange(n).double(), theta ** (-torch.arange(D // 2).double() / (D // 2)))
    return f.cos().float(), f.sin().float()


# ------------------------------------------------------------------- the store


def _store_case(seed, T, Hq, Hkv, D, ps, dt, P=None, max_pos=977):
    g = torch.Generator().manual_seed(seed)
    P = P or -(-T // ps) + 3
    s = {"qkv": (3 * torch.randn(T, (Hq + 2 * Hkv) * D, generator=g)).to(dt),
         "qw": (1 + 0.2 * torch.randn(D, generator=g)).to(dt),
         "kw": (1 + 0.2 * torch.randn(D, generator=g)).to(dt),
         "pos": torch.randint(0, max_pos, (T,), generator=g, dtype=torch.int32)}
    s["cos"], s["sin"] = _tables(D, max_pos)
    at = torch.randperm(P * ps, generator=g)[:T]
    s["page"], s["slot"] = (at // ps).int(), (at % ps).int()
    s["k"], s["v"] = (C.random_pages(g, P, Hkv, ps, D) for _ in range(2))
    return s


def _store(s, Hq, Hkv, D, kp, vp, **kw):
    from nano_vllm_metal_amd import qk_norm_rope_store_mx

    d = {n: s[n].to(DEV) for n in ("qkv", "qw", "kw", "pos", "cos", "sin", "page", "slot")}
    return qk_norm_rope_store_mx(d["qkv"], Hq, Hkv, D, d["qw"], d["kw"], EPS, d["pos"], d["cos"],
                                 d["sin"], d["page"], d["slot"], kp, vp, **kw)


def _check_store(s, Hq, Hkv, D, kp, vp, q, k=None, v=None):
    dt = s["qkv"].dtype
    T = len(s["qkv"])
    x = s["qkv"].double().reshape(T, Hq + 2 * Hkv, D)
    cos, sin = s["cos"][s["pos"].long()], s["sin"][s["pos"].long()]
    qe, qs = C.norm_rope(x[:, :Hq], s["qw"], cos, sin, EPS)
    half = torch.finfo(dt).eps / 2
    tiny = torch.finfo(dt).tiny * half  # a subnormal's rounding
    assert ((q.cpu().double() - qe).abs() <= half * qe.abs() + 2.0 ** -18 * qs + tiny).all()
    ke, ks = C.norm_rope(x[:, Hq:Hq + Hkv], s["kw"], cos, sin, EPS)
    ve = x[:, Hq + Hkv:]
    page, slot = s["page"].long(), s["slot"].long()
    MX.check_quantized(kp.codes.cpu()[page, :, slot], kp.scales.cpu()[page, :, slot], "mxfp4", ke,
                       2.0 ** -40 * ks)
    c, b = MX.quantize(ve, "mxfp4")
    assert torch.equal(MX.pack(c, "mxfp4"), vp.codes.cpu()[page, :, slot])
    assert torch.equal(b.to(torch.uint8), vp.scales.cpu()[page, :, slot])
    # every other slot is as it was
    for pages, before in ((kp, s["k"]), (vp, s["v"])):
        for now, old in ((pages.codes, before[0]), (pages.scales, before[1])):
            now, old = now.cpu().clone(), old.clone()
            now[page, :, slot] = 0
            old[page, :, slot] = 0
            assert torch.equal(now, old)
    if k is not None:
        assert ((k.cpu().double() - ke).abs() <= half * ke.abs() + 2.0 ** -40 * ks + tiny).all()
        assert torch.equal(v.cpu().double(), ve)


@pytest.mark.parametrize("dt", ACTS)
@pytest.mark.parametrize("T,Hq,Hkv,D,ps", [
    (1, 32, 4, 128, 16),
    (5, 14, 2, 64, 24),      # heads of different kinds in a wavefront
    (37, 3, 1, 96, 7),       # twelve of sixteen lanes, odd pages
    (9, 2, 2, 256, 16),
    (3, 1, 1, 32, 1),        # pages of one slot
    (4, 5, 5, 160, 3),
    (300, 32, 4, 128, 16),
])
def test_store_shapes(dt, T, Hq, Hkv, D, ps):
    s = _store_case(T + D, T, Hq, Hkv, D, ps, dt)
    kp, vp = _pages(s["k"]), _pages(s["v"])
    q, k, v = _store(s, Hq, Hkv, D, kp, vp, want_kv=T % 2 == 1)
    assert q.dtype == dt and q.shape == (T, Hq, D) and (k is None) == (T % 2 == 0)
    _check_store(s, Hq, Hkv, D, kp, vp, q, k, v)


def test_store_float32_outputs_hold_the_rounded_values():
    s = _store_case(3, 11, 8, 2, 128, 16, torch.float16)
    kp, vp = _pages(s["k"]), _pages(s["v"])
    a = _store(s, 8, 2, 128, kp, vp, want_kv=True)
    b = _store(s, 8, 2, 128, kp, vp, want_kv=True, out_dtype=torch.float32)
    for x, y in zip(a, b):
        assert y.dtype == torch.float32 and torch.equal(x.float(), y)


def test_store_slots_that_are_not_there():
    """Page ids outside the pool and slots outside a page: nothing is written,
    q is as ever; positions outside the tables are clamped."""
    s = _store_case(5, 8, 4, 2, 64, 16, torch.bfloat16)
    P = len(s["k"][0])
    s["page"][:] = torch.tensor([-1, P, 2 ** 31 - 1, 0, 0, 0, -5, P + 7], dtype=torch.int32)
    s["slot"][:] = torch.tensor([0, 0, 0, -1, 16, 2 ** 31 - 1, 3, 3], dtype=torch.int32)
    s["pos"][:2] = torch.tensor([-3, 10 ** 6], dtype=torch.int32)
    kp, vp = _pages(s["k"]), _pages(s["v"])
    q, _, _ = _store(s, 4, 2, 64, kp, vp)
    for pages, before in ((kp, s["k"]), (vp, s["v"])):
        assert torch.equal(pages.codes.cpu(), before[0])
        assert torch.equal(pages.scales.cpu(), before[1])
    s["pos"][:2] = torch.tensor([0, 976], dtype=torch.int32)
    assert torch.equal(q, _store(s, 4, 2, 64, kp, vp)[0])
    # an id that 32 bits would wrap stays outside
    s["page"] = torch.full((8,), 2 ** 32, dtype=torch.int64)
    s["slot"] = torch.zeros(8, dtype=torch.int64)
    _store(s, 4, 2, 64, kp, vp)
    assert torch.equal(kp.codes.cpu(), s["k"][0])


def test_store_nan_infinity_and_zero_rows():
    """A value that is not finite makes its block NaN (a key that is not: its
    whole row); zeros stand for zeros."""
    s = _store_case(7, 4, 2, 1, 64, 16, torch.bfloat16)
    x = s["qkv"].reshape(4, 4, 64)
    x[0, 2, 5] = float("inf")   # a key
    x[1, 3, 40] = float("nan")  # a value, second block
    x[2, 2:] = 0
    kp, vp = _pages(s["k"]), _pages(s["v"])
    _store(s, 2, 1, 64, kp, vp)
    page, slot = s["page"].long(), s["slot"].long()
    kd, vd = (MX.decode(p.codes.cpu()[page, 0, slot], p.scales.cpu()[page, 0, slot], "mxfp4")
              for p in (kp, vp))
    assert kd[0].isnan().any() and torch.isfinite(kd[1:]).all()
    assert vd[1, 32:].isnan().all() and torch.isfinite(vd[1, :32]).all()
    assert (kd[2] == 0).all() and (vd[2] == 0).all()


def test_store_strides_and_integer_types():
    """qkv with leading dimensions or rows apart, indices of 64 bits."""
    s = _store_case(9, 6, 4, 2, 64, 16, torch.bfloat16)
    kp, vp = _pages(s["k"]), _pages(s["v"])
    q, _, _ = _store(s, 4, 2, 64, kp, vp)
    wide = torch.zeros(6, 1024, dtype=torch.bfloat16)
    wide[:, 3:515] = s["qkv"]
    t = dict(s, qkv=wide[:, 3:515], pos=s["pos"].long(), page=s["page"].long(), slot=s["slot"].long())
    k2, v2 = _pages(s["k"]), _pages(s["v"])
    q2, _, _ = _store(t, 4, 2, 64, k2, v2)
    q3, _, _ = _store(dict(s, qkv=s["qkv"].reshape(2, 3, -1)), 4, 2, 64, k2, v2)
    assert torch.equal(q, q2) and torch.equal(q, q3)
    assert torch.equal(kp.codes, k2.codes) and torch.equal(vp.scales, v2.scales)


# -------------------------------------------------------------------- the read


@pytest.mark.parametrize("dt", ACTS + [torch.float32])
@pytest.mark.parametrize("T,Hkv,D,ps", [(1, 4, 128, 16), (37, 3, 96, 5), (130, 1, 32, 1)])
def test_read(dt, T, Hkv, D, ps):
    from nano_vllm_metal_amd import paged_kv_read_mx

    g = torch.Generator().manual_seed(T)
    P = -(-T // ps) + 1
    k, v = (C.random_pages(g, P, Hkv, ps, D) for _ in range(2))
    k[1][0, 0, 0, 0] = 255
    page = torch.randint(-1, P + 1, (T,), generator=g, dtype=torch.int32)
    slot = torch.randint(-1, ps + 1, (T,), generator=g, dtype=torch.int32)
    page[0] = slot[0] = 0
    got = paged_kv_read_mx(_pages(k), _pages(v), page.to(DEV), slot.to(DEV), dt)
    there = (page >= 0) & (page < P) & (slot >= 0) & (slot < ps)
    for x, (c, s) in zip(got, (k, v)):
        want = MX.decode(c, s, "mxfp4")[page.clamp(0, P - 1).long(), :, slot.clamp(0, ps - 1).long()]
        want = torch.where(there[:, None, None], want, torch.zeros_like(want))
        assert x.dtype == dt and torch.allclose(x.cpu(), want.to(dt), rtol=0, atol=0, equal_nan=True)


def test_pages_dequantize():
    from nano_vllm_metal_amd import MxPages

    k = C.random_pages(torch.Generator().manual_seed(1), 5, 3, 7, 96)
    assert torch.equal(_pages(k).dequantize().cpu().double(), MX.decode(*k, "mxfp4"))
    z = MxPages.zeros(3, 2, 16, 64, DEV)
    assert z.shape == (3, 2, 16, 64) and (z.dequantize(torch.float16) == 0).all()


# --------------------------------------------------------------- the attention


def _attention_case(seed, B, Hq, Hkv, D, ps, lens, L, dt, holes=0, past=0, q_scale=1.0, width=None):
    g = torch.Generator().manual_seed(seed)
    lens = torch.as_tensor(lens, dtype=torch.int32)
    width = width or max(1, int(-(-int(lens.max()) // ps)))
    P = B * width + 2
    q = (q_scale * torch.randn(B, Hq, L, D, generator=g)).to(dt)
    k, v = (C.random_pages(g, P, Hkv, ps, D) for _ in range(2))
    bt = torch.randperm(P, generator=g)[:B * width].reshape(B, width).int()
    for n, value in ((holes, -1), (past, P)):
        for _ in range(n):
            bt[torch.randint(B, (), generator=g), torch.randint(width, (), generator=g)] = value
    return q, k, v, bt, lens


def _check_attention(q, k, v, bt, lens, causal, odt=None, scale=None):
    from nano_vllm_metal_amd import paged_attention_mx

    got = paged_attention_mx(q.to(DEV), _pages(k), _pages(v), bt.to(DEV), lens.to(DEV), scale=scale,
                             mask="causal" if causal else None, out_dtype=odt)
    odt = odt or q.dtype
    assert got.dtype == odt and got.shape == q.shape
    want, bound = C.attention(q, k, v, bt, lens, q.shape[-1] ** -0.5 if scale is None else scale,
                              causal, C.weight_error(*q.shape[2:], odt))
    bound = bound + torch.finfo(odt).eps / 2 * want.abs() + torch.finfo(odt).tiny
    off = (got.cpu().double() - want).abs()
    assert (off <= bound).all(), (f"{int((off > bound).sum())} of {off.numel()} off, "
                                  f"worst {float((off / bound).max()):.3g} of the bound")
    return got


@pytest.mark.parametrize("dt", ACTS + [torch.float32])
@pytest.mark.parametrize("Hq,Hkv,D,ps,lens", [
    (32, 4, 128, 16, [700, 1, 64, 65]),
    (16, 16, 64, 24, [333, 0, 129]),      # a head of keys for each, an empty request
    (14, 2, 64, 5, [511, 513, 700]),      # seven a kv head, around a block's eight tiles
    (16, 1, 128, 128, [90, 257]),         # sixteen
    (40, 2, 128, 16, [1030, 31]),         # twenty
    (6, 2, 96, 16, [77, 300]),            # other head dims
    (2, 1, 32, 16, [100]),
    (4, 4, 256, 3, [50, 2]),
])
def test_decode(dt, Hq, Hkv, D, ps, lens):
    case = _attention_case(Hq + D, len(lens), Hq, Hkv, D, ps, lens, 1, dt, holes=1, past=1)
    _check_attention(*case, causal=D != 64)


@pytest.mark.parametrize("odt", [torch.float16, torch.bfloat16, torch.float32])
def test_decode_output_types(odt):
    case = _attention_case(1, 2, 8, 2, 128, 16, [40, 333], 1, torch.bfloat16)
    _check_attention(*case, causal=True, odt=odt)


@pytest.mark.parametrize("dt", ACTS + [torch.float32])
@pytest.mark.parametrize("q_scale,scale", [(0.01, None), (30.0, None), (3.0, 1.0)])
def test_decode_query_magnitudes(dt, q_scale, scale):
    """Flat and one-sided weights."""
    case = _attention_case(2, 2, 16, 2, 128, 16, [500, 129], 1, dt, q_scale=q_scale)
    _check_attention(*case, causal=True, odt=torch.float32, scale=scale)


@pytest.mark.parametrize("dt", ACTS + [torch.float32])
@pytest.mark.parametrize("Hq,Hkv,D,ps,L,lens,causal", [
    (32, 4, 128, 16, 33, [33, 100, 500], True),   # eight a kv head, a first chunk among them
    (8, 8, 64, 4, 17, [17, 80], True),            # one
    (14, 2, 64, 24, 50, [49, 10, 333], True),     # seven; contexts shorter than the chunk
    (16, 8, 128, 24, 70, [200, 71], False),       # two, not causal
    (40, 2, 128, 16, 9, [300], True),             # twenty
    (6, 2, 96, 16, 5, [77, 300], True),           # other head dims
    (2, 1, 32, 16, 3, [2, 0], True),
    (4, 4, 256, 3, 7, [50, 8], False),
    (4, 1, 128, 16, 2, [1000], True),             # two rows of a long context
])
def test_several_rows(dt, Hq, Hkv, D, ps, L, lens, causal):
    case = _attention_case(L + D, len(lens), Hq, Hkv, D, ps, lens, L, dt, holes=2, past=1)
    _check_attention(*case, causal=causal, odt=torch.float32 if L == 50 else None)


def test_rows_that_see_nothing():
    """No context, no pages, or a causal bound before the first position: zeros."""
    from nano_vllm_metal_amd import paged_attention_mx

    q, k, v, bt, lens = _attention_case(4, 3, 8, 2, 128, 16, [40, 0, 64], 1, torch.bfloat16)
    bt[2] = -1
    got = _check_attention(q, k, v, bt, lens, True)
    assert (got[1] == 0).all() and (got[2] == 0).all() and (got[0] != 0).any()
    q, k, v, bt, lens = _attention_case(5, 2, 8, 2, 64, 16, [3, -7], 6, torch.float16)
    got = _check_attention(q, k, v, bt, lens, True)
    assert (got[0, :, :3] == 0).all() and (got[1] == 0).all()
    # no pages in the table at all, and an empty batch
    none = torch.empty((2, 0), dtype=torch.int32, device=DEV)
    got = paged_attention_mx(q.to(DEV), _pages(k), _pages(v), none, lens.to(DEV))
    assert got.shape == q.shape and (got == 0).all()
    got = paged_attention_mx(q[:0].to(DEV), _pages(k), _pages(v), none[:0], lens[:0].to(DEV))
    assert got.shape == (0, 8, 6, 64)


def test_attention_scale_signs():
    """A negative scale, and zero: all positions alike."""
    for L, D in ((1, 128), (1, 96), (9, 64)):
        q, k, v, bt, lens = _attention_case(13, 2, 8, 2, D, 16, [90, 33], L, torch.float16)
        _check_attention(q, k, v, bt, lens, True, scale=-0.2)
        _check_attention(q, k, v, bt, lens, True, scale=0.0)


@pytest.mark.parametrize("L", [1, 20])
@pytest.mark.parametrize("D", [64, 128, 96])
def test_slots_behind_the_context_do_not_count(L, D):
    """NaN blocks and the largest values in the last page's unused slots, in
    pages of other requests and on page ids past the context: nothing of it
    shows.  A NaN inside the context shows in every row that sees it."""
    from nano_vllm_metal_amd import paged_attention_mx

    q, k, v, bt, lens = _attention_case(6 + D, 2, 8, 2, D, 16, [71, 129], L, torch.bfloat16, width=12)

    def run():
        return paged_attention_mx(q.to(DEV), _pages(k), _pages(v), bt.to(DEV), lens.to(DEV),
                                  mask="causal")

    clean = run()
    used = torch.zeros(k[0].shape[0], 16, dtype=torch.bool)
    for b in range(2):
        j = torch.arange(int(lens[b]))
        used[bt[b].long()[j // 16], j % 16] = True
    for c, s in (k, v):
        c.transpose(1, 2)[~used] = 0x77
        s.transpose(1, 2)[~used] = 255
    assert torch.equal(run(), clean)
    page, slot = int(bt[0, 70 // 16]), 70 % 16
    v[1][page, 1, slot, 0] = 255
    got = run()
    # the last position is visible to the last row only
    assert got[0, 4:, -1, :32].isnan().all() and torch.equal(got[0, :4], clean[0, :4])
    assert torch.equal(got[0, 4:, :-1], clean[0, 4:, :-1]) and torch.equal(got[1], clean[1])
    v[1][page, 1, slot, 0] = 120
    k[1][page, 1, slot, 0] = 255
    got = run()
    assert got[0, 4:, -1].isnan().all() and torch.equal(got[0, :4], clean[0, :4])


def test_attention_query_strides():
    """A token-major query, one with rows apart, and one that has to be copied."""
    from nano_vllm_metal_amd import paged_attention_mx

    for L in (1, 19):
        q, k, v, bt, lens = _attention_case(8, 3, 8, 2, 64, 16, [90, 33, 64], L, torch.float16)
        kp, vp, bt, lens = _pages(k), _pages(v), bt.to(DEV), lens.to(DEV)
        qd = q.to(DEV)
        want = paged_attention_mx(qd, kp, vp, bt, lens, mask="causal")
        tokens = qd.transpose(1, 2).contiguous().transpose(1, 2)
        wide = torch.zeros(3, 9, L, 80, dtype=q.dtype, device=DEV)
        wide[:, 1:, :, 8:72] = qd
        odd = torch.zeros(3, 8, L, 65, dtype=q.dtype, device=DEV)
        odd[..., 1:] = qd
        for x in (tokens, wide[:, 1:, :, 8:72], odd[..., 1:],
                  qd.transpose(2, 3).contiguous().transpose(2, 3)):
            assert torch.equal(paged_attention_mx(x, kp, vp, bt.long(), lens.long(), mask="causal"),
                               want)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lo,hi", [(104, 104), (104, 140), (103, 103), (141, 141), (1, 1), (0, 0), (90, 127),
                                   (200, 200)])
def test_several_rows_value_scales(D, lo, hi):
    """Value scales inside f16's range, at its ends, just beyond and far beyond."""
    g = torch.Generator().manual_seed(lo + hi)
    q, k, v, bt, lens = _attention_case(11, 2, 8, 2, D, 16, [150, 97], 40, torch.bfloat16)
    v[1][:] = torch.where(torch.rand(v[1].shape, generator=g) < 0.5, lo, hi).to(torch.uint8)
    _check_attention(q, k, v, bt, lens, True)


def test_several_rows_many_small_weights():
    """One position far above 3000 others, which weigh 2^-13 to 2^-27 of it."""
    q, k, v, bt, lens = _attention_case(12, 1, 2, 1, 64, 16, [3000], 2, torch.bfloat16)
    q[:] = 1
    k[0][:], k[1][:] = 0x22, 127  # ones
    at = bt[0].long()
    for s, top in ((13.0, 100), (22.0, 2000), (27.0, 5)):
        k[1][at[top // 16], 0, top % 16] = 128  # a score of 64 above the others
        _check_attention(q, k, v, bt, lens, False, scale=s * 0.6931 / 64)
        k[1][at[top // 16], 0, top % 16] = 127


@pytest.mark.parametrize("L", [1, 3])
def test_attention_extreme_scales(L):
    """Blocks at both ends of the scales' range: keys and values of 2^-127 to
    2^-120 and beside them 2^100, queries to match."""
    q, k, v, bt, lens = _attention_case(10, 1, 4, 2, 128, 16, [100], L, torch.float32)
    k[1][:, :, :, 0], k[1][:, :, :, 1] = 3, 227
    q[..., :32] *= 2.0 ** 100
    q[..., 32:64] *= 2.0 ** -100
    v[1][:, :, :, 0], v[1][:, :, :, 1] = 8, 220
    _check_attention(q, k, v, bt, lens, True, odt=torch.float32)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("code", [0x22, 0x00])
@pytest.mark.parametrize("L", [1, 3])
@pytest.mark.parametrize("D", [64, 128, 96])
@pytest.mark.parametrize("odt", ACTS)
def test_key_block_of_nans_whatever_its_codes(odt, D, L, code, sign):
    """A scale of 255 is a NaN, no infinity that a score of one sign would hide:
    rows that see the position are NaN, others are not."""
    from nano_vllm_metal_amd import paged_attention_mx

    q, k, v, bt, lens = _attention_case(9, 2, 4, 2, D, 4, [37, 20], L, odt)
    q = torch.full_like(q, sign)
    at = 37 - L  # the first row's last position of request 0
    page, slot = int(bt[0, at // 4]), at % 4
    k[0][page, 1, slot] = code
    k[1][page, 1, slot, 0] = 255
    got = paged_attention_mx(q.to(DEV), _pages(k), _pages(v), bt.to(DEV), lens.to(DEV),
                             mask="causal").cpu()
    nan = torch.zeros(got.shape, dtype=torch.bool)
    nan[0, 2:] = True
    assert torch.equal(got.isnan(), nan)
    got = paged_attention_mx(q.to(DEV), _pages(k), _pages(v), bt.to(DEV),
                             torch.tensor([at, 20], dtype=torch.int32, device=DEV)).cpu()
    assert not got.isnan().any()
