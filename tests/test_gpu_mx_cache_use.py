"""GPU tests of the 4-bit KV cache and of token_logprobs as programs use them:
one after the other, captured and replayed, on two streams at once, and at
places that 32-bit offsets do not reach.

The kernels add in an order of their own, without atomics, so the same call
gives the same bits: each result here is compared with that of an eager call, or
of the same rows at other places, bit for bit.  (What those are worth is tested
against 64 bits elsewhere.)
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HQ, HKV, D, PS = 16, 4, 128, 16
V = 40009


def _state(seed, B, max_len, dt=torch.bfloat16):
    """A batch of sequences over one pool, and what a step needs."""
    import nano_vllm_metal_amd as P

    g = torch.Generator(device=DEV).manual_seed(seed)
    width = -(-max_len // PS)
    n = B * width + 3
    s = {"kp": P.MxPages.zeros(n, HKV, PS, D, DEV), "vp": P.MxPages.zeros(n, HKV, PS, D, DEV)}
    for pool in (s["kp"], s["vp"]):
        pool.codes.random_(0, 256, generator=g)
        pool.scales.random_(122, 129, generator=g)
    s["bt"] = torch.randperm(n, generator=g, device=DEV)[:B * width].reshape(B, width).int()
    s["qn"] = s["kn"] = torch.ones(D, device=DEV, dtype=dt)
    f = torch.outer(torch.arange(max_len, device=DEV).float(),
                    torch.arange(D // 2, device=DEV) * -0.1)
    s["cos"], s["sin"] = f.cos(), f.sin()
    s["head"] = torch.randn(HQ * D, V, generator=g, device=DEV) / 40
    return s


def _inputs(seed, s, B, L, lens, dt=torch.bfloat16):
    """L new tokens of each sequence, whose lengths with them are lens."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    lens = torch.tensor(lens, device=DEV, dtype=torch.int32)
    pos = (lens[:, None] - L + torch.arange(L, device=DEV)).int()
    page = torch.gather(s["bt"], 1, (pos.clamp_min(0) // PS).long())
    page = torch.where(pos < 0, -1, page).int()
    return {"qkv": torch.randn(B * L, (HQ + 2 * HKV) * D, generator=g, device=DEV).to(dt),
            "lens": lens, "pos": pos.reshape(-1).clamp_min(0), "page": page.reshape(-1),
            "slot": (pos % PS).int().reshape(-1),
            "token": torch.randint(0, V, (B * L,), generator=g, device=DEV)}


def _step(s, x, B, L, k=5):
    """Store, read back, attend, score."""
    import nano_vllm_metal_amd as P

    q, _, _ = P.qk_norm_rope_store_mx(x["qkv"], HQ, HKV, D, s["qn"], s["kn"], 1e-6, x["pos"],
                                      s["cos"], s["sin"], x["page"], x["slot"], s["kp"], s["vp"])
    kr, vr = P.paged_kv_read_mx(s["kp"], s["vp"], x["page"], x["slot"])
    o = P.paged_attention_mx(q.reshape(B, L, HQ, D).transpose(1, 2), s["kp"], s["vp"], s["bt"],
                             x["lens"], mask="causal")
    logits = (o.transpose(1, 2).reshape(B * L, HQ * D).float() @ s["head"]).to(torch.bfloat16)
    return (q, kr, vr, o, *P.token_logprobs(logits, x["token"], k))


def _same(a, b):
    assert len(a) == len(b)
    for i, (x, y) in enumerate(zip(a, b)):
        assert x.dtype == y.dtype and torch.equal(x.contiguous().view(torch.uint8),
                                                  y.contiguous().view(torch.uint8)), i


# one token of sequences of unlike lengths (a split kernel and its sum), one of a
# single short one, several rows of few and of many blocks
CASES = [(3, 1, 4000, [[4000, 17, 1], [1, 1, 3999], [2500, 0, 600], [64, 4000, 4000]]),
         (1, 1, 100, [[1], [100], [33], [64]]),
         (2, 37, 3000, [[3000, 37], [40, 2999], [37, 12], [500, 3000]]),
         (2, 300, 700, [[700, 300], [300, 699], [431, 5], [700, 700]])]


@pytest.mark.parametrize("B,L,max_len,lens", CASES)
def test_captured_and_replayed(B, L, max_len, lens):
    s = _state(L, B, max_len)
    x = _inputs(0, s, B, L, lens[0])
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        _step(s, x, B, L)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = _step(s, x, B, L)
    for turn, ln in enumerate(lens + lens[:1]):
        new = _inputs(10 + turn, s, B, L, ln)
        for n, t in new.items():
            x[n].copy_(t)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        # the eager call stores what is there already
        _same(kept, _step(s, new, B, L))
        torch.cuda.synchronize()


def test_two_graphs_at_once():
    """Each has its workspaces: two that replay at once do not meet."""
    ends = []
    for i, (B, L, max_len, lens) in enumerate((CASES[0], CASES[2])):
        s = _state(20 + i, B, max_len)
        x = _inputs(30 + i, s, B, L, lens[0])
        want = [t.clone() for t in _step(s, x, B, L)]
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = _step(s, x, B, L)
        ends.append((s, x, graph, stream, got, want))
    for _ in range(4):
        torch.cuda.synchronize()
        for _, _, graph, stream, _, _ in ends:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for *_, got, want in ends:
            _same(got, want)


def test_two_streams_at_once():
    runs = []
    for i, (B, L, max_len, lens) in enumerate((CASES[0], CASES[0], CASES[2])):
        s = _state(40 + i, B, max_len)
        x = _inputs(50 + i, s, B, L, lens[0])
        runs.append((s, x, B, L, [t.clone() for t in _step(s, x, B, L)], torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = [[] for _ in runs]
    for _ in range(5):
        for i, (s, x, B, L, _, stream) in enumerate(runs):
            with torch.cuda.stream(stream):
                got[i].append(_step(s, x, B, L))
    torch.cuda.synchronize()
    for i, run in enumerate(runs):
        for g in got[i]:
            _same(g, run[4])


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D,T", [(30, 2, 128, 1111), (33, 1, 64, 2500), (5, 5, 96, 4000),
                                        (9, 1, 256, 1700), (1, 1, 32, 50000)])
def test_many_tokens_are_stored_like_few(dt, Hq, Hkv, D, T):
    """A launch of many tokens takes several heads a group; 97 tokens at a time
    do not."""
    import nano_vllm_metal_amd as P

    g = torch.Generator(device=DEV).manual_seed(T)
    x = (3 * torch.randn(T, (Hq + 2 * Hkv) * D, generator=g, device=DEV)).to(dt)
    w = [(1 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(dt) for _ in range(2)]
    f = torch.outer(torch.arange(800, device=DEV).float(),
                    torch.arange(D // 2, device=DEV) * -0.1)
    pos = torch.randint(0, 800, (T,), generator=g, device=DEV, dtype=torch.int32)
    at = torch.randperm(T + 40, generator=g, device=DEV)[:T]
    page, slot = (at // 8).int(), (at % 8).int()
    n = -(-(T + 40) // 8)
    for odt in (dt, torch.float32):
        a, b = ([P.MxPages.zeros(n, Hkv, 8, D, DEV) for _ in range(2)] for _ in range(2))
        got = P.qk_norm_rope_store_mx(x, Hq, Hkv, D, *w, 1e-6, pos, f.cos(), f.sin(), page, slot,
                                      *a, want_kv=True, out_dtype=odt)
        parts = [P.qk_norm_rope_store_mx(x[i:i + 97], Hq, Hkv, D, *w, 1e-6, pos[i:i + 97], f.cos(),
                                         f.sin(), page[i:i + 97], slot[i:i + 97], *b, want_kv=True,
                                         out_dtype=odt) for i in range(0, T, 97)]
        _same(got, [torch.cat(t) for t in zip(*parts)])
        for u, v in zip(a, b):
            _same((u.codes, u.scales), (v.codes, v.scales))


def test_pages_beyond_four_gibibytes():
    """The same content on the last pages of a pool of 6 GiB of codes and on
    those of a small one."""
    import nano_vllm_metal_amd as P

    n = (6 << 30) // (HKV * PS * D // 2)
    big = [P.MxPages(torch.empty(n, HKV, PS, D // 2, dtype=torch.uint8, device=DEV),
                     torch.empty(n, HKV, PS, D // 32, dtype=torch.uint8, device=DEV))
           for _ in range(2)]
    for B, L, max_len, lens in (CASES[0], CASES[2]):
        s = _state(60, B, max_len)
        small = s["kp"].codes.shape[0]
        x = _inputs(61, s, B, L, lens[0])
        for u, v in zip(big, (s["kp"], s["vp"])):
            u.codes[n - small:].copy_(v.codes)
            u.scales[n - small:].copy_(v.scales)
        want = _step(s, x, B, L)
        far = dict(s, kp=big[0], vp=big[1], bt=s["bt"] + (n - small))
        y = dict(x, page=torch.where(x["page"] < 0, -1, x["page"] + (n - small)).int())
        _same(_step(far, y, B, L), want)
        for u, v in zip(big, (s["kp"], s["vp"])):
            _same((u.codes[n - small:], u.scales[n - small:]), (v.codes, v.scales))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_logits_beyond_32_bits(dt):
    """Rows 2^31 + 100 values apart, and many rows."""
    from nano_vllm_metal_amd import token_logprobs

    g = torch.Generator(device=DEV).manual_seed(3)
    ld = 2 ** 31 + 100
    x = torch.randn(2, V, generator=g, device=DEV).to(dt)
    t = torch.tensor([5, V - 1], device=DEV)
    far = torch.empty(ld + V, dtype=dt, device=DEV)
    wide = far.as_strided((2, V), (ld, 1))
    wide.copy_(x)
    want = token_logprobs(x, t, 7)
    _same(token_logprobs(wide, t, 7), want)
    del far, wide
    N = 2 ** 32 // V + 40
    rows = x[:1].expand(N, V).contiguous()
    rows[N - 1] = x[1]
    got = token_logprobs(rows, t[:1].expand(N).contiguous(), 3)
    one = token_logprobs(x, t[:1].expand(2).contiguous(), 3)
    assert (got.top_ids[:-1] == one.top_ids[0]).all()
    assert torch.equal(got.top_ids[-1], one.top_ids[1])
    assert (got.logprobs[:-1] == got.logprobs[0]).all()
    # (in one part here, in several of a row there: both within 16 u of 64 bits)
    for i, j in ((0, 0), (N - 1, 1)):
        off = (got.logprobs[i] - one.logprobs[j]).abs()
        assert off <= 64 * 2.0 ** -24 * (1 + one.logprobs[j].abs())
