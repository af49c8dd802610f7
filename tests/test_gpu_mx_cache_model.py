"""The 4-bit KV cache and log probabilities in use: PagedKVCache, a layer's
steps one after the other, Qwen3Model and LLM.

A layer's steps are held to the 64-bit oracle on what the cache holds.  The
model is compared with itself on plain operators (the oracle's formulas in
torch), log-probabilities within 5e-2: both round the same bf16 tensors, an
attention output may differ by an ulp (2^-8) now and then, and that difference
travels through two layers, where it can move a key's code.
"""

from __future__ import annotations

import pytest
import torch

from oracle import mx_cache_oracle as C
from oracle import mx_oracle as MX
from test_qwen3_model import _cfg, _model, _tokens

DEV = "cuda:0"


# ---------------------------------------------------------------- CPU


def test_cache_of_four_bits():
    from nano_vllm_metal_amd import MxPages, PagedKVCache

    c = PagedKVCache(2, 3, 64, num_pages=5, page_size=4, device="cpu", kv_bits=4)
    assert type(c.key_pages[1]) is MxPages and c.value_pages[0].shape == (6, 3, 4, 64)
    size = sum(t.numel() for p in c.key_pages for t in (p.codes, p.scales))
    assert size * 8 == 4.25 * 2 * 6 * 3 * 4 * 64
    for kw, match in (({"kv_bits": 8}, "kv_bits"), ({"head_dim": 80, "kv_bits": 4}, "head dim"),
                      ({"head_dim": 288, "kv_bits": 4}, "head dim")):
        args = dict(num_layers=1, num_kv_heads=1, head_dim=64, num_pages=1, page_size=4, device="cpu")
        with pytest.raises(ValueError, match=match):
            PagedKVCache(**(args | kw))


def test_refused_counts_of_alternatives():
    from nano_vllm_metal_amd.llm import _check_top

    for n in (None, 0, 64):
        _check_top("x", n, 1000)
    for n, vocab in ((-1, 1000), (65, 1000), (11, 10)):
        with pytest.raises(ValueError, match="must be in"):
            _check_top("x", n, vocab)


# ---------------------------------------------------------------- GPU


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_cache_write_and_read(dt):
    from nano_vllm_metal_amd import PagedKVCache

    g = torch.Generator().manual_seed(1)
    for bits in (4, 16):
        c = PagedKVCache(2, 2, 64, num_pages=6, page_size=4, dtype=dt, device=DEV, kv_bits=bits)
        c.add(7)
        c.reserve(7, 9)
        pages, slots = c.slot_mapping([7], 9)
        k, v = (torch.randn(1, 9, 2, 64, generator=g).to(dt) for _ in range(2))
        c.write(1, k.to(DEV), v.to(DEV), pages, slots)
        for got, x in zip(c.read(1, pages, slots), (k, v)):
            x = x.reshape(9, 2, 64)
            if bits == 4:
                q, b = MX.quantize(x.double(), "mxfp4")
                x = MX.decode(MX.pack(q, "mxfp4"), b, "mxfp4").to(dt)
            assert got.dtype == dt and torch.equal(got.cpu(), x)
        assert all((t == 0).all() for t in c.read(0, pages, slots))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_steps_of_a_layer(dt):
    """Two requests of unequal length: prompts stored piece by piece, then single
    tokens, store and attention in turn; each step's output against the oracle
    over what the cache holds, and at the end every stored row against the
    oracle's own."""
    from nano_vllm_metal_amd import PagedKVCache, paged_attention_mx, qk_norm_rope_store_mx

    Hq, Hkv, D, ps, eps = 14, 2, 64, 8, 1e-6
    g = torch.Generator().manual_seed(2)
    cache = PagedKVCache(1, Hkv, D, num_pages=40, page_size=ps, dtype=dt, device=DEV, kv_bits=4)
    kp, vp = cache.key_pages[0], cache.value_pages[0]
    f = torch.outer(torch.arange(200).double(), 1e4 ** (-torch.arange(D // 2).double() / (D // 2)))
    cos, sin = f.cos().float(), f.sin().float()
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g)).to(dt) for _ in range(2))
    ids, rows = [3, 5], {3: [], 5: []}
    for s in ids:
        cache.add(s)
    for who, L in (([3], 37), ([5], 20), ([3, 5], 7), ([3, 5], 1), ([5], 1), ([3, 5], 1), ([3], 9)):
        B = len(who)
        qkv = (2 * torch.randn(B, L, (Hq + 2 * Hkv) * D, generator=g)).to(dt)
        pos = torch.tensor([cache.lens[s] + j for s in who for j in range(L)], dtype=torch.int32)
        for s in who:
            cache.reserve(s, L)
        pages, slots = cache.slot_mapping(who, L)
        bt, lens = cache.block_table(who, extra=L)
        q, _, _ = qk_norm_rope_store_mx(qkv.to(DEV), Hq, Hkv, D, qw.to(DEV), kw.to(DEV), eps,
                                        pos.to(DEV), cos.to(DEV), sin.to(DEV), pages, slots, kp, vp)
        q = q.view(B, L, Hq, D).transpose(1, 2)
        got = paged_attention_mx(q, kp, vp, bt, lens, mask="causal")
        cache.advance(who, L)
        held = [(p.codes.cpu(), p.scales.cpu()) for p in (kp, vp)]
        want, bound = C.attention(q.cpu(), *held, bt.cpu(), lens.cpu(), D ** -0.5, True,
                                   C.weight_error(L, D, dt))
        bound = bound + torch.finfo(dt).eps / 2 * want.abs() + torch.finfo(dt).tiny
        assert ((got.cpu().double() - want).abs() <= bound).all(), (who, L)
        for i, s in enumerate(who):
            rows[s].append((qkv[i].double().reshape(L, -1, D), pos[i * L:(i + 1) * L].long()))
    for s in ids:
        x = torch.cat([r[0] for r in rows[s]])
        p = torch.cat([r[1] for r in rows[s]])
        j = torch.arange(len(x))
        assert torch.equal(p, j)
        page = torch.tensor(cache.pages[s])[j // ps]
        ke, ks = C.norm_rope(x[:, Hq:Hq + Hkv], kw, cos[p], sin[p], eps)
        MX.check_quantized(kp.codes.cpu()[page, :, j % ps], kp.scales.cpu()[page, :, j % ps], "mxfp4",
                           ke, 2.0 ** -40 * ks)
        c, b = MX.quantize(x[:, Hq + Hkv:], "mxfp4")
        assert torch.equal(vp.codes.cpu()[page, :, j % ps], MX.pack(c, "mxfp4"))
        assert torch.equal(vp.scales.cpu()[page, :, j % ps], b.to(torch.uint8))


def _plain_store(qkv, Hq, Hkv, D, qw, kw, eps, pos, cos, sin, page_ids, slots, kp, vp, want_kv=False,
                 out_dtype=None):
    dt = qkv.dtype
    x = qkv.reshape(-1, Hq + 2 * Hkv, D)
    c, s = cos[pos.long()], sin[pos.long()]
    q = C.norm_rope(x[:, :Hq], qw, c, s, eps)[0].to(dt)
    k = C.norm_rope(x[:, Hq:Hq + Hkv], kw, c, s, eps)[0]
    v = x[:, Hq + Hkv:]
    for pages, y in ((kp, k), (vp, v)):
        codes, b = MX.quantize(y.double(), "mxfp4")
        pages.codes[page_ids.long(), :, slots.long()] = MX.pack(codes, "mxfp4")
        pages.scales[page_ids.long(), :, slots.long()] = b.to(torch.uint8)
    odt = out_dtype or dt
    return q.to(odt), k.to(dt).to(odt) if want_kv else None, v.to(odt) if want_kv else None


def _plain_attention(q, kp, vp, bt, lens, scale=None, mask=None, out_dtype=None):
    held = [(p.codes.cpu(), p.scales.cpu()) for p in (kp, vp)]
    o, _ = C.attention(q.cpu(), *held, bt.cpu(), lens.cpu(), scale, mask == "causal")
    return o.to(q.device, out_dtype or q.dtype)


@pytest.mark.gpu
def test_model_on_plain_operators(monkeypatch):
    """Initial prefill, a chunk after it, single tokens in a batch."""
    from nano_vllm_metal_amd import qwen3

    m = _model(7)

    def steps():
        cache = m.create_kv_cache(40, page_size=4, kv_bits=4)
        cache.add(0)
        cache.add(1)
        out = [m.forward(torch.tensor([_tokens(12)], device=DEV), cache, [0], last_only=False)[0],
               m.forward(torch.tensor([_tokens(9, 2)], device=DEV), cache, [1], last_only=False)[0],
               m.forward(torch.tensor([_tokens(7, 3)], device=DEV), cache, [0], last_only=False)[0]]
        for t in _tokens(4, 4):
            out.append(m.forward(torch.tensor([[t], [t + 1]], device=DEV), cache, [0, 1]))
        return [torch.log_softmax(x.float(), -1) for x in out]

    got = steps()
    monkeypatch.setattr(qwen3, "qk_norm_rope_store_mx", _plain_store)
    monkeypatch.setattr(qwen3, "paged_attention_mx", _plain_attention)
    for i, (a, b) in enumerate(zip(got, steps())):
        err = float((a - b).abs().max())
        print(f"step {i}: max |log p - log p_plain| = {err:.3g}", flush=True)
        assert err <= 5e-2, i


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("graphs", [False, True])
def test_generate_with_logprobs(bits, graphs):
    """Every request gets the chain and the records it gets alone, eagerly."""
    from nano_vllm_metal_amd import LLM, SamplingParams

    m = _model(4)
    prompts = [_tokens(n, seed=20 + i) for i, n in enumerate((5, 11, 8, 8, 30))]
    llm = LLM(m, max_num_seqs=4, max_model_len=64, page_size=4, use_graphs=graphs, prefill_step=16,
              kv_bits=bits)
    outs = llm.generate(prompts, SamplingParams(max_tokens=6, logprobs=3))
    assert llm.cache.kv_bits == bits and llm.cache.free_pages == llm.cache.num_pages
    for p, o in zip(prompts, outs):
        assert [r.token_id for r in o.logprobs] == o.token_ids and len(o.token_ids) == 6
        cache = m.create_kv_cache(20, page_size=4, kv_bits=bits)
        cache.add(0)
        for s in range(0, len(p), 16):
            logits = m.forward(torch.tensor([p[s:s + 16]], device=DEV), cache, [0])
        for r in o.logprobs:
            x = logits[0].double().cpu()
            lp = torch.log_softmax(x, -1)
            order = torch.sort(x, descending=True, stable=True).indices[:3]
            assert r.token_id == int(torch.argmax(logits[0]))
            assert abs(r.logprob - float(lp[r.token_id])) < 1e-5
            assert abs(r.entropy + float((lp.exp() * lp).sum())) < 1e-5
            assert [i for i, _ in r.top] == order.tolist()
            assert max(abs(v - float(lp[i])) for i, v in r.top) < 1e-5
            logits = m.forward(torch.tensor([[r.token_id]], device=DEV), cache, [0])
    plain = llm.generate(prompts, SamplingParams(max_tokens=6))
    assert [o.token_ids for o in plain] == [o.token_ids for o in outs]
    assert all(o.logprobs is None for o in plain)
    with pytest.raises(ValueError, match="logprobs"):
        llm.generate(prompts, SamplingParams(logprobs=65))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 16])
def test_score(bits):
    """A prompt in one step and in several, of two tokens and of one."""
    from nano_vllm_metal_amd import LLM

    m = _model(8)
    llm = LLM(m, max_num_seqs=2, max_model_len=64, page_size=4, prefill_step=10, kv_bits=bits)
    prompts = [_tokens(n, seed=n) for n in (2, 1, 11, 31, 64)]
    got = llm.score(prompts, top=2)
    assert [len(r) for r in got] == [1, 0, 10, 30, 63]
    assert llm.cache.free_pages == llm.cache.num_pages and not llm.cache.lens
    for p, records in zip(prompts, got):
        assert [r.token_id for r in records] == p[1:]
        cache = m.create_kv_cache(20, page_size=4, kv_bits=bits)
        cache.add(0)
        rows = [m.forward(torch.tensor([p[s:min(s + 10, len(p) - 1)]], device=DEV), cache, [0],
                          last_only=False)[0] for s in range(0, len(p) - 1, 10)]
        if not rows:
            continue
        x = torch.cat(rows).double().cpu()
        lp = torch.log_softmax(x, -1)
        want = lp[torch.arange(len(records)), torch.tensor(p[1:])]
        have = torch.tensor([r.logprob for r in records], dtype=torch.float64)
        assert (have - want).abs().max() < 1e-5
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :2]
        assert [[i for i, _ in r.top] for r in records] == order.tolist()
    assert llm.score(prompts[2])[0] == [type(r)(r.token_id, r.logprob, r.entropy) for r in got[2]]
    for bad, match in (([[]], "empty"), ([_tokens(65)], "exceeds")):
        with pytest.raises(ValueError, match=match):
            llm.score(bad)
    with pytest.raises(ValueError, match="top"):
        llm.score(prompts, top=-1)


@pytest.mark.gpu
def test_score_refuses_ids_outside_the_vocabulary():
    """(Their log probability would count as zero.)"""
    from nano_vllm_metal_amd import LLM

    m = _model(8)
    llm = LLM(m, max_num_seqs=1, max_model_len=64, page_size=4)
    for bad in (-1, m.config.vocab_size):
        with pytest.raises(ValueError, match="token ids"):
            llm.score([_tokens(5), [1, bad, 2]])
    assert llm.cache.free_pages == llm.cache.num_pages
