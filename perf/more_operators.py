"""The 4-bit KV cache and log probabilities, as performance cases.

Pages of the cache hold keys and values in MXFP4: a block of 32 consecutive
values of a head's row shares one power-of-two scale (E8M0, byte b stands for
2^(b - 127)), the values are E2M1, two a byte, the even one in the low half.
Codes are ``[P, Hkv, page_size, D / 2]``, scales ``[P, Hkv, page_size, D /
32]``.  Kinds:

* ``append``    per-head RMSNorm of q and k, rotation, keys and values into
  their slots (``qk_norm_rope_store_mx``), and what the slots then hold
  (``paged_kv_read_mx``)
* ``decode``    one query row a request over its pages (``paged_attention_mx``)
* ``chunk``     several query rows a request, causal (the same)
* ``logprobs``  log probabilities of given tokens, the entropy, and the most
  probable alternatives (``token_logprobs``)

Sizes are the repository's own: the attention of the Qwen3-30B-A3B
configuration (32 query and 4 kv heads of 128, positions up to 40960, a
vocabulary of 151936, pages of 16), prompts and prefill chunks of up to 4096
and 2048 tokens, and generic odd ones.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

BLOCK = 32
EPS = 1e-6
THETA = 1e6
MAX_POS = 40960
DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# query heads, kv heads, head dim
HEADS = [(32, 4, 128), (32, 4, 128), (16, 8, 64), (8, 8, 128), (14, 2, 64), (40, 2, 128), (16, 16, 64)]
MOST_CACHED = 16 * 40960 * 4 * 128  # values of a decode batch's keys
MOST_PAIRS = 2048 * 5120 * 32 * 128  # query rows x positions x heads x dims of a chunk
MOST_LOGITS = 2048 * 151936 * 2  # bytes


def listed():
    return [
        # one decoding request: the step between its q/k/v projection and its attention
        {"name": "append_1", "kind": "append", "T": 1, "q": 32, "kv": 4, "D": 128, "page": 16, "dtype": "bf16"},
        # an odd decode batch of a smaller fp16 model, pages of an odd size
        {"name": "append_37_f16", "kind": "append", "T": 37, "q": 16, "kv": 8, "D": 64, "page": 24, "dtype": "f16"},
        # a prompt of 4096 tokens
        {"name": "append_4096", "kind": "append", "T": 4096, "q": 32, "kv": 4, "D": 128, "page": 16, "dtype": "bf16"},
        # one request of a short conversation: latency
        {"name": "decode_1", "kind": "decode", "B": 1, "lo": 700, "ctx": 700, "q": 32, "kv": 4, "D": 128, "page": 16,
         "holes": 0, "dtype": "bf16"},
        # five requests of an fp16 model without shared heads, one of them empty, some of whose pages were dropped
        {"name": "decode_5_f16", "kind": "decode", "B": 5, "lo": 0, "ctx": 2999, "q": 16, "kv": 16, "D": 64, "page": 24,
         "holes": 3, "dtype": "f16"},
        # a serving batch of unequal contexts
        {"name": "decode_32", "kind": "decode", "B": 32, "lo": 500, "ctx": 4096, "q": 32, "kv": 4, "D": 128, "page": 16,
         "holes": 0, "dtype": "bf16"},
        # long documents, as far as the model's positions go
        {"name": "decode_16_long", "kind": "decode", "B": 16, "lo": 38000, "ctx": 40960, "q": 32, "kv": 4, "D": 128,
         "page": 16, "holes": 0, "dtype": "bf16"},
        # the last, ragged piece of three fp16 prompts, seven query heads a kv head
        {"name": "chunk_100_f16", "kind": "chunk", "B": 3, "L": 100, "lo": 100, "ctx": 1501, "q": 14, "kv": 2, "D": 64,
         "page": 24, "dtype": "f16"},
        # a prefill step of a long prompt over what is cached of it: the largest case
        {"name": "chunk_2048", "kind": "chunk", "B": 1, "L": 2048, "lo": 6144, "ctx": 6144, "q": 32, "kv": 4, "D": 128,
         "page": 16, "dtype": "bf16"},
        # one generated token with five alternatives
        {"name": "logprobs_1", "kind": "logprobs", "N": 1, "V": 151936, "k": 5, "dtype": "bf16"},
        # an odd batch of float32 logits over an odd vocabulary, twenty alternatives
        {"name": "logprobs_33_f32", "kind": "logprobs", "N": 33, "V": 50257, "k": 20, "dtype": "f32"},
        # a prompt's tokens scored, a prefill step at a time
        {"name": "logprobs_2048", "kind": "logprobs", "N": 2048, "V": 151936, "k": 5, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "decode", "chunk", "chunk", "logprobs", "logprobs"])
    if kind == "logprobs":
        V = rng.choice([151936, 50257, _log(rng, 1000, 151936)])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        N = min(_log(rng, 1, 2048), MOST_LOGITS // (V * SIZE[dtype]))
        return {"kind": kind, "N": N, "V": V, "k": rng.choice([0, 1, 5, 20, rng.randint(2, 20)]), "dtype": dtype}
    Hq, Hkv, D = rng.choice(HEADS)
    common = {"kind": kind, "q": Hq, "kv": Hkv, "D": D, "page": rng.choice([16, 16, 24, 64, rng.randint(1, 100)]),
              "dtype": rng.choice(["bf16", "bf16", "f16"])}
    if kind == "append":
        most = 4096 * 40 * 128 // ((Hq + 2 * Hkv) * D)
        return common | {"T": min(_log(rng, 1, 4096), most)}
    if kind == "decode":
        B = _log(rng, 1, 64)
        ctx = min(_log(rng, 1, MAX_POS), MOST_CACHED // (B * Hkv * D))
        return common | {"B": B, "lo": rng.choice([ctx, rng.randint(0, ctx)]), "ctx": ctx,
                         "holes": rng.choice([0, 0, 2])}
    B, L = rng.randint(1, 4), _log(rng, 2, 2048)
    ctx = min(L + rng.choice([0, _log(rng, 1, 8192)]), max(1, MOST_PAIRS // (B * L * Hq * D)))
    return common | {"B": B, "L": L, "lo": rng.choice([ctx, rng.randint(ctx // 2, ctx)]), "ctx": ctx}


def _lens(case):
    """Context lengths of the case's requests: from ``ctx`` down to ``lo``."""
    B, lo, hi = case["B"], case["lo"], case["ctx"]
    return [hi - (hi - lo) * b // max(B - 1, 1) for b in range(B)]


# ------------------------------------------------------------------ plain form


def _pow2(e, dtype):
    return torch.ldexp(torch.ones((), dtype=dtype, device=e.device), e)


def _quantize(x):
    """E2M1 values and scale exponents of rows x [..., n]."""
    g = x.reshape(*x.shape[:-1], -1, BLOCK)
    amax = g.abs().amax(-1)
    e = torch.where(amax > 0, torch.frexp(amax)[1] - 3, -127).clamp(-127, 127)
    v = g * _pow2(-e, x.dtype)[..., None]
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(x.dtype)
    return ((torch.round(a / step) * step).clamp(max=6.0) * torch.sign(v)).reshape(x.shape), e


def _pack(x):
    """Codes and scale bytes of rows x [..., n]."""
    q, e = _quantize(x)
    grid = torch.tensor(E2M1, dtype=x.dtype, device=x.device)
    c = torch.bucketize(q.abs(), grid).to(torch.uint8) + 8 * (q < 0).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _unpack(codes, scales, dtype=torch.float32):
    """What codes and scale bytes stand for, [..., n]."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=dtype, device=codes.device)
    q = table[torch.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], -1).int()]
    s = _pow2(scales.to(torch.int32) - 127, dtype)
    return (q.reshape(*scales.shape, BLOCK) * s[..., None]).reshape(q.shape)


def _norm_rope(x, w, cos, sin):
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    a, b = y.chunk(2, -1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _append(s):
    Hq, Hkv, D = s["heads"]
    x = s["qkv"].reshape(-1, Hq + 2 * Hkv, D)
    p = s["positions"].long()
    cos, sin = s["cos"][p][:, None], s["sin"][p][:, None]
    q = _norm_rope(x[:, :Hq].float(), s["qw"].float(), cos, sin).to(x.dtype)
    # (64 bits: else a key next to a rounding border of 4 bits would go by a sum's last bit)
    k = _norm_rope(x[:, Hq:Hq + Hkv].double(), s["kw"].double(), cos.double(), sin.double())
    at = (s["page_ids"].long(), slice(None), s["slots"].long())
    s["k"][0][at], s["k"][1][at] = _pack(k)
    s["v"][0][at], s["v"][1][at] = _pack(x[:, Hq + Hkv:].float())
    return (q, *(_unpack(c[at], e[at]).to(x.dtype) for c, e in (s["k"], s["v"])))


def _visible(pages, context, L, ps, device):
    """[L, S]: the positions that the rows of a request see."""
    j = torch.arange(len(pages) * ps, device=device)
    i = torch.arange(L, device=device)[:, None]
    there = (pages >= 0).repeat_interleave(ps)
    return there & (j < context) & (j <= i + context - L)


def _attend(s, dtype):
    """softmax(q k^T / sqrt(D)) v of every request, in `dtype`."""
    Hq, Hkv, D = s["heads"]
    q, ps = s["q"], s["k"][0].shape[2]
    B, _, L, _ = q.shape
    out = torch.empty(q.shape, dtype=dtype, device=q.device)
    for b in range(B):
        pages = s["table"][b]
        seen = _visible(pages, s["lens"][b], L, ps, q.device)
        at = pages.clamp(min=0).long()
        # [Hkv, S, D]
        k, v = (_unpack(c[at], e[at], dtype).transpose(0, 1).reshape(Hkv, -1, D) for c, e in (s["k"], s["v"]))
        for h in range(Hkv):
            rows = q[b, h * (Hq // Hkv):(h + 1) * (Hq // Hkv)].to(dtype)
            w = (rows.reshape(-1, D) @ k[h].T).reshape(-1, L, k.shape[1]) * D ** -0.5
            w = torch.where(seen, w, -math.inf)
            # (rows that see nothing come out zero)
            top = w.amax(-1, keepdim=True)
            w = torch.exp(w - torch.where(top == -math.inf, torch.zeros_like(top), top))
            total = w.sum(-1, keepdim=True)
            o = (w.reshape(-1, w.shape[-1]) @ v[h]).reshape(rows.shape)
            out[b, h * (Hq // Hkv):(h + 1) * (Hq // Hkv)] = o / torch.where(total == 0, torch.ones_like(total), total)
    return out


def _logprobs(s):
    x, k = s["logits"].float(), s["k"]
    d = x - x.amax(-1, keepdim=True)
    e = torch.exp(d)
    # (long sums in 64 bits)
    z = e.sum(-1, dtype=torch.float64)
    lse = torch.log(z)
    given = d.gather(1, s["tokens"][:, None])[:, 0] - lse
    entropy = lse - (e * d).sum(-1, dtype=torch.float64) / z
    # the largest, k times: argmax gives the first of equals
    ids = torch.empty((len(x), k), dtype=torch.int64, device=x.device)
    top = torch.empty((len(x), k), dtype=torch.float32, device=x.device)
    for i in range(k):
        at = d.argmax(-1, keepdim=True)
        ids[:, i:i + 1] = at
        top[:, i:i + 1] = d.gather(1, at) - lse[:, None]
        d.scatter_(1, at, -math.inf)
    return given.float(), entropy.float(), ids, top


def _plain(s):
    if s["kind"] == "append":
        return _append(s)
    if s["kind"] == "logprobs":
        return _logprobs(s)
    return _attend(s, torch.float32).to(s["q"].dtype)


# ------------------------------------------------------------ the framework's


def _package():
    if "nano_vllm_metal_amd" in sys.modules:
        return sys.modules["nano_vllm_metal_amd"]
    at = str(Path(__file__).resolve().parent.parent / "nano-vllm-metal_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import nano_vllm_metal_amd

    return nano_vllm_metal_amd


def _pages(P, s, name):
    """The handle of a layer's keys or values, which a program keeps with the cache; it refers to the
    state's own tensors."""
    t = s.get("pages " + name)
    if t is None:
        t = s["pages " + name] = P.MxPages(*s[name])
    return t


def _own(s):
    P = _package()
    if s["kind"] == "logprobs":
        r = P.token_logprobs(s["logits"], s["tokens"], s["k"])
        return r.logprobs, r.entropy, r.top_ids, r.top_logprobs
    k, v = _pages(P, s, "k"), _pages(P, s, "v")
    if s["kind"] == "append":
        Hq, Hkv, D = s["heads"]
        q, _, _ = P.qk_norm_rope_store_mx(s["qkv"], Hq, Hkv, D, s["qw"], s["kw"], EPS, s["positions"], s["cos"],
                                          s["sin"], s["page_ids"], s["slots"], k, v)
        return (q, *P.paged_kv_read_mx(k, v, s["page_ids"], s["slots"], q.dtype))
    return P.paged_attention_mx(s["q"], k, v, s["table"], s["lens"], mask="causal")


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ inputs


def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, device=DEVICE, generator=g)


def _pool(g, P, Hkv, ps, D):
    """Pages of keys or values: dims of different sizes, a few of them much larger."""
    gain = torch.exp(0.3 * _randn(g, Hkv, 1, D))
    gain = torch.where(torch.rand(gain.shape, device=DEVICE, generator=g) < 0.02, 4.0 * gain, gain)
    codes = torch.empty((P, Hkv, ps, D // 2), dtype=torch.uint8, device=DEVICE)
    scales = torch.empty((P, Hkv, ps, D // BLOCK), dtype=torch.uint8, device=DEVICE)
    step = max(1, (1 << 26) // (Hkv * ps * D))
    for p in range(0, P, step):
        n = min(step, P - p)
        codes[p:p + n], scales[p:p + n] = _pack(_randn(g, n, Hkv, ps, D) * gain)
    return codes, scales


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    rng = random.Random(seed)
    dt = DTYPES[case["dtype"]]
    state = {"kind": kind}
    if kind == "logprobs":
        N, V = case["N"], case["V"]
        # rows from undecided to almost certain; of 16-bit logits many are equal
        x = _randn(g, N, V).mul_(2.5)
        sure = torch.randint(0, V, (N, 1), device=DEVICE, generator=g)
        x.scatter_add_(1, sure, 20 * torch.rand((N, 1), device=DEVICE, generator=g))
        other = torch.randint(0, V, (N, 1), device=DEVICE, generator=g)
        tokens = torch.where(torch.rand((N, 1), device=DEVICE, generator=g) < 0.7, sure, other)
        return state | {"logits": x.to(dt), "tokens": tokens[:, 0].contiguous(), "k": case["k"]}
    Hq, Hkv, D = state["heads"] = case["q"], case["kv"], case["D"]
    ps = case["page"]
    if kind == "append":
        T = case["T"]
        pages = -(-T // ps) + 2
        angles = torch.outer(torch.arange(MAX_POS, dtype=torch.float64),
                             THETA ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2)))
        first = rng.randrange(MAX_POS - T)
        # tokens of a prompt one behind the other, of a decode batch anywhere
        slot = torch.arange(T, device=DEVICE) if T > 64 else torch.randperm(pages * ps, device=DEVICE,
                                                                          generator=g)[:T]
        order = torch.randperm(pages, device=DEVICE, generator=g)
        at = torch.arange(T, device=DEVICE) + first if T > 64 else \
            torch.randint(0, MAX_POS, (T,), device=DEVICE, generator=g)
        return state | {
            "qkv": (_randn(g, T, (Hq + 2 * Hkv) * D) * torch.exp(0.3 * _randn(g, (Hq + 2 * Hkv) * D))).to(dt),
            "qw": (1 + 0.1 * _randn(g, D)).to(dt), "kw": (1 + 0.1 * _randn(g, D)).to(dt),
            "cos": torch.cos(angles).float().to(DEVICE), "sin": torch.sin(angles).float().to(DEVICE),
            "positions": at.int(), "page_ids": order[slot // ps].int(), "slots": (slot % ps).int(),
            "k": _pool(g, pages, Hkv, ps, D), "v": _pool(g, pages, Hkv, ps, D)}
    B, L = case["B"], case.get("L", 1)
    lens = _lens(case)
    rng.shuffle(lens)
    width = max(1, -(-case["ctx"] // ps))
    pages = B * width + 1
    table = torch.randperm(pages, device=DEVICE, generator=g)[:B * width].reshape(B, width).int()
    used = torch.tensor([[-(-n // ps)] for n in lens], device=DEVICE)
    table = torch.where(torch.arange(width, device=DEVICE) < used, table, -1)
    for _ in range(case.get("holes", 0)):
        table[rng.randrange(B), rng.randrange(width)] = -1
    # as the step before hands it on: token by token, heads side by side
    q = (1.5 * _randn(g, B, L, Hq, D)).to(dt).transpose(1, 2)
    return state | {"q": q, "k": _pool(g, pages, Hkv, ps, D), "v": _pool(g, pages, Hkv, ps, D),
                    "table": table.int(), "lens": torch.tensor(lens, dtype=torch.int32, device=DEVICE)}


# -------------------------------------------------------- what a pass needs


def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        N, V, k = case["N"], case["V"], case["k"]
        return {"bytes": float(N * V * SIZE[case["dtype"]] + N * (8 + 4 + 4 + 12 * k)), "flops": 6.0 * N * V}
    Hq, Hkv, D = case["q"], case["kv"], case["D"]
    row = 2 * Hkv * (D // 2 + D // BLOCK)  # a position's keys and values
    if kind == "append":
        T = case["T"]
        by = T * (2 * D * (Hq + 2 * Hkv) + 2 * D * Hq + 4 * D + 12) + T * row + T * row + T * 4 * D * Hkv
        return {"bytes": float(by), "flops": 12.0 * T * (Hq + Hkv) * D}
    L, lens = case.get("L", 1), _lens(case)
    pairs = sum(sum(max(0, i + n - L + 1) for i in range(L)) for n in lens)
    by = sum(lens) * row + len(lens) * L * Hq * D * 4
    return {"bytes": float(by), "flops": 4.0 * pairs * Hq * D}


# ------------------------------------------------------------ 64-bit results


def _grid():
    return torch.tensor(E2M1, dtype=torch.float64, device=DEVICE)


def _exact_quantized(x):
    """What x [..., n] (64 bits) is held as, by the nearest place of the grid of values."""
    g = x.reshape(*x.shape[:-1], -1, BLOCK)
    amax = g.abs().amax(-1).contiguous()
    scale = torch.exp2(((amax.view(torch.int64) >> 52) - 1025).clamp(-127, 127).double())
    a, middle = (g.abs() / scale[..., None]).contiguous(), (_grid()[1:] + _grid()[:-1]) / 2
    low, high = torch.bucketize(a, middle), torch.bucketize(a, middle, right=True)
    place = torch.where(low % 2 == 0, low, high)
    return (torch.copysign(_grid()[place], g) * scale[..., None]).reshape(x.shape)


def _exact_values(pages):
    codes, scales = pages
    c = torch.empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=torch.int64, device=DEVICE)
    c[..., 0::2], c[..., 1::2] = codes & 15, codes >> 4
    v = torch.where(c >= 8, -_grid()[c & 7], _grid()[c & 7])
    return v * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, dim=-1)


def _exact_rotated(x, w, cos, sin):
    y = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w
    half = x.shape[-1] // 2
    turned = torch.cat((-y[..., half:], y[..., :half]), -1)
    return y * torch.cat((cos, cos), -1) + turned * torch.cat((sin, sin), -1)


def _exact_attention(s):
    Hq, Hkv, D = s["heads"]
    ps, (B, _, L, _) = s["k"][0].shape[2], s["q"].shape
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(s["lens"].tolist()):
        j = torch.arange(n, device=DEVICE)
        page = s["table"][b].long()[j // ps]
        j, page = j[page >= 0], page[page >= 0]
        if len(j) == 0:
            continue
        hide = j[None, :] > torch.arange(L, device=DEVICE)[:, None] + n - L
        for h in range(Hq):
            kv = h // (Hq // Hkv)
            k, v = (_exact_values((c[page, kv, j % ps], e[page, kv, j % ps])) for c, e in (s["k"], s["v"]))
            w = s["q"][b, h].double() @ k.T / math.sqrt(D)
            p = torch.softmax(w.masked_fill(hide, -math.inf), -1)
            out[b, h] = torch.nan_to_num(p) @ v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "append":
        Hq, Hkv, D = s["heads"]
        q, k, v = s["qkv"].double().reshape(-1, Hq + 2 * Hkv, D).split((Hq, Hkv, Hkv), 1)
        cos, sin = (s[t][s["positions"].long()].double()[:, None] for t in ("cos", "sin"))
        return (_exact_rotated(q, s["qw"].double(), cos, sin),
                _exact_quantized(_exact_rotated(k, s["kw"].double(), cos, sin).contiguous()),
                _exact_quantized(v.contiguous()))
    if s["kind"] == "logprobs":
        parts = []
        for x, t in zip(s["logits"].split(256), s["tokens"].split(256)):
            d = torch.log_softmax(x.double(), -1)
            p = torch.exp(d)
            # by value, equal ones by their place
            order = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :s["k"]]
            parts.append((d.gather(1, t[:, None])[:, 0], -(p * d).sum(-1), order, d.gather(1, order)))
        return tuple(torch.cat(c) for c in zip(*parts))
    return _exact_attention(s)
