"""The 4-bit KV cache in 64 bits, on torch tensors of the CPU — TEST
INFRASTRUCTURE ONLY.

``norm_rope`` is the step between the projections and the attention
(``models/qwen3.py:103-133`` without its roundings), ``attention`` paged
attention over what codes and scales stand for (``oracle/mx_oracle.py``), with
a bound on what float32 sums may be off.
"""

from __future__ import annotations

import torch

from oracle import mx_oracle as MX


def norm_rope(x, w, cos, sin, eps):
    """``x [T, H, D]``, ``w [D]``, ``cos, sin [T, D/2]`` -> float64 rows, and the
    sums of magnitudes that each value is the difference of."""
    x, w = x.double(), w.double()
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w
    half = x.shape[-1] // 2
    a, b = y[..., :half], y[..., half:]
    c, s = cos.double()[:, None], sin.double()[:, None]
    out = torch.cat((a * c - b * s, a * s + b * c), -1)
    size = torch.cat(((a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()), -1)
    return out, size


def weight_error(L, D, out_dtype):
    """What the weights are rounded by: two bf16 parts (2^-17 each, and their sum's
    own), for every number of rows, head dim and output."""
    return 2.0 ** -16


def attention(q, keys, values, table, lens, scale, causal, weights=2.0 ** -16):
    """``q [B, Hq, L, D]``, pages as (codes, scales) -> (float64 ``[B, Hq, L,
    D]``, bound): with n visible positions, scores s_j, largest value V of a
    column, and u = 2^-23 for a float32 addition in any order,
    a score is off by (D + 4) u sum |q k| scale and the exponent it goes into by
    u (|s_j| + |m|) log2 e more, so each weight by d of itself, twice exp's u among
    it; the quotient by 2 d + (2 n + 8) u of V; weights go into the product with
    a rounding of ``weights``, beside their sum without it."""
    kd, vd = (MX.decode(c, s, "mxfp4") for c, s in (keys, values))
    P, Hkv, ps, D = kd.shape
    B, Hq, L, _ = q.shape
    out = torch.zeros((B, Hq, L, D), dtype=torch.float64)
    bound = torch.zeros_like(out)
    u = 2.0 ** -23
    for b in range(B):
        n = min(int(lens[b]), table.shape[1] * ps)
        if n <= 0:
            continue
        j = torch.arange(n)
        page = table[b].long()[j // ps]
        ok = (page >= 0) & (page < P)
        j, page = j[ok], page[ok]
        if len(j) == 0:
            continue
        for h in range(Hq):
            k, v = (t[page, h // (Hq // Hkv), j % ps] for t in (kd, vd))
            x = q[b, h].double()
            s = x @ k.T * scale
            off = (D + 4) * u * abs(scale) * (x.abs() @ k.abs().T)
            seen = torch.ones_like(s, dtype=torch.bool)
            if causal:
                seen = j[None] <= torch.arange(L)[:, None] + int(lens[b]) - L
            for i in range(L):
                if not seen[i].any():
                    continue
                si, vi = s[i][seen[i]], v[seen[i]]
                m = si.max()
                p = torch.exp(si - m)
                d = off[i][seen[i]] + u * 1.45 * (si.abs() + m.abs()) + 4 * u
                # (an error of a weight that hardly counts hardly counts)
                d = float((p * torch.expm1(d)).sum() / p.sum())
                out[b, h, i] = p @ vi / p.sum()
                bound[b, h, i] = (2 * d + (2 * len(si) + 8) * u + weights) * vi.abs().amax(0)
    return out, bound


def random_pages(gen, P, Hkv, ps, D, spread=0.5):
    """(codes, scales) of normal values, dims of different sizes."""
    x = torch.randn(P, Hkv, ps, D, generator=gen, dtype=torch.float64)
    x = x * torch.exp(spread * torch.randn(Hkv, 1, D, generator=gen, dtype=torch.float64))
    c, b = MX.quantize(x, "mxfp4")
    return MX.pack(c, "mxfp4"), b.to(torch.uint8)
