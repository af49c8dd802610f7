"""GPU tests of token_logprobs (include/nvm_logprobs.h) against 64-bit results.

Ids are exact: a stable descending sort of the logits.  With d = x - max and u =
2^-24, the exponent of a term is off by 3 u |d| (a difference, a product, and
log2 e itself; one fma x log2 e - m, m the largest so far, less), exp2 by one
unit (2 u) more; float32 sums of at most eight terms by 7 u.  So log Z is off by Z' = sum p (3 u |d| + 4 u) + 8 u, and the
entropy by that, by sum p |d| (3 u |d| + 8 u) and by sum p |d| (Z' + 8 u); each
result is rounded once (u of itself, and to infinity beyond float32's largest
value: the difference of that type's largest and lowest is 6.8e38).
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _check(x, tokens, k, got=None):
    """x [N, V] and tokens [N] on the CPU, rows with at least one finite logit and no +inf or NaN."""
    from nano_vllm_metal_amd import token_logprobs

    got = got or token_logprobs(x.to(DEV), tokens.to(DEV), k)
    V = x.shape[1]
    lp = torch.log_softmax(x.double(), -1)
    p = lp.exp()
    d = x.double() - x.double().amax(-1, keepdim=True)
    d = torch.where(p > 0, d.abs(), torch.zeros_like(d))
    u = 2.0 ** -24
    dz = (p * (3 * u * d + 4 * u)).sum(-1) + 8 * u
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    de = dz + (p * d * (3 * u * d + 8 * u)).sum(-1) + (p * d).sum(-1) * (dz + 8 * u)
    ok = (tokens >= 0) & (tokens < V)
    want = torch.where(ok, lp.gather(1, tokens.clamp(0, V - 1)[:, None])[:, 0], 0.0)
    a = got.logprobs.cpu().double()
    same = torch.isinf(want.float()) & (a == want.float())
    assert (same | ((a - want).abs() <= dz + u * want.abs())).all()
    assert ((got.entropy.cpu().double() - ent).abs() <= de + u * ent).all()
    order = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :k]
    assert got.top_ids.dtype == torch.int64 and torch.equal(got.top_ids.cpu(), order)
    t, w = got.top_logprobs.cpu().double(), lp.gather(1, order)
    same = torch.isinf(w.float()) & (t == w.float())
    assert (same | ((t - w).abs() <= dz[:, None] + u * w.abs())).all()
    return got


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("N,V,k", [
    (1, 151936, 5), (3, 50257, 20), (2, 151936, 0), (5, 1000, 64), (4, 65, 64), (7, 64, 64),
    (3, 1, 1), (2, 2, 2), (33, 777, 1), (6, 8191, 3), (1, 262144, 33), (130, 5003, 7), (300, 129, 2),
    (40, 33000, 20), (9, 2048, 3), (9, 8192, 3), (5, 4089, 2), (17, 1025, 5),
])
def test_shapes(dt, N, V, k):
    """Odd vocabularies: rows at every alignment (the first at that of the
    tensor, others where they fall)."""
    g = torch.Generator().manual_seed(V + k)
    x = (3 * torch.randn(N, V, generator=g)).to(dt)
    x[:, V // 3] += 12 * torch.rand(N, generator=g).to(dt)
    t = torch.randint(0, V, (N,), generator=g)
    t[0] = V // 3
    if N > 2:
        t[1], t[2] = -1, V
    got = _check(x, t, k)
    if N > 2:
        assert got.logprobs[1] == 0 and got.logprobs[2] == 0


@pytest.mark.parametrize("dt", TYPES)
def test_equal_logits(dt):
    """Constant rows, rows of two values, zeros of both signs: the lowest ids."""
    V = 40007
    g = torch.Generator().manual_seed(1)
    x = torch.zeros(5, V)
    x[1] = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0)
    x[2] = torch.randint(0, 2, (V,), generator=g).float()
    x[3] = torch.randint(0, 12, (V,), generator=g).float()
    x[4, 17::1000] = 1
    for k in (1, 20, 64):
        _check(x.to(dt), torch.arange(5) * 8000, k)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("k", [1, 20, 64])
def test_ordered_rows(dt, k):
    """Ascending, descending and a peak in the middle: every place of the
    largest, and lists that overflow again and again."""
    V = 70001
    up = torch.linspace(-40, 0, V)
    x = torch.stack((up, up.flip(0), torch.cat((up[::2], up[1::2].flip(0)))))
    _check(x.to(dt), torch.tensor([V - 1, 0, V // 2]), k)


@pytest.mark.parametrize("dt", TYPES)
def test_masked_rows(dt):
    """Masks of -infinity and of the type's lowest value: of all but one, of all
    but three (fewer than top_k), of the start and the end of a row; all at the
    lowest value."""
    V, k = 30011, 9
    g = torch.Generator().manual_seed(2)
    for fill in (-float("inf"), torch.finfo(dt).min):
        x = torch.randn(6, V, generator=g).to(dt)
        x[0, torch.arange(V) != 20000] = fill
        x[1, 3:] = fill
        x[2, :V - 3] = fill
        x[3, :15000] = fill
        x[4, 15000:] = fill
        t = torch.tensor([20000, 5, V - 1, 7, 7, 7])
        _check(x, t, k)
    _check(torch.full((2, V), torch.finfo(dt).min, dtype=dt), torch.tensor([0, V - 1]), k)
    # the largest values of the type, and a range that float32 differences overflow
    x = torch.randn(2, V, generator=g).to(dt)
    x[0, 99] = torch.finfo(dt).max
    x[1, 99], x[1, 100] = torch.finfo(dt).max, torch.finfo(dt).min
    _check(x, torch.tensor([99, 100]), k)


@pytest.mark.parametrize("dt", TYPES)
def test_sure_and_undecided_rows(dt):
    """A token of probability 1 - 1e-4 or so, one that nothing comes near, and
    a uniform row."""
    V = 151936
    x = torch.zeros(3, V)
    x[0, 1234], x[1, 1234] = 21.0, 400.0
    got = _check(x.to(dt), torch.tensor([1234, 1234, 7]), 2)
    # (with every d zero the bounds are 12 u)
    assert -12 * 2.0 ** -24 <= got.logprobs[1] <= 0 <= got.entropy[1] <= 12 * 2.0 ** -24
    assert abs(float(got.entropy[2]) - 11.9311) < 1e-3


@pytest.mark.parametrize("dt", TYPES)
def test_rows_without_probabilities(dt):
    """NaN or +infinity in a row, or nothing but -infinity: NaN, in that row
    only; the ids are still those of the largest, a NaN before all."""
    from nano_vllm_metal_amd import token_logprobs

    V = 5001
    x = torch.randn(5, V, generator=torch.Generator().manual_seed(3)).to(dt)
    clean = _check(x, torch.zeros(5, dtype=torch.int64), 4)
    x[0, 4000] = float("nan")
    x[1, 4001] = float("inf")
    x[2] = -float("inf")
    x[3, 17] = float("nan")
    t = torch.tensor([0, 0, 0, V, 0], device=DEV)
    got = token_logprobs(x.to(DEV), t, 4)
    assert got.logprobs[:3].isnan().all() and got.logprobs[3] == 0
    assert got.entropy[:4].isnan().all() and got.top_logprobs[:4].isnan().all()
    assert got.top_ids[0, 0] == 4000 and got.top_ids[1, 0] == 4001 and got.top_ids[3, 0] == 17
    assert got.top_ids[2].tolist() == [0, 1, 2, 3]
    assert got.logprobs[4] == clean.logprobs[4] and torch.equal(got.top_ids[4], clean.top_ids[4])


@pytest.mark.parametrize("dt", TYPES)
def test_strides_and_leading_dimensions(dt):
    from nano_vllm_metal_amd import token_logprobs

    g = torch.Generator().manual_seed(4)
    x = torch.randn(6, 999, generator=g).to(dt)
    t = torch.randint(0, 999, (6,), generator=g)
    want = _check(x, t, 5)
    wide = torch.full((6, 1203), float("nan"), dtype=dt, device=DEV)
    for at in (0, 1, 3, 204):
        wide.fill_(float("nan"))
        wide[:, at:at + 999] = x.to(DEV)
        _check(x, t, 5, token_logprobs(wide[:, at:at + 999], t.to(DEV), 5))
    got = token_logprobs(x.reshape(2, 3, 999).to(DEV), t.reshape(2, 3).int().to(DEV), 5)
    assert got.top_ids.shape == (2, 3, 5) and got.entropy.shape == (2, 3)
    for a, b in zip(got, want):
        assert torch.equal(a.reshape(b.shape), b)
    got = token_logprobs(x.to(DEV).t().contiguous().t(), t.to(DEV), 5)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    got = token_logprobs(x[0].to(DEV), t[0].to(DEV), 5)
    assert got.logprobs.shape == () and torch.equal(got.top_ids, want.top_ids[0])
    got = token_logprobs(x[:0].to(DEV), t[:0].to(DEV), 5)
    assert got.top_ids.shape == (0, 5) and got.logprobs.shape == (0,)
