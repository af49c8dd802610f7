"""GPU tests of token_logprobs where the results are small: tokens that are all but
certain, by relative errors, and what log2 e as a float32 would take away.

With D the distance of the others to the largest logit (at most 21), r the sum of
their exp(-D), and u = 2^-24: log p = -log(1 + r) and the entropy is log(1 + r) + sum
exp(-D) D / (1 + r), sums of one sign.  A term's exponent is rounded where it is taken,
where its lane's maximum moves (by D in all) and where lanes and splits meet, and log2
e itself is off by u / 4: at most 6 u D.  exp2 is off by 2 u in each of the first, at
most 20 moves and 4 meetings, the float32 sum of eight terms by 7 u: 126 + 50 + 7, and
one rounding.  So 200 u of the result.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _exact(x):
    lp = torch.log_softmax(x.double(), -1)
    p = lp.exp()
    return lp, -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("V", [2, 9, 5003, 151936])
@pytest.mark.parametrize("high,low", [(29.0, 10.0), (18.75, 0.0), (-3.0, -23.0), (12.5, 4.0)])
def test_all_but_certain(high, low, V, dt):
    """One logit far above another one: in its vector, elsewhere in its lane, in another
    lane, wavefront and split; everything else at -infinity or e^-70 below."""
    from nano_vllm_metal_amd import token_logprobs

    for fill in (-float("inf"), high - 70.0):
        at = [(0, 1), (V - 1, 0)] + [(V // 2, (V // 2 + n) % V) for n in (1, 7, 64 * 8, 4096) if n < V // 2]
        x = torch.full((len(at), V), fill)
        for i, (a, b) in enumerate(at):
            x[i, a], x[i, b] = high, low
        x = x.to(dt)
        t = torch.tensor([a for a, _ in at])
        for n in (len(at), 1):  # (one row is split)
            lp, ent = _exact(x[:n])
            got = token_logprobs(x[:n].to(DEV), t[:n].to(DEV), 2)
            want = lp.gather(1, t[:n, None])[:, 0]
            assert (want < 0).all() and (want > -1e-3).all()
            u = 2.0 ** -24
            for a, b in ((got.logprobs, want), (got.entropy, ent), (got.top_logprobs[:, 0], want)):
                assert ((a.cpu().double() - b).abs() <= 200 * u * b.abs()).all()


def test_log_probabilities_have_no_temperature():
    """Log probabilities near -0.7 with half of the weight spread out (an entropy of
    6.4): each is rounded to 2^-25, and its other errors are as often above as below;
    the mean of 256 is to be off by less than 2^-25 (a standard error of 2^-29 and the
    systematic part of exp2's, at most u / 4).  A base off by 1.3e-8 of itself shifts
    all of them by 2^-23.5."""
    from nano_vllm_metal_amd import token_logprobs

    g = torch.Generator().manual_seed(1)
    x = 0.3 * torch.randn(256, 151936, generator=g)
    x[:, 77] = 11.95 + 0.1 * torch.rand(256, generator=g)
    t = torch.full((256,), 77)
    want = torch.cat([_exact(y)[0][:, 77] for y in x.split(32)])
    got = token_logprobs(x.to(DEV), t.to(DEV), 0).logprobs.cpu().double()
    assert abs(float((got - want).mean())) < 2.0 ** -25
