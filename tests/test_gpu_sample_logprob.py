"""sample's log-probability where the drawn token is far less likely than the likeliest one.

Given the token, it is (l - M) / t - log S in 64 bits, S the sum of the weights that stay, rounded to fp32 once: half a step is
2^-24 of its size. S is off by at most 2^-44 a token that stays (its weight's rounding, or its weight where that is below
2^-44): 2^19 tokens and S >= 1 make that 2^-25. The place of a logit in bins of 2^(1/32) has 41 bits behind the point: 2^-42 ln
2 / 32, which with the fp64 functions' own errors is far below 2^-30.

No counterpart in the reference (greedy decoding, exactkv/engine.py:93-95)."""
import math

import pytest
import torch

import exactkv_amd as exactkv

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _check(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """Log-probabilities of the tokens that are drawn, from their logits in 64 bits; returns those."""
    token, lp = exactkv.sample(x, u, temperature=t, top_k=k, top_p=p, min_p=m, logprob=True)
    t = float(torch.tensor(t))                                                # (settings are fp32)
    z, at = torch.sort((x.double() - x.double().amax(-1, keepdim=True)) / t, dim=-1, descending=True, stable=True)
    w = torch.exp(z)
    n = (w >= m).sum(-1)
    if k:
        n = n.clamp(max=k)
    stays = torch.arange(x.shape[1], device=DEV) < n[:, None]
    w = torch.where(stays, w, 0.0)
    if p < 1:
        before = torch.cumsum(w, -1) - w
        w = torch.where(before < p * w.sum(-1, keepdim=True), w, 0.0)
    rank = (at == token[:, None]).long().argmax(-1, keepdim=True)
    assert (w.gather(1, rank) > 0).all()
    want = (z.gather(1, rank) - w.sum(-1, keepdim=True).log())[:, 0]
    err = (lp.double() - want).abs()
    assert (err <= 2.0 ** -24 * want.abs() + 2.0 ** -25 + 2.0 ** -30).all(), (lp.tolist(), want.tolist())
    return want


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("V,bits", [(8000, 22), (8000, 30), (50257, 26), (50257, 34), (128256, 30), (128256, 34), (128256, 38), (2 ** 19, 40)])
def test_tokens_under_a_peak(V, bits, dtype):
    """One logit 2^bits times as likely as each of a spread tail, and the largest u, which falls among that."""
    print("[case]", V, bits, dtype, flush=True)
    g = torch.Generator(device=DEV).manual_seed(bits)
    x = (torch.randn(5, V, generator=g, device=DEV) * 0.4).to(dtype)
    x[:, V // 3] = bits * math.log(2)
    u = torch.tensor([1 - 2.0 ** -24, 1 - 2.0 ** -23, 1 - 2.0 ** -22, 0.5, 1 - 2.0 ** -24], device=DEV)
    want = _check(x, u)
    assert float(want.min()) < -(bits - 4) * math.log(2)                      # the tail was drawn from
    _check(x, u, t=0.9)
    _check(x, u, k=V // 2)
    _check(x, u, k=2000)
    _check(x, u, p=1 - 2.0 ** -24)


def test_weights_at_the_end_of_their_range():
    """Log-probabilities down to the last weight that counts: tokens 2^-1 to 2^-43 as likely as the first, each drawn."""
    x = torch.full((43, 9000), -100.0, device=DEV)
    drawn = 0
    for b in range(43):
        x[b, 17] = 0.0
        x[b, 8001] = -(b + 1) * math.log(2)
    for u in (0.3, 0.9, 1 - 2.0 ** -10, 1 - 2.0 ** -24):
        drawn += int((_check(x, torch.full((43,), u, device=DEV)) < -0.7).sum())
    assert drawn > 30


@pytest.mark.parametrize("V", [3, 9000])
def test_a_certain_token(V):
    """Its log-probability is 0, with 0's own sign."""
    x = torch.full((2, V), -math.inf, device=DEV)
    x[:, V - 1] = 3.0
    token, lp = exactkv.sample(x, torch.tensor([0.0, 0.9], device=DEV), logprob=True)
    assert token.tolist() == [V - 1] * 2 and lp.tolist() == [0.0, 0.0] and not torch.signbit(lp).any()
