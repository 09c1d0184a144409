"""prompt_attention over values of bf16's whole range: a softmax's weights sum to 1, so finite values
give finite results whatever their size, in every instance of the kernel and with split keys.

Tolerance, per value: as in test_gpu_prompt (which see for the terms); a row that is computed again
keeps its weights in fp32 and stays within the same.

No counterpart in the reference (its prefill is the model's own forward pass, engine.py:42-49)."""
import math

import pytest
import torch

import exactkv_amd as exactkv
from tests.test_gpu_prompt import _check, _cu, _formula, _inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"
MAX = torch.finfo(torch.bfloat16).max

# (queries, keys, query heads, KV heads, window): whole prompts, a continued and a split one, a window, and at
# head dim 256 few and many row tiles
CALLS = [([70, 1, 200], [70, 1, 200], 8, 2, 0), ([130], [400], 4, 2, 50), ([30, 9], [2500, 1200], 8, 2, 0),
         ([1], [3000], 4, 4, 0), ([520], [520], 64, 64, 300)]


def _run(q, k, v, lens, keys, window):
    return exactkv.prompt_attention(q, k, v, _cu(lens), cu_seqlens_k=_cu(keys), window=window)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,keys,Hq,Hkv,window", CALLS, ids=lambda x: str(x)[:20])
@pytest.mark.parametrize("scale", [2.0 ** 88, 2.0 ** 112, 2.0 ** 119, 2.0 ** 121, 2.0 ** 126])
def test_large_values_of_either_sign(scale, lens, keys, Hq, Hkv, window, D):
    q, k, v = _inputs(lens, keys, Hq, Hkv, D, 61)
    v = (v.float() * scale).clamp(-MAX, MAX).bfloat16()
    print("[case]", scale, lens, keys, Hq, Hkv, window, D, flush=True)
    _check(_run(q, k, v, lens, keys, window), *_formula(q, k, v, lens, keys, window))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,keys,Hq,Hkv,window", CALLS, ids=lambda x: str(x)[:20])
@pytest.mark.parametrize("sign", [1, -1])
def test_the_largest_value_everywhere(sign, lens, keys, Hq, Hkv, window, D):
    """All values alike: so is every result, to fp32 (nothing rounds past the largest bf16)."""
    q, k, v = _inputs(lens, keys, Hq, Hkv, D, 62)
    v.fill_(sign * MAX)
    got = _run(q, k, v, lens, keys, window)
    assert (got == sign * MAX).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,keys,Hq,Hkv,window", CALLS, ids=lambda x: str(x)[:20])
def test_large_values_beside_bad_ones(lens, keys, Hq, Hkv, window, D):
    """Channel 5 of one key is infinite: the rows that see it have it there and are right elsewhere; the others
    do not take it."""
    q, k, v = _inputs(lens, keys, Hq, Hkv, D, 63)
    v = (v.float() * 2.0 ** 121).clamp(-MAX, MAX).bfloat16()
    want, mag = _formula(q, k, v, lens, keys, window)
    at = keys[0] - 1                                   # the first sequence's last key: its last query sees it
    v[at, 0, 5] = math.inf
    got = _run(q, k, v, lens, keys, window)
    rows = slice(lens[0] - 1, lens[0]), slice(0, Hq // Hkv), 5
    assert (got[rows] == math.inf).all()
    got[rows], want[rows] = 0, 0
    _check(got, want, mag)


def test_a_score_that_is_not_finite_stays_so():
    """Large values do not send a row of NaN scores through the second look to another answer."""
    q, k, v = _inputs([90], [90], 4, 2, 128, 64)
    v = (v.float() * 2.0 ** 121).clamp(-MAX, MAX).bfloat16()
    want, mag = _formula(q, k, v, [90], [90], 0)
    k[40, 1] = math.nan
    got = _run(q, k, v, [90], [90], 0)
    assert got[40:, 2:].isnan().all()
    _check(got[:40], want[:40], mag[:40])
    _check(got[:, :2], want[:, :2], mag[:, :2])
