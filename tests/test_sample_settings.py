"""Settings that are no numbers of their type: refused as such, whatever they are.

No counterpart in the reference (greedy decoding, exactkv/engine.py:93-95)."""
import math

import pytest
import torch

import exactkv_amd as exactkv
from exactkv_amd.sampling import _setting

BAD = [("top_k", math.inf), ("top_k", -math.inf), ("top_k", math.nan), ("temperature", 10 ** 400), ("top_p", -10 ** 400)]


@pytest.mark.parametrize("name,v", BAD, ids=["inf", "-inf", "nan", "10^400", "-10^400"])
def test_refused(name, v):
    kind, dtype = (int, torch.int32) if name == "top_k" else (float, torch.float32)
    with pytest.raises(ValueError, match=name):
        _setting(v, 1, dtype, 0, name, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("name,v", BAD, ids=["inf", "-inf", "nan", "10^400", "-10^400"])
def test_refused_by_the_call(name, v):
    with pytest.raises(ValueError, match=name):
        exactkv.sample(torch.zeros(2, 5, device="cuda"), torch.zeros(2, device="cuda"), **{name: v})
