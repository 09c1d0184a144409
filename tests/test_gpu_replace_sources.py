"""CompressedKV.replace from tensors whose rows lie anywhere: strides and addresses that are no whole number of words.

No counterpart in the reference, whose caches only grow."""
import pytest
import torch

import exactkv_amd as exactkv
from exactkv_amd import kernels
from tests.conftest import same_bits

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("n", [7, 16, 40])
@pytest.mark.parametrize("first", [0, 1])
def test_rows_at_odd_places(n, first):
    g = torch.Generator(device=DEV).manual_seed(n)
    c = exactkv.CompressedKV(2, 64, 2, 64)
    old = torch.randn(2, 50, 2, 64, generator=g, device=DEV).bfloat16()
    for b in range(2):
        c.prefill_slot(b, old[b:b + 1])
    x = torch.randn(2, n, 2, 65, generator=g, device=DEV).bfloat16()[..., first:first + 64]
    for y in (x, torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(x.shape)):    # (rows of 65, and whole ones behind one element)
        c.replace(y)
    assert c.T == n and int(c.state[0]) == n and same_bits(kernels.decode_to_bf16(c, n), x)
