"""add_norm over more rows than one grid holds.

No counterpart in the reference (the model's own modules do this, engine.py:75-91)."""
import pytest
import torch

import exactkv_amd as exactkv
from tests.conftest import same_bits

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("C,N", [(1, (1 << 26) + 70), (1, (1 << 27) + 5), (520, (1 << 25) + 3)])
def test_more_rows_than_a_grid_holds(C, N):
    """Rows behind a grid's last are as if they came alone: in the second launch, and the third."""
    g = torch.Generator(device=DEV).manual_seed(C)
    period = 4099                                      # rows repeat, so that the expected ones are few
    x, r, gate = (torch.randn(period, C, generator=g, device=DEV).bfloat16() for _ in range(3))
    w = torch.randn(C, generator=g, device=DEV).bfloat16()
    n = N // period * period

    def tile(t):
        whole = torch.empty(N, C, dtype=torch.bfloat16, device=DEV)
        whole[:n].view(-1, period, C).copy_(t)
        whole[n:].copy_(t[:N - n])
        return whole
    if C == 1:
        want = exactkv.add_norm(x, r, w, gate=gate, scale=0.5)
        got = exactkv.add_norm(tile(x), tile(r), w, gate=tile(gate), scale=0.5)
    else:                                              # 35 GB a tensor: as few as may be
        want = exactkv.add_norm(x, None, w, gate=gate[0], scale=0.5)
        got = exactkv.add_norm(tile(x), None, w, gate=gate[0], scale=0.5)
    for a, b in zip(got, want):
        for i in range(0, n, 1024 * period):
            rows = a[i:min(i + 1024 * period, n)].view(-1, period, C).view(torch.int16)
            assert (rows == b.view(torch.int16)).all()
        assert same_bits(a[n:], b[:N - n])


def test_rows_past_32_bits_are_refused():
    x = torch.ones(1, 1, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="rows"):
        exactkv.add_norm(x.expand((1 << 32) + 4, 1), None, x[0])
