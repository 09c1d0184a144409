"""attention_mass's workspace: by the tokens that a call has, not by what its cache could hold.

No counterpart in the reference, which keeps no weights."""
import pytest
import torch

import exactkv_amd as exactkv
from exactkv_amd import _lib


@pytest.mark.parametrize("B,Hq,Hkv,T", [(1, 32, 8, 1), (1, 32, 8, 0), (64, 32, 8, 1000), (3, 14, 2, 131072)])
def test_a_short_call_over_a_long_cache(B, Hq, Hkv, T):
    """Scores of the tokens, rounded up to a page, and 256 partial sums a query head at most."""
    need = _lib.load().exkv_mass_workspace(B, Hq, Hkv, T, 131072, 0, 0)
    assert 0 < need <= B * Hq * (4 * (T + 15) + 8 * 256)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 16, 1000, 4096])
def test_a_short_call_takes_little(T):
    """And gives what the call on a cache of its own length gives."""
    g = torch.Generator(device="cuda").manual_seed(T)
    B, TS, Hq, Hkv, D = 8, 16384, 32, 2, 64
    k = torch.randn(B, TS, Hkv, D, generator=g, device="cuda").bfloat16()
    q = torch.randn(B, Hq, D, generator=g, device="cuda").bfloat16()
    out = torch.zeros(B, Hkv, TS, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    exactkv.attention_mass(q, k, T, out=out)
    # (torch's allocator rounds up to 512 bytes, and hands out a block of its large pool whole where 2^20 bytes or less would remain of it;
    # the cache's capacity would be 2^24)
    assert torch.cuda.max_memory_allocated() - before <= B * Hq * (4 * (T + 15) + 8 * 256) + 512 + 2 ** 20
    assert torch.equal(out[..., :T], exactkv.attention_mass(q, k[:, :T].contiguous(), T)) and (out[..., T:] == 0).all()
    short = exactkv.attention_mass(q, k, lens=torch.tensor([T], dtype=torch.int32, device="cuda"))
    assert torch.allclose(short[..., :T], out[..., :T], rtol=1e-4, atol=1e-9)
