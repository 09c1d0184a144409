"""The raw pool of paged compressed caches over many evictions: what a budget bounds stays bounded.

No counterpart in the reference, whose caches keep every token (exactkv/cache.py)."""
import pytest
import torch

import exactkv_amd as exactkv
from tests.conftest import same_bits

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _rows(g, *shape):
    """Rows of which most are stored raw: exponents all over their range."""
    x = torch.randn(*shape, generator=g, device=DEV)
    return (x * torch.exp2(torch.randint(-40, 40, shape, generator=g, device=DEV).float())).bfloat16()


@pytest.mark.parametrize("layers", [1, 2])
def test_evictions_leave_no_raw_rows_behind(layers):
    """Two of three sequences generate 16 tokens and are cut to 32, forty times: at most 3 x 64 tokens of 2 heads are held at
    once, so a pool that keeps what is held and grows by the caches' rule (to twice its rows, or 5/4 of what it needs) stays
    below 8 x 384 rows; keeping every evicted row would take more than 40 x 2 x 32 x 2 = 5,120. The third one, which is
    not cut, and the kept rows stay bit for bit."""
    g = torch.Generator(device=DEV).manual_seed(layers)
    H, D = 2, 64
    table = exactkv.PageTable(20, 3, 4)
    pairs = [(exactkv.PagedCompressedKV(table, H, D=D), exactkv.PagedCompressedKV(table, H, D=D)) for _ in range(layers)]
    caches = [c for pair in pairs for c in pair]
    slots = [table.add(n) for n in (32, 50, 32)]
    held = []
    for c in caches:
        held.append([_rows(g, n, H, D) for n in (32, 50, 32)])
        for s, x in zip(slots, held[-1]):
            c.prefill(s, x[None])
    for turn in range(40):
        for _ in range(16):
            table.begin_step([slots[0], slots[2]])
            for c, rows in zip(caches, held):
                x = _rows(g, 2, H, D)
                c.append(x)
                for i, r in enumerate((0, 2)):
                    rows[r] = torch.cat([rows[r], x[i:i + 1]])
            exactkv.check_overflow(caches)
        mass = [torch.rand(3, H, 64, generator=g, device=DEV) for _ in pairs]
        index = exactkv.evict([p[0] for p in pairs], [p[1] for p in pairs], mass, 32, slots=[slots[2], slots[0]])
        for i, rows in enumerate(held):
            for at, r in ((0, 2), (1, 0)):
                rows[r] = rows[r].gather(0, index[i // 2][at].long().t()[..., None].expand(-1, -1, D))
        if turn % 8 == 7:
            for c, rows in zip(caches, held):
                for s, x in zip(slots, rows):
                    at = torch.arange(x.shape[0], dtype=torch.int32, device=DEV).expand(1, H, -1).contiguous()
                    got = exactkv.gather_tokens(c, c, at, block_table=table.block_table[s:s + 1].contiguous())[0][0]
                    assert same_bits(got, x), (turn, s)
    for c in caches:
        assert int(c.cnt) <= c.cap < 8 * 3 * 64 * H, (int(c.cnt), c.cap)
