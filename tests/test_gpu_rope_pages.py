"""rope_append_paged on tensors where a token fills its page: which pages' metadata it touches.

No counterpart in the reference (paged caches; the model's own modules rotate, engine.py:75-91)."""
import pytest
import torch

import exactkv_amd as exactkv
from exactkv_amd import kernels
from tests.conftest import same_bits
from tests.test_gpu_rope import _rows, _tables

pytestmark = pytest.mark.gpu
DEV = "cuda"
P, N, HQ, H, PAGES = 16, 3, 4, 2, 12


def _caches(D):
    """Two compressed caches over a pool of twelve pages, metadata and raw rows that no append would write."""
    t = exactkv.PageTable(PAGES, N, 3)
    pair = [exactkv.PagedCompressedKV(t, H, D) for _ in range(2)]
    for c in pair:
        c.rowmask.fill_(0x1234)
        c.rowoff.fill_(7)
        c.raw.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    return t, pair


def _meta(c):
    return c.rowmask.clone(), c.rowoff.clone()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("entry", [-1, PAGES, 2 ** 31 - 1, -2 ** 31])
def test_an_entry_outside_the_pool_opens_no_page(entry, D):
    """Slot 0 fills its first page; the next entry names none, and the pool's last page, which slot 1
    holds, keeps its metadata."""
    t, pair = _caches(D)
    g = torch.Generator(device=DEV).manual_seed(2)
    table = torch.tensor([[4, entry, 0], [PAGES - 1, 3, 0], [6, 2, 0]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([16, 5, 9], dtype=torch.int32, device=DEV)
    q, k, v = _rows(g, N, HQ, D), _rows(g, N, H, D), _rows(g, N, H, D)
    before = [_meta(c) for c in pair]
    cos, sin = _tables(64, D)
    exactkv.rope_append_paged(q, k, v, cos, sin, *(c._buf() for c in pair), lens, table)
    assert kernels.error_bits() == 0x80
    for c, (mask, off) in zip(pair, before):
        changed = (c.rowmask[0] != mask[0]).any(1) | (c.rowoff[0] != off[0]).any(1)
        assert changed.nonzero().view(-1).tolist() == [4]


@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_filled_page_touches_its_own_and_the_claimed_next(D):
    t, pair = _caches(D)
    g = torch.Generator(device=DEV).manual_seed(3)
    table = torch.tensor([[4, 8, 0], [PAGES - 1, 3, 0], [6, 2, 9]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([16, 5, 48], dtype=torch.int32, device=DEV)     # slot 2's last page of the table: none behind it
    q, k, v = _rows(g, N, HQ, D), _rows(g, N, H, D), _rows(g, N, H, D)
    before = [_meta(c) for c in pair]
    cos, sin = _tables(64, D)
    exactkv.rope_append_paged(q, k, v, cos, sin, *(c._buf() for c in pair), lens, table)
    assert kernels.error_bits() == 0
    for c, (mask, off) in zip(pair, before):
        changed = (c.rowmask[0] != mask[0]).any(1) | (c.rowoff[0] != off[0]).any(1)
        assert changed.nonzero().view(-1).tolist() == [4, 8, 9]
        assert (c.rowmask[0, 8] == 0xFFFF).all()
        assert c.rowoff[0, 8].tolist() == [c.cap, c.cap + P]


def test_a_slot_without_room_gets_its_query_row_and_nothing_else():
    D = 128
    t, pair = _caches(D)
    g = torch.Generator(device=DEV).manual_seed(4)
    table = torch.tensor([[4, 8, 0], [5, 3, 0], [6, 2, 9]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([0, 49, 3], dtype=torch.int32, device=DEV)
    q, k, v = _rows(g, N, HQ, D), _rows(g, N, H, D), _rows(g, N, H, D)
    before = [(_meta(c), c.raw.clone()) for c in pair]
    cos, sin = _tables(64, D)
    got = exactkv.rope_append_paged(q, k, v, cos, sin, *(c._buf() for c in pair), lens, table)
    assert kernels.error_bits() == 0x40
    assert same_bits(got[:2], q[:2])                   # position 0 turns by nothing
    for c, ((mask, off), raw) in zip(pair, before):
        assert torch.equal(c.rowmask, mask) and torch.equal(c.rowoff, off)
        same = (c.raw.view(torch.int16) == raw.view(torch.int16)).all(1)
        rows = (~same).nonzero().view(-1).tolist()
        assert rows == [c.cap + (2 * H + h) * P + 2 for h in range(H)]
