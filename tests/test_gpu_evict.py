"""select_tokens and gather_tokens against sorts and indexing in torch: exact, for whole numbers and stored values alike.

No counterpart in the reference, which keeps every token."""
import math

import pytest
import torch

import exactkv_amd as exactkv
from exactkv_amd import kernels
from tests.conftest import same_bits

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _expect(mass, n, keep, sinks, recent):
    """(index, kept) of one row [TS] on the CPU: a stable sort by value."""
    index, kept = torch.full((keep,), -1, dtype=torch.int32), torch.zeros(keep)
    m = mass[:n]
    if n <= keep:
        at = torch.arange(n)
    else:
        mid = m[sinks:n - recent]
        mid = torch.where(torch.isnan(mid), torch.tensor(-math.inf), mid).double()
        mid[torch.isnan(m[sinks:n - recent])] = -1e300     # behind -infinity
        mid = torch.where(mid == -math.inf, torch.tensor(-1e299, dtype=torch.float64), mid)
        best = torch.sort(mid, descending=True, stable=True).indices[: keep - sinks - recent] + sinks
        at = torch.cat([torch.arange(sinks), best.sort().values, torch.arange(n - recent, n)])
    index[: len(at)], kept[: len(at)] = at.int(), m[at]
    return index, kept


def _check(mass, lens, keep, sinks=0, recent=0, T=None):
    B, H, TS = mass.shape
    if T is None:
        index, kept = exactkv.select_tokens(mass, keep, lens=torch.tensor(lens, dtype=torch.int32, device=DEV), sinks=sinks, recent=recent)
    else:
        index, kept = exactkv.select_tokens(mass, keep, T, sinks=sinks, recent=recent)
        lens = [T] * B
    m = mass.cpu()
    for b in range(B):
        for h in range(H):
            wi, wk = _expect(m[b, h], lens[b], keep, sinks, recent)
            assert torch.equal(index[b, h].cpu(), wi), (b, h)
            assert torch.equal(torch.nan_to_num(kept[b, h].cpu(), -7.0), torch.nan_to_num(wk, -7.0)), (b, h)
    return index


SIZES = [1, 2, 15, 63, 64, 65, 1000, 1023, 1024, 1025, 4095, 4096, 4097, 8191, 8192, 8193, 16383, 16384, 16385, 40001]


@pytest.mark.parametrize("T", SIZES)
def test_sizes(T):
    print("[case]", T, flush=True)
    mass = torch.exp(2 * torch.randn(2, 3, T, generator=_gen(T), device=DEV))
    for keep in sorted({1, 2, T // 4, T // 2, T - 1, T, T + 3} - {0}):
        _check(mass, None, keep, T=T)
        _check(mass, None, keep, sinks=min(4, keep), recent=min(keep - min(4, keep), 10), T=T)
    _check(mass, None, T // 2 + 1, sinks=T // 2 + 1, T=T)                     # nothing between
    _check(mass, None, T // 2 + 1, recent=T // 2 + 1, T=T)


@pytest.mark.parametrize("TS", [100, 5000, 20000])
def test_ragged_batches(TS):
    mass = torch.rand(6, 2, TS, generator=_gen(TS), device=DEV)
    _check(mass, [0, 1, TS, TS // 2, 41, TS - 1], min(TS, 40), 4, 10)
    view = mass[:, :, 7:]                                                     # rows not 16-byte aligned, strided
    _check(view, [0, 1, TS - 7, 39, 40, 41], 40, 0, 0)
    _check(mass.transpose(0, 1).contiguous().transpose(0, 1), [5, 6, TS, 0, 1, 2], 7, 1, 1)


@pytest.mark.parametrize("T", [700, 9000, 20000])
def test_ties_and_odd_values(T):
    """Equal masses go by index; none, negative, infinite, NaN, subnormal and zeros of both signs are in order."""
    g = _gen(T)
    few = torch.randint(0, 3, (1, 2, T), generator=g, device=DEV).float()
    for keep in (1, T // 7, T // 2, T - 3):
        _check(few, None, keep, T=T)
        _check(torch.zeros_like(few), None, keep, min(2, keep), 0, T=T)
    odd = torch.randn(1, 2, T, generator=g, device=DEV)
    pick = torch.randint(0, 9, odd.shape, generator=g, device=DEV)
    for i, v in enumerate((0.0, -0.0, math.inf, -math.inf, math.nan, 1e-42, -1e-42)):
        odd[pick == i] = v
    for keep in (1, T // 9, T // 3, T - T // 9, T - 1):
        _check(odd, None, keep, T=T)
    _check(torch.full_like(odd, math.nan), None, T // 2, T=T)


def _caches(B, T, H, D, seed):
    """A compressed and a bf16 pair of the same tokens, with raw rows, and their rows."""
    g = _gen(seed)
    TS = -(-T // 16) * 16 + 16
    out = []
    xs = [torch.randn(B, T, H, D, generator=g, device=DEV).bfloat16() for _ in range(2)]
    for x in xs:
        x[:, 1::5, -1, 2] *= 2.0 ** -24
        x[:, ::9, 0, 1] = 0
        pair = exactkv.CompressedKV(B, TS, H, D), exactkv.BF16KV(B, TS, H, D)
        for c in pair:
            for b in range(B):
                c.prefill_slot(b, x[b:b + 1])
        out.append(pair)
    return xs, out


def _index(B, H, T, n, seed):
    g = _gen(seed)
    index = torch.randint(0, T, (B, H, n), generator=g, device=DEV, dtype=torch.int32)
    index[torch.rand(index.shape, generator=g, device=DEV) < 0.1] = -1
    return index


def _gathered(x, index):
    at = index.clamp(min=0).long().transpose(1, 2)[..., None].expand(-1, -1, -1, x.shape[-1])
    return x.gather(1, at).masked_fill((index < 0).transpose(1, 2)[..., None], 0)


@pytest.mark.parametrize("B,T,H,D,n", [(1, 1, 1, 64, 1), (1, 40, 8, 128, 17), (3, 333, 2, 64, 100), (2, 100, 3, 256, 33), (2, 1000, 8, 128, 1500), (1, 17, 5, 128, 1)])
def test_gather(B, T, H, D, n):
    print("[case]", B, T, H, D, n, flush=True)
    xs, (ks, vs) = _caches(B, T, H, D, T)
    index = _index(B, H, T, n, n)
    want = [_gathered(x, index) for x in xs]
    for k, v in list(zip(ks, vs)) + [(ks[0].buffers(), vs[0].buffers()), tuple(xs)]:
        got = exactkv.gather_tokens(k, v, index)
        assert all(same_bits(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("kind", ["compressed", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_gather_from_pages(kind, D):
    g = _gen(D)
    H, lens = 3, [5, 100, 33, 64]
    table = exactkv.PageTable(60, 6, 10)
    cls = exactkv.PagedCompressedKV if kind == "compressed" else exactkv.PagedBF16KV
    k, v = cls(table, H, D=D), cls(table, H, D=D)
    hole = table.add(50)
    xs = [[torch.randn(n, H, D, generator=g, device=DEV).bfloat16() for n in lens] for _ in "kv"]
    slots = [table.add(n) for n in lens]
    table.release(hole)
    for c, rows in ((k, xs[0]), (v, xs[1])):
        for s, x in zip(slots, rows):
            c.prefill(s, x[None])
    index = torch.cat([_index(1, H, n, 21, n) for n in lens])
    bt = table.block_table[torch.tensor(slots, device=DEV)].contiguous()
    pools = [c.buffers() if kind == "compressed" else c.buf for c in (k, v)]
    for got in (exactkv.gather_tokens(*pools, index, block_table=bt), exactkv.gather_tokens(k, v, index, block_table=bt)):
        for rows, out in zip(xs, got):
            for i, x in enumerate(rows):
                assert same_bits(out[i:i + 1], _gathered(x[None], index[i:i + 1]))
    every = torch.full((6, H, 2), -1, dtype=torch.int32, device=DEV)          # a row for each slot
    every[slots[1]] = 7
    got = exactkv.gather_tokens(k, v, every)[0]
    assert same_bits(got[slots[1], 0], xs[0][1][7]) and got[slots[0]].abs().sum() == 0


def test_indexes_outside_the_cache_are_reported():
    xs, (ks, vs) = _caches(1, 40, 2, 128, 1)
    index = torch.tensor([[[0, 1000, -1], [-2, 5, 2 ** 31 - 1]]], dtype=torch.int32, device=DEV)
    for k, v in zip(ks, vs):
        out = exactkv.gather_tokens(k, v, index)[0]
        assert kernels.error_bits(clear=True) == 0x200
        assert same_bits(out[0, 0, 0], xs[0][0, 0, 0]) and same_bits(out[0, 1, 1], xs[0][0, 5, 1])
        assert out[0, 1:, 0].abs().sum() == 0 and out[0, 0, 1].abs().sum() == 0


def test_selected_tokens_gathered_in_a_graph():
    """Selection and gathering as one captured step, on a second stream."""
    xs, (ks, vs) = _caches(2, 500, 4, 128, 2)
    mass = torch.rand(2, 4, 512, generator=_gen(1), device=DEV)
    lens = torch.tensor([500, 300], dtype=torch.int32, device=DEV)

    def step():
        index, kept = exactkv.select_tokens(mass, 100, lens=lens, sinks=4, recent=20)
        return index, kept, *exactkv.gather_tokens(ks[0], vs[0], index)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        mass.copy_(torch.rand(2, 4, 512, generator=_gen(i + 2), device=DEV))
        lens.copy_(torch.tensor([500 - i, 90 + 4 * i]))
        graph.replay()
        torch.cuda.synchronize()
        index = _check(mass, lens.tolist(), 100, 4, 20)
        assert torch.equal(out[0], index)
        for x, rows in zip(xs, out[2:]):
            assert same_bits(rows, _gathered(x, index))


def test_rows_of_no_tokens():
    for kw in (dict(T=0), dict(lens=torch.zeros(1, dtype=torch.int32, device="cuda"))):
        index, kept = exactkv.select_tokens(torch.zeros(2, 3, 0, device="cuda"), 4, **kw)
        assert (index == -1).all() and index.shape == (2, 3, 4) and (kept == 0).all()


def test_refusals():
    mass = torch.rand(2, 2, 50, device=DEV)
    for a, kw in (((mass.double(), 5, 50), {}), ((mass[0], 5, 50), {}), ((mass, 0, 50), {}), ((mass, 5, 51), {}), ((mass, 5), {}), ((mass, 5, 50), dict(sinks=6)),
                  ((mass, 5, 50), dict(sinks=3, recent=3)), ((mass, 5, 50), dict(recent=-1)), ((mass.transpose(1, 2), 5, 2), {}), ((mass.cpu(), 5, 50), {}),
                  ((mass, 5), dict(lens=torch.tensor([3, 4], device=DEV)))):
        with pytest.raises(ValueError):
            exactkv.select_tokens(*a, **kw)
    xs, (ks, vs) = _caches(2, 40, 2, 128, 3)
    index = torch.zeros(2, 2, 3, dtype=torch.int32, device=DEV)
    other = exactkv.CompressedKV(2, 64, 2, 64)
    for a, kw in (((ks[0], vs[1], index), {}), ((ks[0], other, index), {}), ((ks[0], vs[0], index.long()), {}), ((ks[0], vs[0], index[:, :1].contiguous()), {}),
                  ((ks[0], vs[0], index.cpu()), {}), ((ks[1], vs[1], index.expand(2, 2, 3)[..., ::2]), {}),
                  ((ks[0], vs[0], torch.zeros(3, 2, 1, dtype=torch.int32, device=DEV)), {}),
                  ((ks[0], vs[0], index), dict(block_table=torch.zeros(1, 3, dtype=torch.int32, device=DEV)))):
        with pytest.raises(ValueError):
            exactkv.gather_tokens(*a, **kw)
