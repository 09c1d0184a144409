"""attention_mass and prompt_mass against the definition in 64 bits: every kind of cache, head dims, head groups, lengths from
none and one token on, windows, ragged batches, split sequences, hidden keys that are not finite, strides, graphs.

Tolerance, per entry, relative to the weights that it sums: a score is a sum of D exact products in fp32, off by at most
(D + 4) 2^-24 of the sum A of their sizes (in log2 units, times log2(e) / sqrt(D)), A's largest over the row; a weight by
ln 2 times twice that (its own score, the row's sum), by 2^-20 for the exponential, the logarithm of the row's sum
(2^-22 (|s| + |lse|) <= 2^-22 2 A) and the rounding of their difference, and by n 2^-24 for sums of n <= keys + queries terms.

No counterpart in the reference, which keeps no weights."""
import math

import pytest
import torch

import exactkv_amd as exactkv
from exactkv_amd import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rows(g, *shape):
    x = torch.randn(*shape, generator=g, device=DEV) * torch.exp(0.5 * torch.randn(*shape[-2:], generator=g, device=DEV))
    return x.bfloat16()


def _weights(q, k, pos, window):
    """Weights [Hq, m, n] of queries q [m, Hq, D] standing at keys pos [m] over keys k [n, Hkv, D], and their relative bound."""
    m, Hq, D = q.shape
    n, Hkv, _ = k.shape
    qd = q.double().view(m, Hkv, Hq // Hkv, D).permute(1, 2, 0, 3)           # [Hkv, G, m, D]
    kd = torch.nan_to_num(k.double(), 0.0, 0.0, 0.0).permute(1, 2, 0).contiguous()[:, None]    # [Hkv, 1, D, n]
    z = torch.matmul(qd, kd) / math.sqrt(D)
    j = torch.arange(n, device=DEV)
    seen = j <= pos[:, None]
    if window:
        seen &= j > pos[:, None] - window
    size = torch.matmul(qd.abs(), kd.abs()) / math.sqrt(D) * math.log2(math.e)
    A = size.masked_fill(~seen, 0).amax(-1, keepdim=True)
    z = z.masked_fill(~seen, -math.inf)
    top = z.amax(-1, keepdim=True)
    w = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total == 0, 1.0, total)
    rel = 2 * math.log(2) * (D + 4) * 2.0 ** -24 * A + 2.0 ** -20 + 2.0 ** -21 * A + (n + m) * 2.0 ** -24
    return w.flatten(0, 1), (w * rel).flatten(0, 1)


def _want(q, ks, mass, lens, window, TS):
    """(entries [B, Hkv, TS], their bounds) from each sequence's keys ks[b] [n, Hkv, D]."""
    B, Hq, D = q.shape
    Hkv = ks[0].shape[1]
    out = torch.zeros(B, Hkv, TS, dtype=torch.float64, device=DEV) if mass is None else mass.double().clone()
    bound = torch.zeros_like(out)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        w, e = _weights(q[b:b + 1], ks[b][:n], torch.tensor([n - 1], device=DEV), window)
        out[b, :, :n] += w.view(Hkv, -1, n).sum(1)
        bound[b, :, :n] = e.view(Hkv, -1, n).sum(1) + 2.0 ** -24 * out[b, :, :n].abs()
    return out, bound


def _near(got, want, bound):
    err = (got.double() - want).abs() - bound
    assert (err <= 1e-37).all(), float(err.max())


SHAPES = [(1, 1, 32, 8, 128), (1, 2, 8, 8, 128), (2, 15, 32, 8, 64), (3, 16, 14, 2, 64), (1, 17, 16, 1, 256), (2, 33, 40, 1, 128),
          (2, 255, 28, 4, 128), (5, 997, 32, 8, 128), (2, 2047, 64, 4, 64), (1, 4099, 8, 1, 256), (3, 1024, 6, 3, 128), (1, 9000, 20, 1, 64)]


@pytest.mark.parametrize("B,T,Hq,Hkv,D", SHAPES)
def test_bf16_cache(B, T, Hq, Hkv, D):
    print("[case]", B, T, Hq, Hkv, D, flush=True)
    g = _gen(T)
    k, q = _rows(g, B, T, Hkv, D), torch.randn(B, Hq, D, generator=g, device=DEV).bfloat16()
    mass = torch.rand(B, Hkv, T, generator=g, device=DEV)
    for window in (0, 1, 100, T + 5):
        got = exactkv.attention_mass(q, k, T, mass=mass, window=window)
        _near(got, *_want(q, list(k), mass, [T] * B, window, T))
    got = exactkv.attention_mass(q, k, T)
    _near(got, *_want(q, list(k), None, [T] * B, 0, T))
    assert torch.equal(got, exactkv.attention_mass(q, k, T))                  # the same bits each time


@pytest.mark.parametrize("B,T,Hq,Hkv,D", SHAPES)
def test_cache_objects(B, T, Hq, Hkv, D):
    """Prefilled and appended caches of both kinds, raw rows among the pages, agree with each other and with the definition."""
    print("[case]", B, T, Hq, Hkv, D, flush=True)
    g = _gen(T + 1)
    TS = -(-(T + 1) // 16) * 16 + 32
    x, q = _rows(g, B, T, Hkv, D), torch.randn(B, Hq, D, generator=g, device=DEV).bfloat16()
    x[:, ::7, 0, 3] *= 2.0 ** -24                                             # rows that are stored raw
    c, f = exactkv.CompressedKV(B, TS, Hkv, D), exactkv.BF16KV(B, TS, Hkv, D)
    for cache in (c, f):
        for b in range(B):
            cache.prefill_slot(b, x[b:b + 1, : T - 1])
        cache.append(x[:, T - 1].contiguous())
    exactkv.check_overflow([c])
    mass = torch.rand(B, Hkv, TS, generator=g, device=DEV)
    for window in (0, 40):
        want = _want(q, list(x), mass, [T] * B, window, TS)
        for cache in (c, f, c.buffers()):
            kw = dict(T=T) if isinstance(cache, dict) else {}
            got = exactkv.attention_mass(q, cache, mass=mass, window=window, out=mass.clone(), **kw)
            _near(got, *want)
        new = exactkv.attention_mass(q, c, mass=mass, window=window)
        _near(new[..., :T], want[0][..., :T], want[1][..., :T])
        assert (new[..., T:] == 0).all()
        assert torch.equal(new[..., :T], got[..., :T])                        # both kinds, the same bits


@pytest.mark.parametrize("kind", ["compressed", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (14, 2, 64), (4, 2, 256)])
def test_pools_of_pages(kind, Hq, Hkv, D):
    lens = [1, 15, 16, 17, 500, 33, 1000]
    g = _gen(D)
    table = exactkv.PageTable(300, 8, 80)
    cls = exactkv.PagedCompressedKV if kind == "compressed" else exactkv.PagedBF16KV
    kc = cls(table, Hkv, D=D)
    xs = [_rows(g, n, Hkv, D) for n in lens]
    hole = table.add(100)                                                     # pages in no order
    slots = []
    for n, x in zip(lens, xs):
        slots.append(table.add(n - 1))
        kc.prefill(slots[-1], x[None, : n - 1].contiguous())
    table.release(hole)
    order = [slots[i] for i in (3, 0, 6, 1, 5, 2, 4)]
    table.begin_step(order)
    rows = [xs[slots.index(s)] for s in order]
    kc.append(torch.stack([x[-1] for x in rows]))
    exactkv.check_overflow([kc])
    q = torch.randn(7, Hq, D, generator=g, device=DEV).bfloat16()
    ns = [x.shape[0] for x in rows]
    mass = torch.rand(7, Hkv, table.capacity, generator=g, device=DEV)
    for window in (0, 50):
        want = _want(q, rows, mass, ns, window, table.capacity)
        _near(exactkv.attention_mass(q, kc, mass=mass, window=window, out=mass.clone()), *want)
        _, bt, ln = table.step_rows()
        pool = kc.buffers() if kind == "compressed" else kc.buf
        _near(exactkv.attention_mass(q, pool, mass=mass, lens=ln, block_table=bt.contiguous(), window=window, out=mass.clone()), *want)


def test_lens_on_the_device_and_none_at_all():
    g = _gen(3)
    B, TS, Hq, Hkv, D = 6, 700, 8, 2, 128
    k, q = _rows(g, B, TS, Hkv, D), torch.randn(B, Hq, D, generator=g, device=DEV).bfloat16()
    ns = [0, 1, 699, 700, 16, 350]
    lens = torch.tensor(ns, dtype=torch.int32, device=DEV)
    before = torch.rand(B, Hkv, TS, generator=g, device=DEV)
    out = before.clone()
    assert exactkv.attention_mass(q, k, mass=out, lens=lens, out=out) is out   # in place
    _near(out, *_want(q, list(k), before, ns, 0, TS))
    for b, n in enumerate(ns):
        assert torch.equal(out[b, :, n:], before[b, :, n:])                   # behind the tokens: as it was
    new = exactkv.attention_mass(q, k, lens=lens)
    assert all((new[b, :, n:] == 0).all() for b, n in enumerate(ns))
    one = torch.tensor([41], dtype=torch.int32, device=DEV)
    _near(exactkv.attention_mass(q, k, lens=one), *_want(q, list(k), None, [41] * B, 0, TS))


def test_rows_behind_a_sequence_that_are_not_finite():
    g = _gen(4)
    k, q = _rows(g, 2, 100, 2, 128), torch.randn(2, 8, 128, generator=g, device=DEV).bfloat16()
    k[:, 70:] = math.nan
    k[:, 80:] = math.inf
    k[0, :20] = math.nan
    lens = torch.tensor([70, 65], dtype=torch.int32, device=DEV)
    got = exactkv.attention_mass(q, k, lens=lens, window=40)
    _near(got, *_want(q, list(k), None, [70, 65], 40, 100))


def test_weights_add_up_and_a_nan_stays_in_its_head():
    g = _gen(5)
    k, q = _rows(g, 2, 300, 4, 128), torch.randn(2, 16, 128, generator=g, device=DEV).bfloat16()
    got = exactkv.attention_mass(q, k, 300)
    assert (got.sum(-1) - 4).abs().max() < 4 * 2.0 ** -14
    k[1, 5, 2, 0] = math.nan
    bad = exactkv.attention_mass(q, k, 300)
    assert torch.isnan(bad[1, 2]).all()
    bad[1, 2] = got[1, 2]
    assert torch.equal(bad, got)


def test_sharp_and_flat_scores():
    g = _gen(6)
    k, q = _rows(g, 1, 500, 2, 128), torch.randn(1, 4, 128, generator=g, device=DEV).bfloat16()
    for s in (30.0, 2.0 ** -20, 0.0):
        qs = (q * s).bfloat16()
        _near(exactkv.attention_mass(qs, k, 500), *_want(qs, list(k), None, [500], 0, 500))


def test_captured_with_a_device_length():
    g = _gen(7)
    B, TS, Hq, Hkv, D = 2, 640, 32, 8, 128
    c = exactkv.CompressedKV(B, TS, Hkv, D)
    x = _rows(g, B, TS, Hkv, D)
    for b in range(B):
        c.prefill_slot(b, x[b:b + 1, :600])
    q = torch.randn(B, Hq, D, generator=g, device=DEV).bfloat16()
    mass = torch.zeros(B, Hkv, TS, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        exactkv.attention_mass(q, c, lens=c.state[:1], mass=mass, out=mass)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        exactkv.attention_mass(q, c, lens=c.state[:1], mass=mass, out=mass)
    mass.zero_()
    want = torch.zeros_like(mass)
    for i in range(5):
        q.copy_(torch.randn(B, Hq, D, generator=g, device=DEV))
        c.append(x[:, 600 + i].contiguous())
        graph.replay()
        torch.cuda.synchronize()
        want = exactkv.attention_mass(q, c, mass=want)
        assert torch.equal(mass, want)


# ---------------------------------------------------------------- prompts

def _offsets(lens):
    return torch.tensor([0] + list(lens), device=DEV).cumsum(0).int()


def _check_prompt(q, k, lens, keys, window=0, last=0, tail=0):
    got = exactkv.prompt_mass(q, k, _offsets(lens), cu_seqlens_k=_offsets(keys), window=window, last=last)
    Hkv = k.shape[1]
    assert got.shape == (Hkv, k.shape[0]) and got.dtype == torch.float32
    a = b = 0
    for n, nk in zip(lens, keys):
        m = min(n, last) if last else n
        want = torch.zeros(Hkv, nk, dtype=torch.float64, device=DEV)
        bound = torch.zeros_like(want)
        for i in range(0, m, 1024):
            r = min(1024, m - i)
            at = a + n - m + i
            pos = nk - m + i + torch.arange(r, device=DEV)
            w, e = _weights(q[at:at + r], k[b:b + nk], pos, window)
            want += w.view(Hkv, -1, nk).sum(1)
            bound += e.view(Hkv, -1, nk).sum(1) + want * 2.0 ** -24 * m
        _near(got[:, b:b + nk], want, bound)
        a, b = a + n, b + nk
    assert (got[:, b:] == 0).all()
    return got


def _prompt(g, N, NK, Hq, Hkv, D):
    return torch.randn(N, Hq, D, generator=g, device=DEV).bfloat16(), _rows(g, NK, Hkv, D)


LENGTHS = [([1], [1]), ([2], [2]), ([31], [31]), ([32], [32]), ([33], [33]), ([64], [64]), ([65], [65]), ([127, 1], [127, 1]), ([300], [300]),
           ([0, 70, 0, 1, 500, 0], [0, 70, 0, 1, 500, 0]), ([5, 0, 64], [1000, 100, 64]), ([300, 20], [100, 5]), ([1500], [1500]), ([1, 1], [2000, 7]),
           ([256, 255, 257], [256, 255, 257])]


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (7, 1, 64), (4, 4, 256), (3, 3, 64), (6, 2, 128)])
@pytest.mark.parametrize("lens,keys", LENGTHS, ids=str)
def test_prompts(lens, keys, Hq, Hkv, D):
    print("[case]", lens, keys, Hq, Hkv, D, flush=True)
    q, k = _prompt(_gen(sum(lens)), sum(lens), sum(keys), Hq, Hkv, D)
    for window, last in ((0, 0), (1, 0), (50, 0), (0, 1), (0, 70), (300, 33), (10 ** 6, 10 ** 6)):
        _check_prompt(q, k, lens, keys, window, last)


@pytest.mark.parametrize("lens,keys,last", [([2500], [2500], 0), ([700], [9000], 0), ([64], [16385], 0), ([512], [8192], 64), ([40] * 70, [40] * 70, 0),
                                            ([3] * 130, [90] * 130, 2)], ids=lambda v: str(v)[:24])
def test_larger_prompts(lens, keys, last):
    """Many tiles, tiles cut into parts, more sequences than a wavefront has lanes."""
    print("[case]", len(lens), keys[0], last, flush=True)
    q, k = _prompt(_gen(len(lens)), sum(lens), sum(keys), 8, 2, 128)
    got = _check_prompt(q, k, lens, keys, 0, last)
    assert torch.equal(got, exactkv.prompt_mass(q, k, _offsets(lens), cu_seqlens_k=_offsets(keys), last=last))
    _check_prompt(q, k, lens, keys, 700, last)


def test_rows_behind_the_last_sequence():
    g = _gen(11)
    q, k = _prompt(g, 500, 600, 8, 2, 128)
    _check_prompt(q, k, [100, 30], [110, 200])
    _check_prompt(q, k, [], [])
    assert exactkv.prompt_mass(q[:0], k, _offsets([0]), cu_seqlens_k=_offsets([600])).abs().sum() == 0


def test_hidden_keys_that_are_not_finite():
    """Keys that no query sees, or only later ones, give nothing to the others."""
    g = _gen(12)
    q, k = _prompt(g, 200, 200, 4, 2, 128)
    clean = exactkv.prompt_mass(q, k, _offsets([200]))
    k[150:] = math.nan
    w, e = _weights(q[:150], k[:150], torch.arange(150, device=DEV), 0)
    want, bound = w.view(2, -1, 150).sum(1), e.view(2, -1, 150).sum(1)
    for got in (exactkv.prompt_mass(q[:150], k[:150], _offsets([150])), exactkv.prompt_mass(q, k, _offsets([150, 50]))):
        _near(got[:, :150], want, bound + want * 2.0 ** -24 * 150)
    assert torch.isnan(got[:, 150:]).all()
    k2 = k.clone()
    k2[:150] = k[:150]
    seen = exactkv.prompt_mass(q, k2, _offsets([200]), window=30)
    assert torch.isfinite(seen[:, :121]).all() and torch.isnan(seen[:, 150:]).all()
    assert torch.isfinite(clean).all()


def test_scores_far_apart():
    """Rows whose first tile holds scores far below later ones: their sums leave fp32 and are made again."""
    g = _gen(13)
    q, k = _prompt(g, 400, 400, 4, 2, 128)
    q = (q.float() * 40).bfloat16()
    k[:100] *= -1
    k = (k.float() * torch.linspace(0.1, 4, 400, device=DEV)[:, None, None]).bfloat16()
    _check_prompt(q, k, [400], [400])
    _check_prompt(q, k, [150, 250], [150, 250], window=77)
    z = torch.zeros_like(q)
    _check_prompt(z, k, [400], [400])


@pytest.mark.parametrize("scale", [0, 7, 14, 20, 40])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_equal_keys_share_alike_whatever_their_scores(D, scale):
    """Keys that are all one row have one score each, up to about 2^(2 scale + 7) here; each row's weights are equal and
    add up to 1. An entry sums up to n weights 1 / k that are off by the sums they were divided by (n 2^-24) and a few roundings."""
    g = _gen(16)
    n, Hq, Hkv = 300, 6, 2
    q = (torch.randn(n, Hq, D, generator=g, device=DEV) * 2.0 ** scale).bfloat16()
    row = (torch.randn(1, Hkv, D, generator=g, device=DEV) * 2.0 ** scale).bfloat16()
    k = row.expand(n, Hkv, D).contiguous()
    share = 3.0 / torch.arange(1, n + 1, dtype=torch.float64, device=DEV)
    rel = 2 * n * 2.0 ** -24 + 2.0 ** -20
    want = share.flip(0).cumsum(0).flip(0).expand(Hkv, n)
    _near(exactkv.prompt_mass(q, k, _offsets([n])), want, want * rel)
    _near(exactkv.prompt_mass(q[:40].contiguous(), k, _offsets([40]), cu_seqlens_k=_offsets([n]), last=1),
          share[-1].expand(Hkv, n), share[-1] * rel)
    _near(exactkv.attention_mass(q[:1], k[None], n), share[-1].expand(1, Hkv, n), share[-1] * rel)


@pytest.mark.parametrize("scale", [10, 30, 55])
def test_weights_add_up_to_one_whatever_the_scores(scale):
    """Scores of any size, split keys and not: every row's weights add up to 1 (to the n 2^-24 of its sum and of the
    entries', and the exponentials' 2^-22), and none is negative."""
    g = _gen(17)
    for n, nk, last in ((500, 500, 0), (64, 4000, 0), (700, 700, 33)):
        q, k = _prompt(g, n, nk, 8, 2, 128)
        q, k = (q.float() * 2.0 ** scale).bfloat16(), (k.float() * 2.0 ** scale).bfloat16()
        got = exactkv.prompt_mass(q, k, _offsets([n]), cu_seqlens_k=_offsets([nk]), last=last)
        rows = 4 * (last or n)
        assert (got >= 0).all() and (got.double().sum(-1) - rows).abs().max() < rows * 2 * (nk + rows) * 2.0 ** -24
        got = exactkv.attention_mass(q[:1], k[None], nk)
        assert (got >= 0).all() and (got.double().sum(-1) - 4).abs().max() < 8 * nk * 2.0 ** -24


def test_strided_views_and_streams():
    g = _gen(14)
    Hq, Hkv, D, N = 8, 2, 128, 333
    x = torch.randn(N, (Hq + 2 * Hkv) * D, generator=g, device=DEV).bfloat16()
    q, k = x[:, : Hq * D].view(N, Hq, D), x[:, Hq * D:(Hq + Hkv) * D].view(N, Hkv, D)
    want = exactkv.prompt_mass(q.contiguous(), k.contiguous(), _offsets([333]))
    assert torch.equal(exactkv.prompt_mass(q, k, _offsets([333])), want)
    heads = q.transpose(0, 1).contiguous().transpose(0, 1)                    # [1, H, N, D] seen as rows
    assert torch.equal(exactkv.prompt_mass(heads, k, _offsets([333])), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = exactkv.prompt_mass(q, k, _offsets([333]))
    s.synchronize()
    assert torch.equal(got, want)


def test_prompt_mass_is_the_sum_of_its_tokens():
    """The steps' attention_mass over a growing cache, added up."""
    g = _gen(15)
    q, k = _prompt(g, 40, 40, 8, 2, 128)
    mass = torch.zeros(1, 2, 40, device=DEV)
    for n in range(1, 41):
        exactkv.attention_mass(q[n - 1:n].contiguous(), k[None].contiguous(), n, mass=mass, out=mass)
    assert (exactkv.prompt_mass(q, k, _offsets([40])) - mass[0]).abs().max() < 40 * 4 * 2.0 ** -18


def test_captured_prompt_follows_its_offsets():
    g = _gen(16)
    q, k = _prompt(g, 600, 600, 8, 2, 128)
    cu = _offsets([200, 400])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        exactkv.prompt_mass(q, k, cu, last=100)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = exactkv.prompt_mass(q, k, cu, last=100)
    for lens in ([200, 400], [600, 0], [1, 599], [50, 300]):
        cu.copy_(_offsets(lens))
        q.copy_(torch.randn(q.shape, generator=g, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, exactkv.prompt_mass(q, k, cu, last=100))
        _check_prompt(q, k, lens, lens, 0, 100)


def test_broken_offsets_are_reported():
    g = _gen(17)
    q, k = _prompt(g, 100, 100, 4, 2, 128)
    for cu in ([0, 120], [5, 100], [0, 60, 40]):
        exactkv.prompt_mass(q, k, torch.tensor(cu, dtype=torch.int32, device=DEV))
        assert kernels.error_bits(clear=True) == 0x20


def test_refusals():
    g = _gen(18)
    q, k = _prompt(g, 10, 10, 4, 2, 128)
    cu = _offsets([10])
    for a, kw in (((q.float(), k, cu), {}), ((q, k[:, :, :64], cu), {}), ((q[:, :3], k, cu), {}), ((q, k, cu.long()), {}), ((q, k, cu.cpu()), {}),
                  ((q, k[:9], cu), {}), ((q, k, cu), dict(window=-1)), ((q, k, cu), dict(last=-1)), ((q, k, cu), dict(cu_seqlens_k=_offsets([4, 6]))),
                  ((q.cpu(), k, cu), {})):
        with pytest.raises(ValueError):
            exactkv.prompt_mass(*a, **kw)
    with pytest.raises(RuntimeError, match="16-byte"):
        exactkv.prompt_mass(q.flatten()[4:4 + 4 * 512].view(4, 4, 128), k[:4], _offsets([4]))
    t = _rows(g, 2, 32, 2, 128)
    q2 = torch.randn(2, 4, 128, device=DEV).bfloat16()
    m = torch.zeros(2, 2, 32, device=DEV)
    lens = torch.tensor([3, 4], dtype=torch.int32, device=DEV)
    for a, kw in (((q2, t), {}), ((q2, t, 33), {}), ((q2.float(), t, 3), {}), ((q2, t.float(), 3), {}), ((q2, t[:1], 3), {}), ((q2, t, 3), dict(mass=m[:1])),
                  ((q2, t, 3), dict(mass=m.double())), ((q2, t, 3), dict(out=m[..., :16])), ((q2, t, 3), dict(window=-2)), ((q2, t), dict(lens=lens.long())),
                  ((q2, t), dict(lens=lens.cpu())), ((q2[:, :3], t, 3), {}), ((q2, t, 3), dict(mass=m.cpu())),
                  ((q2, t), dict(lens=lens, block_table=torch.zeros(1, 2, dtype=torch.int32, device=DEV)))):
        with pytest.raises(ValueError):
            exactkv.attention_mass(*a, **kw)
    both = torch.zeros(2 * 2 * 32 + 64, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        exactkv.attention_mass(q2, t, 3, mass=both[:128].view(2, 2, 32), out=both[64:192].view(2, 2, 32))
