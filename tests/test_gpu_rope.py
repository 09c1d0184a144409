"""The rotation on the way into the caches: rotate_prompt against the formula in 64 bits, and
rope_append against the caches' own appends given the rotated keys, byte for byte, in every kind
of cache, over page ends, raw rows, pool growth, slot orders and graph replays.

Tolerance of a rotated value, per value: the store rounds by at most 2^-8 of it; the two products
and their difference by 2^-23 of |a c| + |b s|; with a norm, the sum of D squares (D 2^-24), the
reciprocal root (2^-22) and the products with it and the weight (2^-23): below 2^-15 for D <= 256,
of the normed |a c| + |b s|.

No counterpart in the reference (the model's own modules rotate, engine.py:75-91)."""
import pytest
import torch

import exactkv_amd as exactkv
from exactkv_amd import kernels, layer, synthetic
from tests.conftest import same_bits

pytestmark = pytest.mark.gpu
DEV = "cuda"
P = 16


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _rows(g, n, H, D):
    return (_randn(g, n, H, D) * torch.exp(_randn(g, H, D))).bfloat16()


def _tables(rows, D, theta=1e6):
    inv = theta ** (-torch.arange(D // 2, device=DEV, dtype=torch.float64) / (D // 2))
    ang = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _norms(g, D):
    return (1 + 0.2 * _randn(g, D)).bfloat16(), (1 + 0.2 * _randn(g, D)).bfloat16()


def _formula(x, cos, sin, pos, w=None, eps=1e-6):
    """(rotated rows, |a c| + |b s|) in 64 bits."""
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    a, b = x.chunk(2, dim=-1)
    mag = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1), mag


def _check(got, want, mag, normed):
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -15 if normed else 2.0 ** -22) * mag + 1e-37
    assert ((got.double() - want).abs() <= bound).all()


def _cu(lens):
    return torch.tensor([0] + list(lens), device=DEV).cumsum(0).int()


# ---------------------------------------------------------------- whole prompts

@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,Hq,Hkv", [([1], 1, 1), ([7, 0, 33, 1], 14, 2), ([100, 257], 32, 8), ([0, 0, 5], 5, 5),
                                         ([129], 40, 8)], ids=str)
def test_rotate_prompt(lens, Hq, Hkv, D, normed):
    g = torch.Generator(device=DEV).manual_seed(sum(lens) + Hq)
    N = sum(lens)
    q, k = _rows(g, N, Hq, D), _rows(g, N, Hkv, D)
    cos, sin = _tables(400, D)
    wq, wk = _norms(g, D) if normed else (None, None)
    print("[case]", lens, Hq, Hkv, D, normed, flush=True)
    qr, kr = exactkv.rotate_prompt(q, k, cos, sin, _cu(lens), q_norm=wq, k_norm=wk, eps=1e-5)
    pos = torch.cat([torch.arange(n, device=DEV) for n in lens])
    _check(qr, *_formula(q, cos, sin, pos, wq, 1e-5), normed)
    _check(kr, *_formula(k, cos, sin, pos, wk, 1e-5), normed)
    # from a later position on
    start = torch.randint(0, 140, (len(lens),), generator=g, device=DEV).int()
    qr, kr = exactkv.rotate_prompt(q, k, cos, sin, _cu(lens), start=start, q_norm=wq, k_norm=wk, eps=1e-5)
    pos = pos + torch.repeat_interleave(start.long(), torch.tensor(lens, device=DEV))
    _check(qr, *_formula(q, cos, sin, pos, wq, 1e-5), normed)
    _check(kr, *_formula(k, cos, sin, pos, wk, 1e-5), normed)


def test_rotate_prompt_strides_and_rows_behind():
    g = torch.Generator(device=DEV).manual_seed(1)
    N, Hq, Hkv, D = 50, 8, 2, 128
    q, k = _rows(g, N, Hq, D), _rows(g, N, Hkv, D)
    cos, sin = _tables(64, D)
    want = exactkv.rotate_prompt(q, k, cos, sin, _cu([30, 20]))
    for pad in (2, 6, 8):                              # rows 4-byte aligned, then 16
        wide = torch.zeros(N, (Hq + Hkv) * D + pad, dtype=torch.bfloat16, device=DEV)
        qv = wide[:, pad:pad + Hq * D].view(N, Hq, D)
        kv = wide[:, pad + Hq * D:].view(N, Hkv, D)
        qv.copy_(q)
        kv.copy_(k)
        got = exactkv.rotate_prompt(qv, kv, cos, sin, _cu([30, 20]))
        assert same_bits(got[0], want[0]) and same_bits(got[1], want[1])
    hq, hk = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k))
    got = exactkv.rotate_prompt(hq, hk, cos, sin, _cu([30, 20]))
    assert same_bits(got[0], want[0]) and same_bits(got[1], want[1])
    got = exactkv.rotate_prompt(q, k, cos, sin, _cu([30]))
    assert same_bits(got[0][:30], want[0][:30]) and (got[0][30:] == 0).all() and (got[1][30:] == 0).all()


def test_offsets_past_32_bits():
    """Rows so far apart that element offsets pass 2^31, whole prompts and appends."""
    n, pitch, Hq, Hkv, D = 300, 1 << 23, 4, 2, 128
    g = torch.Generator(device=DEV).manual_seed(21)
    q, k, v = _rows(g, n, Hq, D), _rows(g, n, Hkv, D), _rows(g, n, Hkv, D)
    cos, sin = _tables(n, D)
    wide = torch.empty(n * pitch, dtype=torch.bfloat16, device=DEV)
    far = [wide.as_strided(t.shape, (pitch, D, 1), at) for t, at in ((q, 0), (k, 4096), (v, 8192))]
    for dst, src in zip(far, (q, k, v)):
        dst.copy_(src)
    for a, b in zip(exactkv.rotate_prompt(far[0], far[1], cos, sin, _cu([n])), exactkv.rotate_prompt(q, k, cos, sin, _cu([n]))):
        assert same_bits(a, b)
    pair = [[exactkv.CompressedKV(n, 16, Hkv, D) for _ in range(2)] for _ in range(2)]
    assert same_bits(exactkv.rope_append(*far, cos, sin, *pair[0]), exactkv.rope_append(q, k, v, cos, sin, *pair[1]))
    for a, b in zip(*pair):
        _same_cache(a, b)


def test_positions_and_offsets_out_of_range_are_reported():
    g = torch.Generator(device=DEV).manual_seed(2)
    q, k = _rows(g, 40, 4, 128), _rows(g, 40, 2, 128)
    cos, sin = _tables(32, 128)
    got = exactkv.rotate_prompt(q, k, cos, sin, _cu([40]))
    assert kernels.error_bits() == 0x40
    fine = exactkv.rotate_prompt(q[:32], k[:32], cos, sin, _cu([32]))
    assert kernels.error_bits() == 0 and same_bits(got[0][:32], fine[0])
    exactkv.rotate_prompt(q, k, cos, sin, _cu([30]), start=torch.tensor([-3], dtype=torch.int32, device=DEV))
    assert kernels.error_bits() == 0x40
    exactkv.rotate_prompt(q, k, cos, sin, torch.tensor([2, 30], dtype=torch.int32, device=DEV))
    assert kernels.error_bits() & 0x20


# ---------------------------------------------------------------- decode steps, contiguous caches

def _same_cache(a, b):
    if isinstance(a, (exactkv.BF16KV, exactkv.PagedBF16KV)):
        assert same_bits(a.buf, b.buf)
        if isinstance(a, exactkv.BF16KV):
            assert a.T == b.T and torch.equal(a.state, b.state)
        return
    assert a.cap == b.cap and a.grows == b.grows and a._pending == b._pending
    for name in ("sm", "code", "base", "rowmask", "rowoff", "cnt", "_before"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    assert same_bits(a.raw, b.raw)
    if isinstance(a, exactkv.CompressedKV):
        assert a.T == b.T and torch.equal(a.state, b.state)
    else:
        assert torch.equal(a._arrivals, b._arrivals)


def _keys(B, T, H, D, seed, raw=0.05):
    return synthetic.make_kv(B, T, H, D, kind="v", seed=seed, raw_row_rate=raw, zero_rate=1e-3).to(DEV)


@pytest.mark.parametrize("kind", ["CompressedKV", "BF16KV"])
@pytest.mark.parametrize("B,Hq,Hkv,D,normed", [(1, 1, 1, 128, False), (3, 8, 2, 64, True), (2, 8, 1, 256, False),
                                               (9, 32, 8, 128, True), (70, 28, 4, 128, False), (200, 16, 8, 64, False)])
def test_rope_append_contiguous(kind, B, Hq, Hkv, D, normed):
    cls = getattr(exactkv, kind)
    T0, steps = 13, 22                                 # page ends at 16 and 32
    TS = 48
    g = torch.Generator(device=DEV).manual_seed(B)
    cos, sin = _tables(TS, D)
    wq, wk = _norms(g, D) if normed else (None, None)
    ks, vs = _keys(B, T0 + steps, Hkv, D, 2 * B), _keys(B, T0 + steps, Hkv, D, 2 * B + 1)
    print("[case]", kind, B, Hq, Hkv, D, normed, flush=True)
    mine, twin = [[cls(B, TS, Hkv, D) for _ in range(2)] for _ in range(2)]
    for pair in (mine, twin):
        for b in range(B):
            pair[0].prefill_slot(b, ks[b:b + 1, :T0])
            pair[1].prefill_slot(b, vs[b:b + 1, :T0])
    for t in range(T0, T0 + steps):
        q, k, v = _rows(g, B, Hq, D), ks[:, t], vs[:, t]
        got = exactkv.rope_append(q, k, v, cos, sin, *mine, q_norm=wq, k_norm=wk)
        pos = torch.full((B,), t, dtype=torch.int32, device=DEV)
        qr, kr = exactkv.rotate_prompt(q, k, cos, sin, _cu([1] * B), start=pos, q_norm=wq, k_norm=wk)
        assert same_bits(got, qr)
        twin[0].append(kr)
        twin[1].append(v)
        if (t + 1) % P == 0:
            assert exactkv.check_overflow(mine) == exactkv.check_overflow(twin)
        for a, b in zip(mine, twin):
            _same_cache(a, b)
    if kind == "CompressedKV" and B > 1:
        assert int(mine[0].cnt.item()) > 0             # raw rows were placed on the way
    o = exactkv.decode_attention(got, *mine)
    assert same_bits(o, exactkv.decode_attention(qr, *twin))


def test_rope_append_grows_a_full_pool():
    B, Hq, Hkv, D = 4, 8, 8, 128
    cos, sin = _tables(64, D)
    g = torch.Generator(device=DEV).manual_seed(3)
    pairs = [[exactkv.CompressedKV(B, 64, Hkv, D) for _ in range(2)] for _ in range(2)]
    for c in pairs[0] + pairs[1]:
        c.cap = 8                                      # room for 8 escaped rows, then the open pages
        c.raw = torch.zeros(8 + c._step_rows, D, dtype=torch.bfloat16, device=DEV)
        c._open_page()
    ks = _keys(B, 40, Hkv, D, 5, raw=0.4)
    for t in range(40):
        q = _rows(g, B, Hq, D)
        got = exactkv.rope_append(q, ks[:, t], ks[:, t], cos, sin, *pairs[0])
        pos = torch.full((B,), t, dtype=torch.int32, device=DEV)
        qr, kr = exactkv.rotate_prompt(q, ks[:, t], cos, sin, _cu([1] * B), start=pos)
        pairs[1][0].append(kr)
        pairs[1][1].append(ks[:, t])
        if (t + 1) % P == 0:
            assert exactkv.check_overflow(pairs[0]) == exactkv.check_overflow(pairs[1])
    assert pairs[0][0].grows > 0
    for a, b in zip(*pairs):
        _same_cache(a, b)


def test_a_full_contiguous_cache_is_refused():
    c = [exactkv.CompressedKV(1, 16, 2, 128) for _ in range(2)]
    cos, sin = _tables(16, 128)
    x = torch.ones(1, 2, 128, dtype=torch.bfloat16, device=DEV)
    for t in range(16):
        exactkv.rope_append(x, x, x, cos, sin, *c)
        if t == 15:
            with pytest.raises(AssertionError, match="check_overflow"):
                exactkv.rope_append(x, x, x, cos, sin, *c)
            exactkv.check_overflow(c)
    with pytest.raises(AssertionError, match="full"):
        exactkv.rope_append(x, x, x, cos, sin, *c)


@pytest.mark.parametrize("kind", ["CompressedKV", "BF16KV"])
@pytest.mark.parametrize("B", [2, 40])
def test_captured_steps(kind, B):
    """Captured appends and attention replayed over page ends, beside an eager twin."""
    Hq, Hkv, D, T0 = 8, 2, 128, 14
    cls = getattr(exactkv, kind)
    g = torch.Generator(device=DEV).manual_seed(7)
    cos, sin = _tables(64, D)
    ks, vs = _keys(B, 64, Hkv, D, 11), _keys(B, 64, Hkv, D, 12)
    mine, twin = [[cls(B, 64, Hkv, D) for _ in range(2)] for _ in range(2)]
    for pair in (mine, twin):
        for b in range(B):
            pair[0].prefill_slot(b, ks[b:b + 1, :T0])
            pair[1].prefill_slot(b, vs[b:b + 1, :T0])
    q, k, v = (torch.zeros(B, H, D, dtype=torch.bfloat16, device=DEV) for H in (Hq, Hkv, Hkv))

    def attend(qr, kc, vc):
        f = exactkv.attention_compressed if kind == "CompressedKV" else (
            lambda q, k, v, T, **kw: exactkv.attention_reference(q, k.buf, v.buf, T, **kw))
        return f(qr, kc, vc, 64, lens=kc.state[:1])

    def step():
        return attend(layer.launch_rope_append(q, k, v, cos, sin, *mine), *mine)
    stream, graph, out = torch.cuda.Stream(), None, None
    for t in range(T0, T0 + 21):
        q.copy_(_rows(g, B, Hq, D))
        k.copy_(ks[:, t])
        v.copy_(vs[:, t])
        torch.cuda.synchronize()
        if t == T0:                                    # eager once on the graph's stream: workspaces
            with torch.cuda.stream(stream):
                out = step()
        else:
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    out = step()
            graph.replay()
        torch.cuda.synchronize()
        for c in mine:
            c._advance()
        want = attend(exactkv.rope_append(q, k, v, cos, sin, *twin), *twin)
        assert same_bits(out, want), t
        if (t + 1) % P == 0:
            grown = exactkv.check_overflow(mine)
            assert grown == exactkv.check_overflow(twin)
            if grown:                                  # other buffers: captured again, as the engine does
                graph = None
        for a, b in zip(mine, twin):
            _same_cache(a, b)


# ---------------------------------------------------------------- decode steps, paged caches

@pytest.mark.parametrize("kind", ["PagedCompressedKV", "PagedBF16KV"])
@pytest.mark.parametrize("lens,Hq,Hkv,D,normed", [([5], 2, 1, 128, False), ([15, 1, 30, 14], 8, 2, 64, True),
                                                  ([40, 15, 16, 31, 2, 47], 28, 4, 128, True), ([15] * 40, 16, 8, 128, False),
                                                  (list(range(1, 90)), 8, 1, 256, False)], ids=lambda x: str(x)[:24])
def test_rope_append_paged(kind, lens, Hq, Hkv, D, normed):
    cls = getattr(exactkv, kind)
    n, steps = len(lens), 20
    g = torch.Generator(device=DEV).manual_seed(n)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(n)).tolist()
    max_pages = (max(lens) + steps) // P + 2
    num_pages = sum((L + steps) // P + 2 for L in lens)
    cos, sin = _tables(max(lens) + steps, D)
    wq, wk = _norms(g, D) if normed else (None, None)
    ks, vs = _keys(n, max(lens) + steps, Hkv, D, n), _keys(n, max(lens) + steps, Hkv, D, n + 1)
    print("[case]", kind, lens, Hq, Hkv, D, normed, flush=True)
    sides = []
    for _ in range(2):
        t = exactkv.PageTable(num_pages, n, max_pages)
        pair = [cls(t, Hkv, D) for _ in range(2)]
        for i in order:                                # slots' pages in no order
            s = t.add(lens[i], slot=i)
            pair[0].prefill(s, ks[i:i + 1, :lens[i]].contiguous())
            pair[1].prefill(s, vs[i:i + 1, :lens[i]].contiguous())
        sides.append((t, pair))
    (t1, mine), (t2, twin) = sides
    length = list(lens)
    for step in range(steps):
        # every slot; then some, in another order
        slots = list(range(n)) if step % 3 else [s for s in order if (s + step) % 2 or n == 1]
        t1.begin_step(slots)
        t2.begin_step(slots)
        at = [length[s] for s in slots]
        q = _rows(g, len(slots), Hq, D)
        k = torch.stack([ks[s, p] for s, p in zip(slots, at)])
        v = torch.stack([vs[s, p] for s, p in zip(slots, at)])
        got = exactkv.rope_append(q, k, v, cos, sin, *mine, q_norm=wq, k_norm=wk)
        pos = torch.tensor(at, dtype=torch.int32, device=DEV)
        qr, kr = exactkv.rotate_prompt(q, k, cos, sin, _cu([1] * len(slots)), start=pos, q_norm=wq, k_norm=wk)
        assert same_bits(got, qr)
        twin[0].append(kr)
        twin[1].append(v)
        for s in slots:
            length[s] += 1
        assert exactkv.check_overflow(mine) == exactkv.check_overflow(twin)
        for a, b in zip(mine, twin):
            _same_cache(a, b)
        assert same_bits(exactkv.decode_attention(got, *mine), exactkv.decode_attention(qr, *twin))


def test_a_slot_without_room_is_left_alone():
    """lens 0 or past the table: nothing is written for that row, the others' rows are."""
    n, Hkv, D = 3, 2, 128
    g = torch.Generator(device=DEV).manual_seed(9)
    cos, sin = _tables(64, D)
    q, k, v = _rows(g, n, 4, D), _rows(g, n, Hkv, D), _rows(g, n, Hkv, D)
    pools = [torch.full((1, 64, Hkv, D), 3.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    table = torch.tensor([[0, 1], [2, 3], [1, 0]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([0, 18, 33], dtype=torch.int32, device=DEV)
    exactkv.rope_append_paged(q, k, v, cos, sin, *pools, lens, table)
    bits = kernels.error_bits()
    assert bits == 0x40                                # no position for two of the rows
    qr, kr = exactkv.rotate_prompt(q[1:2], k[1:2], cos, sin, _cu([1]), start=lens[1:2] - 1)
    want = [torch.full_like(p, 3.0) for p in pools]
    want[0][0, 3 * P + 1] = kr[0]
    want[1][0, 3 * P + 1] = v[1]
    assert all(same_bits(a, b) for a, b in zip(pools, want))


def test_pages_out_of_the_pool_are_clamped():
    g = torch.Generator(device=DEV).manual_seed(10)
    cos, sin = _tables(64, 128)
    q, k, v = _rows(g, 2, 4, 128), _rows(g, 2, 2, 128), _rows(g, 2, 2, 128)
    pools = [torch.zeros(1, 32, 2, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    table = torch.tensor([[0, 7], [-1, 0]], dtype=torch.int32, device=DEV)
    exactkv.rope_append_paged(q, k, v, cos, sin, *pools, torch.tensor([17, 1], dtype=torch.int32, device=DEV), table)
    # both land in the last page's row 0, and nothing else changes
    for h in range(2):
        assert same_bits(pools[1][0, 16, h], v[0, h]) or same_bits(pools[1][0, 16, h], v[1, h])
    for p in pools:
        p[0, 16] = 0
        assert (p == 0).all()


def test_more_rows_than_one_list_of_fills():
    """More than 1,024 sequences, a page filled by some in each list."""
    n, Hkv, D = 1500, 1, 64
    g = torch.Generator(device=DEV).manual_seed(12)
    cos, sin = _tables(64, D)
    sides = []
    for _ in range(2):
        t = exactkv.PageTable(2 * n, n, 2)
        pair = [exactkv.PagedCompressedKV(t, Hkv, D) for _ in range(2)]
        for s in range(n):
            t.add(0)
        sides.append((t, pair))
    ks = _keys(n, 17, Hkv, D, 13, raw=0.1)
    for step in range(17):
        q = _rows(g, n, 2, D)
        for t, _ in sides:
            t.begin_step()
        k = ks[:, step].contiguous()
        got = exactkv.rope_append(q, k, k, cos, sin, *sides[0][1])
        pos = torch.full((n,), step, dtype=torch.int32, device=DEV)
        qr, kr = exactkv.rotate_prompt(q, k, cos, sin, _cu([1] * n), start=pos)
        assert same_bits(got, qr)
        sides[1][1][0].append(kr)
        sides[1][1][1].append(k)
        assert exactkv.check_overflow(sides[0][1]) == exactkv.check_overflow(sides[1][1])
    for a, b in zip(sides[0][1], sides[1][1]):
        _same_cache(a, b)


def test_unaligned_rows_and_views():
    B, Hq, Hkv, D = 3, 4, 2, 128
    g = torch.Generator(device=DEV).manual_seed(14)
    cos, sin = _tables(32, D)
    q, k, v = _rows(g, B, Hq, D), _rows(g, B, Hkv, D), _rows(g, B, Hkv, D)
    want = None
    for pad in (0, 2, 8):
        wide = torch.zeros(B, (Hq + 2 * Hkv) * D + pad, dtype=torch.bfloat16, device=DEV)
        wide[:, pad:] = torch.cat([q, k, v], dim=1).view(B, -1)
        h = wide[:, pad:].view(B, Hq + 2 * Hkv, D) if pad == 0 else wide[:, pad:].unflatten(1, (Hq + 2 * Hkv, D))
        c = [exactkv.CompressedKV(B, 32, Hkv, D) for _ in range(2)]
        got = exactkv.rope_append(h[:, :Hq], h[:, Hq:Hq + Hkv], h[:, Hq + Hkv:], cos, sin, *c)
        if want is None:
            want = got, c
        assert same_bits(got, want[0])
        for a, b in zip(c, want[1]):
            _same_cache(a, b)


@pytest.mark.parametrize("what", ["kinds", "one cache", "shape", "tokens", "table rows", "table type", "rows", "norm", "odd"])
def test_refusals(what):
    B, H, D = 2, 2, 128
    kc, vc = exactkv.CompressedKV(B, 32, H, D), exactkv.CompressedKV(B, 32, H, D)
    x = torch.ones(B, H, D, dtype=torch.bfloat16, device=DEV)
    q, k, v, (cos, sin), kw = x, x, x, _tables(32, D), {}
    if what == "kinds":
        vc = exactkv.BF16KV(B, 32, H, D)
    elif what == "one cache":
        vc = kc
    elif what == "shape":
        vc = exactkv.CompressedKV(B, 32, H, 64)
    elif what == "tokens":
        vc.append(x)
    elif what == "table rows":
        for _ in range(3):
            exactkv.rope_append(q, k, v, cos, sin, kc, vc)
        cos, sin = _tables(3, D)
    elif what == "table type":
        cos, sin = cos.bfloat16(), sin.bfloat16()
    elif what == "rows":
        q = torch.ones(B + 1, H, D, dtype=torch.bfloat16, device=DEV)
    elif what == "norm":
        kw["q_norm"] = torch.ones(64, dtype=torch.bfloat16, device=DEV)
    else:
        k = torch.ones(B * H * D + 2, dtype=torch.bfloat16, device=DEV)[1:-1].view(B, H, D)
    T = kc.T
    with pytest.raises((ValueError, TypeError, RuntimeError)):
        exactkv.rope_append(q, k, v, cos, sin, kc, vc, **kw)
    assert kc.T == T and int(kc.state[0]) == T
