"""Caches under a budget: replace, evict and the engines that run past their caches -- the operators together, as they are used.

  * evict leaves in each kind of cache exactly the rows that its index names, ready for appends and attention;
  * an Engine with a budget equals one without, bit for bit, until its first eviction; both caches agree throughout, and a
    captured step equals an eager one, over evictions;
  * a step after evictions equals the model in 64 bits over the kept keys at their true positions, to the roundings of a
    layer walk (about 14 a layer of 2^-8 each, two layers and the head: 30 x 2^-8 in the 2-norm);
  * engines draw their tokens with a Sampler.

No counterpart in the reference, whose caches end when they are full (exactkv/cache.py:102)."""
import math

import pytest
import torch

import exactkv_amd as exactkv
from exactkv_amd import kernels
from tests.conftest import same_bits
from tests.test_gpu_engine_layers import _ids, _model

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rows(g, *shape):
    x = torch.randn(*shape, generator=g, device=DEV).bfloat16()
    x[..., ::7, 0, 3] *= 2.0 ** -24
    return x


def _held(c, n):
    """The first n rows [B, n, H, D] of a contiguous cache."""
    return c.buf[:, :n] if isinstance(c, exactkv.BF16KV) else kernels.decode_to_bf16(c, max(n, 1))[:, :n]


@pytest.mark.parametrize("cls", [exactkv.CompressedKV, exactkv.BF16KV])
@pytest.mark.parametrize("B,H,D,T,n", [(1, 2, 128, 100, 0), (2, 3, 64, 100, 15), (3, 2, 128, 90, 64), (2, 8, 256, 112, 33), (1, 1, 128, 5, 112)])
def test_replace(cls, B, H, D, T, n):
    g = _gen(n)
    c = cls(B, 112, H, D)
    old, new = _rows(g, B, T, H, D), _rows(g, B, n, H, D)
    for b in range(B):
        c.prefill_slot(b, old[b:b + 1])
    c.replace(new)
    assert c.T == n and int(c.state[0]) == n and same_bits(_held(c, n), new)
    fresh = cls(B, 112, H, D)
    if cls is exactkv.CompressedKV and n:
        for b in range(B):
            fresh.prefill_slot(b, new[b:b + 1])
        assert int(c.cnt) == int(fresh.cnt)
        full = n // 16
        for name in ("sm", "code", "base", "rowmask", "rowoff"):
            per = 16 if name in ("sm", "code") else 1
            assert torch.equal(getattr(c, name)[:, : full * per], getattr(fresh, name)[:, : full * per]), name
    rows = [new[:, i] for i in range(n)]
    for i in range(min(20, 112 - n)):                                         # over a page end
        x = _rows(g, B, 8, H, D)[:, 1].contiguous()
        c.append(x)
        exactkv.check_overflow([c])
        rows.append(x)
    assert same_bits(_held(c, len(rows)), torch.stack(rows, 1))


def test_replace_grows_the_raw_pool_and_refuses():
    g = _gen(1)
    c = exactkv.CompressedKV(1, 320, 2, 128, reserve=0.0)
    x = torch.randn(1, 300, 2, 128, generator=g, device=DEV).bfloat16()
    x[:, :, :, 5] *= torch.where(torch.arange(300, device=DEV) % 2 == 0, 1.0, 2.0 ** -30)[None, :, None]     # most rows raw
    c.replace(x)
    assert c.grows > 0 and same_bits(_held(c, 300), x)
    for bad in (x[:, :, :1], x.float(), x.cpu(), x[..., ::2], x.expand(2, -1, -1, -1)):
        with pytest.raises(ValueError):
            c.replace(bad)
    with pytest.raises(AssertionError):
        c.replace(torch.zeros(1, 321, 2, 128, device=DEV, dtype=torch.bfloat16))


def _padded(x, TS):
    """Rows [B, n, H, D] with zeros behind them up to TS."""
    return torch.nn.functional.pad(x, (0, 0, 0, 0, 0, TS - x.shape[1])).contiguous()


def _gathered(x, index):
    at = index.clamp(min=0).long().transpose(1, 2)[..., None].expand(-1, -1, -1, x.shape[-1])
    return x.gather(1, at).masked_fill((index < 0).transpose(1, 2)[..., None], 0)


@pytest.mark.parametrize("cls", [exactkv.CompressedKV, exactkv.BF16KV])
@pytest.mark.parametrize("T,keep,sinks,recent", [(100, 40, 4, 10), (96, 32, 0, 0), (97, 96, 50, 46), (64, 64, 1, 1), (30, 64, 1, 1), (100, 1, 0, 1)])
def test_evict_contiguous(cls, T, keep, sinks, recent):
    g = _gen(T)
    B, H, D, Hq = 2, 4, 128, 8
    k, v = cls(B, 112, H, D), cls(B, 112, H, D)
    xs = [_rows(g, B, T, H, D) for _ in "kv"]
    for c, x in zip((k, v), xs):
        for b in range(B):
            c.prefill_slot(b, x[b:b + 1])
    mass = torch.rand(B, H, 112, generator=g, device=DEV)
    mass[..., T:] = 0
    want = exactkv.select_tokens(mass, keep, T, sinks=sinks, recent=recent)
    n = min(T, keep)
    before = mass.clone()
    index = exactkv.evict(k, v, mass, keep, sinks=sinks, recent=recent)
    assert torch.equal(index, want[0]) and k.T == v.T == n and int(k.state[0]) == n
    for c, x in zip((k, v), xs):
        assert same_bits(_held(c, n), _gathered(x, index[..., :n]))
    assert torch.equal(mass[..., :n], before.gather(2, index[..., :n].long())) and (mass[..., n:] == 0).all()
    step = [_rows(g, B, 8, H, D)[:, 1].contiguous() for _ in "kv"]
    for c, x in zip((k, v), step):
        c.append(x)
    exactkv.check_overflow([k, v])
    q = torch.randn(B, Hq, D, generator=g, device=DEV).bfloat16()
    plain = [_padded(torch.cat([_gathered(x, index[..., :n]), s[:, None]], 1), 112) for x, s in zip(xs, step)]
    assert same_bits(exactkv.decode_attention(q, k, v, nsplit=1, split_len=112), exactkv.attention_reference(q, *plain, n + 1, nsplit=1, split_len=112))
    exactkv.attention_mass(q, k, mass=mass, out=mass)
    exactkv.evict(k, v, mass, max(1, n // 2), recent=1)                        # again
    assert k.T == max(1, n // 2) or n + 1 <= max(1, n // 2)


@pytest.mark.parametrize("kind", ["compressed", "bf16"])
def test_evict_paged(kind):
    g = _gen(9)
    H, D, Hq, lens = 2, 128, 8, [100, 20, 50, 81]
    table = exactkv.PageTable(40, 5, 10)
    cls = exactkv.PagedCompressedKV if kind == "compressed" else exactkv.PagedBF16KV
    k, v = cls(table, H, D=D), cls(table, H, D=D)
    slots = [table.add(n) for n in lens]
    xs = [[_rows(g, n, H, D) for n in lens] for _ in "kv"]
    for c, rows in zip((k, v), xs):
        for s, x in zip(slots, rows):
            c.prefill(s, x[None])
    mass = torch.rand(5, H, 160, generator=g, device=DEV)
    free, before = table.free_pages(), mass.clone()
    index = exactkv.evict(k, v, mass, 32, sinks=2, recent=8, slots=[slots[3], slots[1], slots[0]])
    assert [table.length(s) for s in slots] == [32, 20, 50, 32] and table.free_pages() == free + 4 + 3
    assert table.lens[: len(slots)].tolist() == [32, 20, 50, 32]
    kept = {0: _gathered(xs[0][0][None], index[2:3])[0], 1: xs[0][1], 2: xs[0][2], 3: _gathered(xs[0][3][None], index[0:1])[0]}
    keptv = {0: _gathered(xs[1][0][None], index[2:3])[0], 1: xs[1][1], 2: xs[1][2], 3: _gathered(xs[1][3][None], index[0:1])[0]}
    assert torch.equal(mass[slots[2]], before[slots[2]]) and torch.equal(mass[slots[1]], before[slots[1]])
    assert torch.equal(mass[slots[0], :, :32], before[slots[0]].gather(1, index[2].long())) and (mass[slots[0], :, 32:] == 0).all()
    other = table.add(60)                                                     # the pages that came back serve others
    for c in (k, v):
        c.prefill(other, _rows(g, 1, 60, H, D))
    for i in range(20):
        order = [slots[2], slots[0], slots[3], slots[1]]
        table.begin_step(order)
        new = [_rows(g, 4, 8, H, D)[:, 1].contiguous() for _ in "kv"]
        k.append(new[0])
        v.append(new[1])
        exactkv.check_overflow([k, v])
        for r, s in enumerate((2, 0, 3, 1)):
            kept[s], keptv[s] = torch.cat([kept[s], new[0][r:r + 1]]), torch.cat([keptv[s], new[1][r:r + 1]])
        q = torch.randn(4, Hq, D, generator=g, device=DEV).bfloat16()
        out = exactkv.decode_attention(q, k, v, nsplit=1, split_len=160)
        for r, s in enumerate((2, 0, 3, 1)):
            want = exactkv.attention_reference(q[r:r + 1], _padded(kept[s][None], 160), _padded(keptv[s][None], 160), kept[s].shape[0], nsplit=1,
                                               split_len=160)
            assert same_bits(out[r:r + 1], want), (i, s)
    if kind == "compressed":
        k.compact()
        v.compact()
    assert exactkv.evict(k, v, mass, 150).shape == (5, H, 150)                 # all live slots; none is that long


def test_evict_refusals():
    k, v, b = exactkv.CompressedKV(1, 32, 2, 64), exactkv.CompressedKV(1, 32, 2, 64), exactkv.BF16KV(1, 32, 2, 64)
    mass = torch.zeros(1, 2, 32, device=DEV)
    for a, kw, err in (((k, b, mass, 4), {}, TypeError), ((k, k, mass, 4), {}, ValueError), ((k, v, mass[..., :16], 4), {}, ValueError),
                       ((k, v, mass, 0), {}, ValueError), ((k, v, mass, 4), dict(sinks=5), ValueError), ((k, v, mass, 4), dict(slots=[0]), ValueError),
                       ((k, v, mass.double(), 4), {}, ValueError), ((k, exactkv.CompressedKV(1, 48, 2, 64), mass, 4), {}, ValueError)):
        with pytest.raises(err):
            exactkv.evict(*a, **kw)
    x = torch.randn(1, 16, 2, 64, device=DEV).bfloat16()
    for c in (k, v):
        for i in range(16):
            c.append(x[:, i].contiguous())
    with pytest.raises(RuntimeError, match="check_overflow"):
        exactkv.evict(k, v, mass, 4)
    exactkv.check_overflow([k, v])
    exactkv.evict(k, v, mass, 4)
    t = exactkv.PageTable(8, 2, 4)
    pk, pv = exactkv.PagedCompressedKV(t, 2, D=64), exactkv.PagedCompressedKV(t, 2, D=64)
    m = torch.zeros(2, 2, 64, device=DEV)
    assert exactkv.evict(pk, pv, m, 2).shape == (0, 2, 2)                      # no sequence yet
    t.add(5)
    assert exactkv.evict(pk, pv, m, 2, slots=[]).shape == (0, 2, 2) and t.length(0) == 5
    for slots in ([1], [0, 0], [-1], [2]):
        with pytest.raises(ValueError):
            exactkv.evict(pk, pv, m, 2, slots=slots)


@pytest.mark.parametrize("kind", ["compressed", "bf16"])
def test_layers_of_one_table_are_cut_together(kind):
    """Two layers over one PageTable: one of them alone is refused and left as it was; both keep what their masses say."""
    g = _gen(10)
    H, D, lens = 2, 64, [70, 33, 8]
    table = exactkv.PageTable(24, 3, 8)
    cls = exactkv.PagedCompressedKV if kind == "compressed" else exactkv.PagedBF16KV
    layers = [(cls(table, H, D=D), cls(table, H, D=D)) for _ in range(2)]
    for n in lens:
        table.add(n)
    xs = [[[_rows(g, 1, n, 8, D)[:, :, :H].contiguous() for n in lens] for _ in "kv"] for _ in layers]
    for pair, rows in zip(layers, xs):
        for c, r in zip(pair, rows):
            for s, x in enumerate(r):
                c.prefill(s, x)
    mass = [torch.rand(3, H, 128, generator=g, device=DEV) for _ in layers]
    before = [m.clone() for m in mass]
    for bad in ((*layers[0], mass[0]), ([layers[0][0]], [layers[0][1]], mass[:1]), ([layers[0][0]] * 2, [p[1] for p in layers], mass),
                ([p[0] for p in layers], [p[1] for p in layers], mass[:1])):
        with pytest.raises(ValueError):
            exactkv.evict(*bad, 20)
    assert [table.length(s) for s in range(3)] == lens and all(torch.equal(m, b) for m, b in zip(mass, before))
    index = exactkv.evict([p[0] for p in layers], [p[1] for p in layers], mass, 20, recent=4)
    assert [table.length(s) for s in range(3)] == [20, 20, 8] and table.free_pages() == 24 - 2 - 2 - 1
    for pair, rows, at, m, b in zip(layers, xs, index, mass, before):
        assert torch.equal(at, exactkv.select_tokens(b, 20, lens=torch.tensor(lens, dtype=torch.int32, device=DEV), recent=4)[0])
        want = [_padded(torch.cat([_padded(_gathered(x, at[s:s + 1, :, : min(20, n)]), 20) for s, (n, x) in enumerate(zip(lens, r))]), 128) for r in rows]
        table.begin_step()
        table.truncate(0, 20), table.truncate(1, 20), table.truncate(2, 8)     # (lengths only, for the comparison)
        n = torch.tensor([20, 20, 8], dtype=torch.int32, device=DEV)
        q = torch.randn(3, 4, D, generator=g, device=DEV).bfloat16()
        kw = dict(lens=n, nsplit=1, split_len=128)
        if kind == "compressed":
            got = exactkv.attention_compressed(q, *pair, 0, block_table=table.block_table, **kw)
        else:
            got = exactkv.attention_reference(q, pair[0].buf, pair[1].buf, 0, block_table=table.block_table, **kw)
        assert same_bits(got, exactkv.attention_reference(q, *want, 0, **kw))
        for s, n in enumerate((20, 20, 8)):
            assert torch.equal(m[s, :, :n], b[s].gather(1, at[s, :, :n].long())) and (s == 2 or (m[s, :, n:] == 0).all())


def test_a_step_is_whole_before_an_eviction():
    table = exactkv.PageTable(8, 2, 4)
    k, v = exactkv.PagedBF16KV(table, 2, D=64), exactkv.PagedBF16KV(table, 2, D=64)
    g = _gen(12)
    table.add(30)
    for c in (k, v):
        c.prefill(0, _rows(g, 1, 30, 8, 64)[:, :, :2].contiguous())
    mass = torch.rand(2, 2, 64, generator=g, device=DEV)
    table.begin_step()
    k.append(_rows(g, 1, 2, 64))
    with pytest.raises(RuntimeError, match="step"):
        exactkv.evict(k, v, mass, 8)
    with pytest.raises(ValueError, match="lengths"):
        exactkv.attention_mass(_rows(g, 1, 4, 64), k, lens=table.lens[:1])
    v.append(_rows(g, 1, 2, 64))
    exactkv.evict(k, v, mass, 8)
    assert table.length(0) == 8


# ---------------------------------------------------------------- engines

KEEP = dict(sinks=3, recent=10)


def _run(eng, ids, T):
    out = [eng.step(ids[:, t]) for t in range(T, ids.shape[1])]
    return torch.stack(out, dim=1)


@pytest.mark.parametrize("kind", ["llama", "qwen3"])
def test_engine_past_its_caches(kind):
    """Teacher-forced steps over two evictions: equal to an engine without a budget before the first, the same bits from both
    caches and from captured and eager steps, and finite throughout."""
    m = _model(kind)
    B, T, N, room = 2, 40, 90, 64
    ids = _ids(B, T + N)
    full = exactkv.Engine(m, B, T + N, layer_kernels=True)
    first = full.prefill(ids[:, :T])
    want = _run(full, ids, T)
    got = {}
    for backend in ("exactkv", "bf16"):
        for graph in (True, False):
            eng = exactkv.Engine(m, B, room, backend=backend, graph=graph, layer_kernels=True, budget=exactkv.Budget(30, **KEEP))
            assert torch.equal(eng.prefill(ids[:, :T]), first)
            got[backend, graph] = _run(eng, ids, T)
            assert eng.dropped + eng.kv[0][0].T == T + N and eng.kv[0][0].T <= room and eng.dropped > 34
    base = got["exactkv", True]
    assert same_bits(base[:, : room - T], want[:, : room - T])
    assert all(same_bits(base, x) for x in got.values()) and torch.isfinite(base.float()).all()
    assert not torch.equal(base[:, room - T:], want[:, room - T:])             # fewer keys from there on


def _exact_step(m, eng, tok, position):
    """Logits of one step in 64 bits: the engine's cached rows (as bf16 holds them) and the token at `position`."""
    cfg, mm = m.config, m.model
    Hq, Hkv, D = cfg.num_attention_heads, cfg.num_key_value_heads, eng.D
    cos, sin = (t[position].double() for t in (eng._layers.cos, eng._layers.sin))

    def norm(x, mod):
        return x / (x.square().mean(-1, keepdim=True) + mod.variance_epsilon).sqrt() * mod.weight.double()

    def lin(x, mod):
        y = x @ mod.weight.double().t()
        return y if mod.bias is None else y + mod.bias.double()

    def turn(x):
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    h = mm.embed_tokens(tok).double()
    for layer, (kc, vc) in zip(mm.layers, eng.kv):
        att, x = layer.self_attn, norm(h, layer.input_layernorm)
        q, k, v = (lin(x, p).view(-1, n, D) for p, n in ((att.q_proj, Hq), (att.k_proj, Hkv), (att.v_proj, Hkv)))
        if eng.qk_norm:
            q, k = norm(q, att.q_norm), norm(k, att.k_norm)
        n = kc.T
        ks = torch.cat([_held(kc, n).double(), turn(k)[:, None]], 1).repeat_interleave(Hq // Hkv, 2)
        vs = torch.cat([_held(vc, n).double(), v[:, None]], 1).repeat_interleave(Hq // Hkv, 2)
        w = torch.softmax((turn(q)[:, None] * ks).sum(-1) / math.sqrt(D), 1)
        h = h + lin((w[..., None] * vs).sum(1).flatten(1), att.o_proj)
        x, mlp = norm(h, layer.post_attention_layernorm), layer.mlp
        h = h + lin(torch.nn.functional.silu(lin(x, mlp.gate_proj)) * lin(x, mlp.up_proj), mlp.down_proj)
    return lin(norm(h, mm.norm), m.lm_head)


@pytest.mark.parametrize("kind", ["llama", "qwen3"])
@pytest.mark.parametrize("T", [40, 150])
def test_steps_stand_at_their_positions(kind, T):
    """After a prompt that fits, and one longer than the caches, and over evictions: each step against 64 bits."""
    m = _model(kind)
    ids = _ids(3, T + 45)
    eng = exactkv.Engine(m, 3, 64, layer_kernels=True, budget=exactkv.Budget(40, **KEEP))
    eng.prefill(ids[:, :T])
    assert eng.kv[0][0].T == min(T, 40) and eng.dropped == max(0, T - 40)
    with torch.no_grad():
        for t in range(T, T + 45):
            eng._make_room()
            want = _exact_step(m, eng, ids[:, t], t)
            got = eng.step(ids[:, t])
            assert ((got.double() - want).norm() / want.norm()).item() < 30 * 2.0 ** -8, t


def test_prompt_longer_than_the_caches_keeps_what_its_weights_say():
    m = _model("llama")
    B, T, keep = 2, 200, 50
    ids = _ids(B, T)
    full = exactkv.Engine(m, B, T, layer_kernels=True)
    for backend in ("exactkv", "bf16"):
        eng = exactkv.Engine(m, B, 64, backend=backend, layer_kernels=True, budget=exactkv.Budget(keep, last=32, **KEEP))
        assert torch.equal(eng.prefill(ids), full.prefill(ids)) and eng.dropped == T - keep
        for (kc, vc), (fk, fv), mass in zip(eng.kv, full.kv, eng.mass):
            assert (mass[..., keep:] == 0).all() and (mass[..., :keep] >= 0).all()
            rows, all_rows = _held(kc, keep), _held(fk, T)
            for b in range(B):
                for h in range(2):                                            # each kept row is one of the prompt's, ascending
                    at = (rows[b, :, h, None].view(torch.int16) == all_rows[b, None, :, h].view(torch.int16)).all(-1).float().argmax(1)
                    assert same_bits(rows[b, :, h], all_rows[b, at, h]) and same_bits(_held(vc, keep)[b, :, h], _held(fv, T)[b, at, h])
                    assert (at.diff() > 0).all() and at[:3].tolist() == [0, 1, 2] and at[-10:].tolist() == list(range(T - 10, T))


def test_a_second_prefill_starts_over():
    m = _model("llama")
    ids = _ids(2, 120)
    eng = exactkv.Engine(m, 2, 64, layer_kernels=True, budget=exactkv.Budget(30, **KEEP))
    runs = []
    for _ in range(2):
        runs.append((eng.prefill(ids[:, :20]), _run(eng, ids, 20)))
        assert eng.dropped > 0
    assert torch.equal(runs[0][0], runs[1][0]) and same_bits(runs[0][1], runs[1][1])


def test_engine_budget_refusals():
    m = _model("llama")
    for kw in (dict(layer_kernels=False), dict(layer_kernels=True, attn=lambda *a: None), dict(layer_kernels=True, before_step=lambda *a: None)):
        with pytest.raises(AssertionError):
            exactkv.Engine(m, 1, 64, budget=exactkv.Budget(30), **kw)
    with pytest.raises(AssertionError):
        exactkv.Engine(m, 1, 64, layer_kernels=True, budget=exactkv.Budget(64))
    with pytest.raises(AssertionError):
        exactkv.Engine(_model("qwen2", 24), 1, 64, layer_kernels=True, budget=exactkv.Budget(30))
    m.config.max_position_embeddings = 80
    eng = exactkv.Engine(m, 1, 64, layer_kernels=True, budget=exactkv.Budget(30))
    m.config.max_position_embeddings = 4096
    with pytest.raises(AssertionError):
        eng.prefill(_ids(1, 81))
    eng.prefill(_ids(1, 70))
    for t in range(10):
        eng.step(_ids(1, 80)[:, 70 + t])
    with pytest.raises(RuntimeError, match="position 80"):
        eng.step(_ids(1, 1)[:, 0])


def test_engines_draw_their_tokens():
    m = _model("llama")
    ids = _ids(3, 20)

    def draw(seed, **kw):
        return exactkv.Sampler(generator=_gen(seed), **kw)
    for kw in (dict(), dict(layer_kernels=True)):
        greedy, logits = exactkv.Engine(m, 3, 64, **kw).generate(ids, 30)
        same, slogits = exactkv.Engine(m, 3, 64, **kw).generate(ids, 30, choose=draw(1, temperature=0.0))
        assert torch.equal(greedy, same) and same_bits(logits, slogits)
        a, la = exactkv.Engine(m, 3, 64, **kw).generate(ids, 30, choose=draw(2, temperature=1.5, top_k=200, top_p=0.95))
        b, _ = exactkv.Engine(m, 3, 64, **kw).generate(ids, 30, choose=draw(2, temperature=1.5, top_k=200, top_p=0.95))
        assert torch.equal(a, b) and not torch.equal(a, greedy)
        assert torch.isin(a[:, 1:].flatten(), torch.arange(1024, device=DEV)).all()
        rank = (la > la.gather(2, a[:, 1:, None])).sum(-1)
        assert (rank < 200).all()
    eng = exactkv.PagedEngine(m, 4, 64)
    s, t = eng.add(ids[0], choose=draw(3, top_k=1))
    slots, ts = eng.add_many([ids[1], ids[2, :7]], choose=draw(3, top_k=1))
    other = exactkv.PagedEngine(m, 4, 64)
    assert int(other.add(ids[0])[1]) == int(t) and torch.equal(other.add_many([ids[1], ids[2, :7]])[1], ts)
    choose = draw(4, temperature=0.8)
    tok = torch.cat([t[None], ts])
    for _ in range(20):
        tok = choose(eng.step(tok))
    assert tok.shape == (3,)


def test_a_generation_under_a_budget_with_sampling():
    """All of it as a user runs it: a prompt, a generation three times the caches, tokens drawn, two evictions and more."""
    m = _model("qwen3")
    ids = _ids(2, 50)
    out = []
    for backend in ("exactkv", "bf16"):
        eng = exactkv.Engine(m, 2, 64, backend=backend, layer_kernels=True, budget=exactkv.Budget(32, **KEEP))
        tokens, logits = eng.generate(ids, 150, choose=exactkv.Sampler(0.9, top_p=0.95, min_p=0.01, generator=_gen(5)))
        assert eng.dropped + eng.kv[0][0].T == 50 + 149 and torch.isfinite(logits.float()).all()
        out.append((tokens, logits))
    assert torch.equal(out[0][0], out[1][0]) and same_bits(out[0][1], out[1][1])


@pytest.mark.parametrize("layer_kernels", [False, True])
def test_settings_of_their_own_for_each_sequence(layer_kernels):
    """A Sampler with a setting per sequence draws the prompts' tokens too: a temperature of 0 is the greedy engine's choice."""
    m = _model("llama")
    ids = _ids(3, 20)
    t = torch.tensor([0.0, 1.5, 0.0], device=DEV)
    eng = exactkv.Engine(m, 3, 48, layer_kernels=layer_kernels)
    tokens, logits = eng.generate(ids, 12, choose=exactkv.Sampler(t, generator=_gen(3)))
    greedy = exactkv.Engine(m, 3, 48, layer_kernels=layer_kernels).generate(ids, 12)[0]
    assert torch.equal(tokens[::2], greedy[::2]) and not torch.equal(tokens[1], greedy[1])
