"""After an eviction a token's place in its cache is no longer its position: what takes the one for the other says so
instead of rotating wrongly.

No counterpart in the reference, whose caches keep every token (exactkv/cache.py)."""
import pytest
import torch

import exactkv_amd as exactkv
from tests.test_engine_host import _tiny
from tests.test_gpu_engine_layers import _ids, _model

DEV = "cuda"


def test_a_page_table_counts_what_was_cut():
    t = exactkv.PageTable(20, 3, 10, device="cpu")
    a, b = t.add(100), t.add(40)
    assert t.dropped(a) == t.dropped(b) == 0
    t.cut(a, 30)
    assert t.length(a) == 30 and t.dropped(a) == 70 and t.dropped(b) == 0
    t.begin_step([a, b])
    t.cut(a, 20)
    assert t.length(a) == 20 and t.dropped(a) == 81
    t.truncate(a, 18)                                  # the latest two are taken back: the others stay where they stand
    assert t.dropped(a) == 81
    t.truncate(a, 0)                                   # a sequence that starts over
    assert t.dropped(a) == 0
    t.cut(b, 41)                                       # (all of it: begin_step counted one more)
    assert t.dropped(b) == 0
    t.cut(b, 7)
    t.release(b)
    assert t.add(5) == b and t.dropped(b) == 0
    for n in (-1, 6):
        with pytest.raises(ValueError):
            t.cut(b, n)
    import copy
    t.cut(b, 1)
    assert copy.deepcopy(t).dropped(b) == 4


def test_a_paged_engine_does_not_go_on():
    """Its steps take a sequence's length for its position: slots that were cut are refused before anything changes."""
    eng = exactkv.PagedEngine(_tiny("llama").bfloat16(), 3, 64, backend="bf16", graph=False)
    slots = [eng.add(torch.arange(n))[0] for n in (20, 30)]
    eng.table.cut(slots[1], 10)
    for which in (None, [slots[1]], slots):
        with pytest.raises(RuntimeError, match="cut"):
            eng.step(torch.zeros(2, dtype=torch.long), which)
    assert [eng.table.length(s) for s in slots] == [20, 10] and eng.table.step == 0
    eng.release(slots[1])
    assert eng.add(torch.arange(30))[0] == slots[1]


def test_slots_are_read_once():
    """A step's slots may be any iterable, beside slots that were cut too."""
    eng = exactkv.PagedEngine(_tiny("llama").bfloat16(), 3, 64, backend="bf16", graph=False)
    slots = [eng.add(torch.arange(n))[0] for n in (20, 30)]
    eng.table.cut(slots[1], 10)
    seen = []
    eng.table.begin_step = lambda which: seen.append(list(which)) or [][0]     # (the step's kernels need a GPU: it ends here)
    for which in (iter(slots[:1]), slots[:1], (s for s in slots[:1])):
        with pytest.raises(IndexError):
            eng.step(torch.zeros(1, dtype=torch.long), which)
    assert seen == [[0]] * 3


def test_one_table_of_angles_is_one_distance():
    """rope_append over pages has one table for all rows of a step: slots that were cut by different numbers of tokens are refused."""
    t = exactkv.PageTable(20, 3, 10, device="cpu")
    k, v = exactkv.PagedBF16KV(t, 2, D=64), exactkv.PagedBF16KV(t, 2, D=64)
    for n in (40, 30, 30):
        t.add(n)
    t.cut(0, 20)
    x, q, angles = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(100, 32)
    t.begin_step()
    with pytest.raises(RuntimeError, match="cut"):
        exactkv.rope_append(q, x, x, angles, angles, k, v)
    t.cut(1, 11), t.cut(2, 11)                         # all by 20
    t.begin_step()
    with pytest.raises(ValueError, match="GPU"):       # (past that check)
        exactkv.rope_append(q, x, x, angles, angles, k, v)


@pytest.mark.gpu
@pytest.mark.parametrize("layer_kernels", [False, True])
def test_evicting_a_paged_engines_caches(layer_kernels):
    m = _model("llama")
    ids = _ids(2, 60)
    eng = exactkv.PagedEngine(m, 3, 96, layer_kernels=layer_kernels)
    slots = [eng.add(x)[0] for x in ids]
    mass = [torch.rand(3, 2, eng.table.capacity, device=DEV) for _ in eng.kv]
    exactkv.evict(*zip(*eng.kv), mass, 80)                                     # nobody is that long
    eng.step(ids[:, 0])
    exactkv.evict(*zip(*eng.kv), mass, 30, slots=[slots[0]])
    assert eng.table.dropped(slots[0]) == 31 and eng.table.dropped(slots[1]) == 0
    with pytest.raises(RuntimeError, match="cut"):
        eng.step(ids[:, 0])
    eng.step(ids[1:, 0], [slots[1]])
    eng.release(slots[0])
    assert eng.add(ids[0])[0] == slots[0]
    assert eng.step(ids[:, 1]).shape == (2, 1024)


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [exactkv.CompressedKV, exactkv.BF16KV])
def test_contiguous_caches_count_what_was_cut(cls):
    k, v = cls(1, 64, 2, 64), cls(1, 64, 2, 64)
    x = torch.randn(1, 40, 2, 64, device=DEV).bfloat16()
    for c in (k, v):
        c.prefill_slot(0, x)
        assert c.dropped == 0
    mass = torch.rand(1, 2, 64, device=DEV)
    exactkv.evict(k, v, mass, 30)
    assert k.dropped == v.dropped == 10
    for c in (k, v):
        c.append(x[:, 0].contiguous())
    exactkv.evict(k, v, mass, 12)
    assert k.dropped == v.dropped == 29 and k.T == 12
    k.replace(x)
    v.prefill_slot(0, x)
    assert k.dropped == v.dropped == 0


@pytest.mark.gpu
@pytest.mark.parametrize("budget", [None, exactkv.Budget(20, 2, 4)])
def test_evicting_an_engines_caches_from_outside(budget):
    """An Engine counts the evictions that it makes itself; of others' it says so, until the next prefill."""
    m = _model("llama")
    ids = _ids(2, 60)
    eng = exactkv.Engine(m, 2, 64, layer_kernels=budget is not None, budget=budget)
    eng.prefill(ids[:, :40])
    mass = [torch.rand(2, 2, 64, device=DEV) for _ in eng.kv]
    exactkv.evict(*zip(*eng.kv), mass, 30)
    with pytest.raises(RuntimeError, match="cut"):
        eng.step(ids[:, 40])
    assert eng.kv[0][0].T == 30
    eng.prefill(ids[:, :40])
    assert eng.step(ids[:, 40]).shape == (2, 1024) and eng.kv[0][0].T == 41
