"""The refusals of sampling and eviction that need no GPU: the C entry points' checks of shapes, strides, alignment and
workspaces (nothing is launched), and the wrappers' checks of devices."""
import pytest
import torch

import exactkv_amd as exactkv
from exactkv_amd import _lib


def _fails(name, args, words):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == 1
    assert words.encode() in lib.exkv_last_error(), lib.exkv_last_error()


def _sample(**kw):
    a = dict(logits=16, stride=100, type=0, B=4, V=100, u=16, t=None, k=None, p=None, m=None, t0=1.0, k0=0, p0=1.0, m0=0.0, token=16, lp=None, ws=None,
             wsb=0)
    a.update(kw)
    return (*a.values(), None)


@pytest.mark.parametrize("kw,words", [
    (dict(type=3), "type"), (dict(type=-1), "type"), (dict(V=0), "bad shape"), (dict(V=2 ** 19 + 1), "bad shape"), (dict(B=-1), "bad shape"),
    (dict(stride=-1), "bad shape"), (dict(B=2 ** 23), "too many rows"), (dict(logits=None), "null pointer"), (dict(u=None), "null pointer"),
    (dict(token=None), "null pointer"), (dict(logits=17), "aligned"), (dict(type=2, logits=18), "aligned"), (dict(V=9000), "workspace"),
    (dict(V=9000, ws=16, wsb=100), "workspace"), (dict(V=9000, ws=24, wsb=1 << 30), "workspace"),
], ids=str)
def test_sample_arguments(kw, words):
    _fails("exkv_sample", _sample(**kw), words)


_MASS = dict(table=None, tstride=0, pages=0, B=2, Hq=32, Hkv=8, D=128, T=100, TS=128, lens=None, ls=0, window=0, scale=0.1, mass=None, out=16,
             fresh=0, ws=16, wsb=1 << 30)


def _mass(bf16, **kw):
    a = dict(q=16, k=16) if bf16 else dict(q=16, sm=16, code=16, base=16, mask=16, off=16, raw=16, rows=10)
    a.update(_MASS)
    a.update(kw)
    return (*a.values(), None)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kw,words", [
    (dict(D=96), "head dim"), (dict(Hq=30), "query heads"), (dict(Hkv=0), "query heads"), (dict(T=129), "bad shape"), (dict(window=-1), "bad shape"),
    (dict(B=-1), "bad shape"), (dict(ls=-1), "negative stride"), (dict(q=None), "null pointer"), (dict(out=None), "null pointer"),
    (dict(ws=None), "null pointer"), (dict(wsb=100), "workspace"), (dict(ws=24), "workspace"), (dict(table=16, tstride=7, pages=9), "page table"),
    (dict(table=16, tstride=8, pages=0), "page table"), (dict(TS=2 ** 31 - 16, T=0), "TS="), (dict(B=2 ** 22, wsb=2 ** 62), "too many workgroups"),
    (dict(Hq=32768, Hkv=8), "query heads"),
], ids=str)
def test_attention_mass_arguments(bf16, kw, words):
    _fails("exkv_attention_mass_bf16" if bf16 else "exkv_attention_mass", _mass(bf16, **kw), words)


def test_attention_mass_caches():
    _fails("exkv_attention_mass", _mass(False, TS=120), "multiple")
    _fails("exkv_attention_mass", _mass(False, sm=None), "null pointer")
    _fails("exkv_attention_mass", _mass(False, rows=0), "null pointer")
    _fails("exkv_attention_mass_bf16", _mass(True, k=None), "null pointer")
    _fails("exkv_attention_mass_bf16", _mass(True, table=16, tstride=8, pages=9, TS=120), "multiple")


def _prompt(**kw):
    a = dict(q=16, sq_t=4096, sq_h=128, k=16, sk_t=1024, sk_h=128, cu_q=4, cu_k=4, S=1, N=10, NK=10, Hq=32, Hkv=8, D=128, window=0, last=0,
             scale=0.1, out=16, ws=16, wsb=1 << 40)
    a.update(kw)
    return (*a.values(), None)


@pytest.mark.parametrize("kw,words", [
    (dict(D=96), "head dim"), (dict(Hq=30), "query heads"), (dict(window=-1), "bad shape"), (dict(last=-1), "bad shape"), (dict(N=-1), "bad shape"),
    (dict(q=None), "null pointer"), (dict(k=None), "null pointer"), (dict(out=None), "null pointer"), (dict(q=24), "aligned"), (dict(sk_h=100), "aligned"),
    (dict(sq_t=-8), "aligned"), (dict(sk_t=64), "elements apart"), (dict(sq_t=1 << 24), "elements apart"), (dict(N=1 << 30, Hq=64), "too many rows"),
    (dict(NK=1 << 30), "too many rows"), (dict(S=1 << 30), "too many rows"), (dict(wsb=16), "workspace"), (dict(ws=24), "workspace"), (dict(ws=None), "workspace"),
], ids=str)
def test_prompt_mass_arguments(kw, words):
    _fails("exkv_prompt_mass", _prompt(**kw), words)


@pytest.mark.parametrize("S,N,NK,Hq,Hkv,D,window,last", [(1, 1, 1, 1, 1, 64, 0, 0), (1, 8192, 8192, 32, 8, 128, 0, 0), (3, 17, 50000, 14, 2, 256, 0, 0),
                                                         (1, 512, 16385, 32, 8, 128, 0, 64), (200, 200, 9000, 8, 1, 64, 512, 1)])
def test_workspaces_hold_what_the_calls_need(S, N, NK, Hq, Hkv, D, window, last):
    lib = _lib.load()
    need = lib.exkv_prompt_mass_workspace(S, N, NK, Hq, Hkv, D, window, last)
    assert need >= 4 * Hq * N                                                 # a sum a row
    _fails("exkv_prompt_mass", _prompt(S=S, N=N, NK=NK, Hq=Hq, Hkv=Hkv, D=D, window=window, last=last, sq_t=Hq * D, sk_t=Hkv * D, wsb=need - 1),
           "workspace")
    B, TS = 3, -(-NK // 16) * 16
    for lens in (0, 1):
        need = lib.exkv_mass_workspace(B, Hq, Hkv, NK, TS, lens, window)
        assert need >= 4 * B * Hq * TS + 8 * B * Hq
        _fails("exkv_attention_mass", _mass(False, B=B, Hq=Hq, Hkv=Hkv, D=D, T=NK, TS=TS, lens=16 if lens else None, window=window, wsb=need - 1),
               "workspace")


def _select(**kw):
    a = dict(mass=16, s_b=100, s_h=50, lens=None, ls=0, T=40, B=2, H=2, TS=50, keep=10, sinks=1, recent=2, index=16, kept=16)
    a.update(kw)
    return (*a.values(), None)


@pytest.mark.parametrize("kw,words", [
    (dict(T=51), "bad shape"), (dict(H=0), "bad shape"), (dict(sinks=9), "tokens of"), (dict(recent=-1), "tokens of"), (dict(keep=-1), "tokens of"),
    (dict(mass=None), "null pointer"), (dict(index=None), "null pointer"), (dict(kept=None), "null pointer"), (dict(s_b=-1), "negative"),
    (dict(B=2 ** 22), "too many rows"),
], ids=str)
def test_select_tokens_arguments(kw, words):
    _fails("exkv_select_tokens", _select(**kw), words)


def _gather(bf16, **kw):
    cache = dict(sm=16, code=16, base=16, mask=16, off=16, raw=16, rows=10)
    a = dict(k=16, v=16) if bf16 else {s + n: x for s in "kv" for n, x in cache.items()}
    a.update(table=None, ts=0, pages=0, B=2, H=2, TS=48, D=128, index=16, keep=10, ko=16, vo=16)
    a.update(kw)
    return (*a.values(), None)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kw,words", [
    (dict(D=32), "head dim"), (dict(H=0), "bad shape"), (dict(keep=-1), "bad shape"), (dict(table=16, ts=2, pages=5), "page table"),
    (dict(table=16, ts=3, pages=0), "page table"), (dict(index=None), "null pointer"), (dict(ko=None), "null pointer"),
    (dict(B=2 ** 20, keep=2 ** 12), "too many rows"),
], ids=str)
def test_gather_tokens_arguments(bf16, kw, words):
    _fails("exkv_gather_tokens_bf16" if bf16 else "exkv_gather_tokens", _gather(bf16, **kw), words)


def test_gather_tokens_caches():
    _fails("exkv_gather_tokens", _gather(False, TS=40), "TS=40")
    _fails("exkv_gather_tokens", _gather(False, vrows=0), "raw rows")
    _fails("exkv_gather_tokens", _gather(False, kcode=None), "null pointer")
    _fails("exkv_gather_tokens_bf16", _gather(True, v=None), "null pointer")


def test_tensors_must_be_on_a_gpu():
    z = torch.zeros
    with pytest.raises(ValueError, match="GPU"):
        exactkv.sample(z(2, 5), z(2))
    with pytest.raises(ValueError, match="GPU"):
        exactkv.attention_mass(z(1, 4, 64, dtype=torch.bfloat16), z(1, 16, 2, 64, dtype=torch.bfloat16), 3)
    with pytest.raises(ValueError, match="GPU"):
        exactkv.prompt_mass(z(3, 4, 64, dtype=torch.bfloat16), z(3, 2, 64, dtype=torch.bfloat16), z(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        exactkv.select_tokens(z(1, 2, 16), 4, 16)
    with pytest.raises(ValueError, match="GPU"):
        exactkv.gather_tokens(z(1, 16, 2, 64, dtype=torch.bfloat16), z(1, 16, 2, 64, dtype=torch.bfloat16), z(1, 2, 4, dtype=torch.int32))


def test_truncated_sequences_give_their_pages_back():
    t = exactkv.PageTable(20, 2, 10, device="cpu")
    a, b = t.add(100), t.add(40)
    held, free = t.pages(a), t.free_pages()
    t.truncate(a, 33)
    assert t.length(a) == 33 and t.pages(a) == held[:3] and t.free_pages() == free + 4 and int(t.lens[a]) == 33
    t.truncate(a, 32)                                  # its open page, the third, stays
    assert t.pages(a) == held[:3]
    with pytest.raises(RuntimeError):
        t.step_rows()
    t.begin_step([a, b])
    assert t.length(a) == 33
    t.truncate(a, 0)
    assert t.pages(a) == held[:1]
    for slot, T in ((a, 1), (b, -1), (b, 100)):
        with pytest.raises(ValueError):
            t.truncate(slot, T)
    t.release(b)
    with pytest.raises(ValueError):
        t.truncate(b, 0)


def test_budgets():
    b = exactkv.Budget(100)
    assert (b.keep, b.sinks, b.recent, b.last) == (100, 4, 25, 0)
    for a in ((0,), (10, 11), (10, 4, 7), (10, -1), (10, 0, -1), (10, 0, 0, -1)):
        with pytest.raises(ValueError):
            exactkv.Budget(*a)


@pytest.mark.parametrize("how", ["deepcopy", "pickle"])
def test_copies_of_a_page_table_and_its_caches(how):
    """A table knows the caches over it, the copies' as well, and keeps none of them alive."""
    import copy
    import gc
    import pickle
    table = exactkv.PageTable(8, 2, 4, device="cpu")
    k, v = exactkv.PagedBF16KV(table, 2, D=64), exactkv.PagedBF16KV(table, 2, D=64)
    table.add(20)
    assert {id(c) for c in table.caches()} == {id(k), id(v)}
    t2, k2, v2 = copy.deepcopy((table, k, v)) if how == "deepcopy" else pickle.loads(pickle.dumps((table, k, v)))
    assert k2.table is t2 and {id(c) for c in t2.caches()} == {id(k2), id(v2)} and t2.length(0) == 20 and t2.free_pages() == table.free_pages()
    del v
    gc.collect()
    assert table.caches() == [k]
