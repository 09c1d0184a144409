"""The refusals of the decoder-layer operators that need no GPU: the C entry points' checks of
shapes, strides and alignment (nothing is launched), and the wrappers' checks of types and
devices."""
import pytest
import torch

import exactkv_amd as exactkv
from exactkv_amd import _lib


def _fails(name, args, words):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == 1
    assert words.encode() in lib.exkv_last_error(), lib.exkv_last_error()


def _prompt(**kw):
    a = dict(q=16, sq_t=4096, sq_h=128, k=16, sk_t=1024, sk_h=128, v=16, sv_t=1024, sv_h=128, out=16, cu_q=4, cu_k=4, S=1,
             N=10, NK=10, Hq=32, Hkv=8, D=128, window=0, zero=0, scale=0.1, ws=None, wsb=0)
    a.update(kw)
    return (*a.values(), None)


@pytest.mark.parametrize("kw,words", [
    (dict(D=96), "head dim"), (dict(Hq=30), "query heads"), (dict(Hkv=0), "query heads"), (dict(window=-1), "bad shape"),
    (dict(N=-1), "bad shape"), (dict(q=None), "null pointer"), (dict(v=None), "null pointer"), (dict(q=24), "aligned"),
    (dict(sk_h=100), "aligned"), (dict(sq_t=-8), "aligned"), (dict(sk_t=64), "elements apart"),
    (dict(sv_t=1 << 24), "elements apart"), (dict(N=1 << 30, Hq=64), "too many rows"), (dict(S=1 << 30), "too many rows"),
    (dict(NK=1 << 30), "too many rows"),
], ids=str)
def test_prompt_attention_arguments(kw, words):
    _fails("exkv_prompt_attention", _prompt(**kw), words)


def _rotate(**kw):
    a = dict(q=16, sq_t=4096, sq_h=128, k=16, sk_t=1024, sk_h=128, cos=16, sin=16, rows=64, qn=None, kn=None, eps=1e-6,
             q_out=16, k_out=16, cu=4, start=None, S=1, N=10, Hq=32, Hkv=8, D=128)
    a.update(kw)
    return (*a.values(), None)


@pytest.mark.parametrize("kw,words", [
    (dict(D=32), "head dim"), (dict(rows=0), "bad shape"), (dict(Hkv=0), "bad shape"), (dict(cos=None), "null pointer"),
    (dict(q=18), "4-byte"), (dict(sk_t=1023), "4-byte"), (dict(qn=8), "16-byte"), (dict(q_out=8), "16-byte"),
    (dict(N=2 ** 31 - 1), "too many rows"),
], ids=str)
def test_rotate_prompt_arguments(kw, words):
    _fails("exkv_rotate_prompt", _rotate(**kw), words)


_ROWS = dict(q=16, sq_n=4096, sq_h=128, k=16, sk_n=1024, sk_h=128, v=16, sv_n=1024, sv_h=128, cos=16, sin=16, rows=64,
             qn=None, kn=None, eps=1e-6, out=16, n=2, Hq=32, Hkv=8)


def _append(tail, **kw):
    a = dict(_ROWS, **tail)
    a.update(kw)
    return (*a.values(), None)


def _cache(prefix, raw):
    return {prefix + x: 16 for x in ("sm", "code", "base", "mask", "off")} | {prefix + "raw": raw, prefix + "cnt": 4,
                                                                              prefix + "before": 4}


CONTIGUOUS = {**_cache("k", 16), "ks": 4, "kcap": 10, "krows": 1000, **_cache("v", 32), "vs": 4, "vcap": 10, "vrows": 1000,
              "TS": 64, "D": 128}
CONTIGUOUS_BF16 = dict(kbuf=16, ks=4, vbuf=32, vs=4, TS=64, D=128)
TABLE = dict(slots=None, lens=4, bt=4, stride=8, seqs=4, pages=8, pool=16, D=128)
PAGED = {**_cache("k", 16), "arr": 4, "kcap": 10, "krows": 1000, **_cache("v", 32), "vcap": 10, "vrows": 1000, **TABLE}
PAGED_BF16 = dict(kbuf=16, vbuf=32, **TABLE)
ENTRIES = [("exkv_rope_append", CONTIGUOUS), ("exkv_rope_append_bf16", CONTIGUOUS_BF16), ("exkv_rope_append_paged", PAGED),
           ("exkv_rope_append_paged_bf16", PAGED_BF16)]


@pytest.mark.parametrize("name,tail", ENTRIES, ids=[e[0] for e in ENTRIES])
@pytest.mark.parametrize("kw,words", [
    (dict(D=96), "head dim"), (dict(Hq=0), "bad shape"), (dict(rows=0), "bad shape"), (dict(n=-1), "bad shape"),
    (dict(q=None), "null pointer"), (dict(k=18), "4-byte"), (dict(sv_n=1023), "4-byte"), (dict(out=8), "16-byte"),
    (dict(cos=8), "16-byte"), (dict(n=1 << 27), "too many rows"),
], ids=str)
def test_rope_append_rows(name, tail, kw, words):
    _fails(name, _append(tail, **kw), words)


@pytest.mark.parametrize("name,tail,kw,words", [
    ("exkv_rope_append", CONTIGUOUS, dict(TS=60), "bad shape"),
    ("exkv_rope_append", CONTIGUOUS, dict(krows=100), "tail area"),
    ("exkv_rope_append", CONTIGUOUS, dict(vraw=16), "one cache"),
    ("exkv_rope_append", CONTIGUOUS, dict(vs=None), "null pointer"),
    ("exkv_rope_append_bf16", CONTIGUOUS_BF16, dict(vbuf=16), "one cache"),
    ("exkv_rope_append_bf16", CONTIGUOUS_BF16, dict(TS=0), "bad shape"),
    ("exkv_rope_append_paged", PAGED, dict(seqs=1), "bad shape"),
    ("exkv_rope_append_paged", PAGED, dict(stride=4), "page table"),
    ("exkv_rope_append_paged", PAGED, dict(vrows=300), "tail area"),
    ("exkv_rope_append_paged", PAGED, dict(arr=None), "null pointer"),
    ("exkv_rope_append_paged_bf16", PAGED_BF16, dict(vbuf=16), "one pool"),
    ("exkv_rope_append_paged_bf16", PAGED_BF16, dict(pool=0), "page table"),
], ids=str)
def test_rope_append_caches(name, tail, kw, words):
    _fails(name, _append(tail, **kw), words)


@pytest.mark.parametrize("kw,words", [
    (dict(C=0), "channels"), (dict(C=16385), "channels"), (dict(x=None), "null pointer"), (dict(sx=-1), "negative"),
    (dict(r=17), "unaligned"),
], ids=str)
def test_add_norm_arguments(kw, words):
    a = dict(x=16, sx=64, r=16, sr=64, w=16, pw=None, gate=None, sg=0, scale=1.0, eps=1e-6, h=16, y=16, N=4, C=64)
    a.update(kw)
    _fails("exkv_add_norm", (*a.values(), None), words)


def test_no_rows_is_no_call():
    lib = _lib.load()
    assert lib.exkv_prompt_attention(*_prompt(N=0)) == 0
    assert lib.exkv_rotate_prompt(*_rotate(N=0)) == 0
    for name, tail in ENTRIES:
        assert getattr(lib, name)(*_append(tail, n=0)) == 0
    assert lib.exkv_add_norm(16, 64, None, 0, 16, None, None, 0, 1.0, 1e-6, 16, 16, 0, 64, None) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    t = torch.zeros(8, 64)
    with pytest.raises(ValueError, match="GPU"):
        exactkv.prompt_attention(x, x, x, cu)
    with pytest.raises(ValueError, match="GPU"):
        exactkv.rotate_prompt(x, x, t, t, cu)
    with pytest.raises(ValueError, match="GPU"):
        exactkv.rope_append_paged(x, x, x, t, t, x[None], x[None], cu, cu[None])
    with pytest.raises(ValueError, match="GPU"):
        exactkv.add_norm(x, x, x[0, 0])
    with pytest.raises(TypeError, match="one kind"):
        exactkv.rope_append(x, x, x, t, t, x, x)
