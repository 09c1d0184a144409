"""An Engine's budget where its work comes in pieces or ends halfway: prompts prefilled by b0=, an eviction that fails.

No counterpart in the reference, whose caches end when they are full (exactkv/cache.py:102)."""
import pytest
import torch

import exactkv_amd as exactkv
from tests.conftest import same_bits
from tests.test_gpu_budget import KEEP, _held, _run
from tests.test_gpu_engine_layers import _ids, _model

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("first,then", [(100, 140), (140, 100), (30, 100), (100, 30), (40, 30), (64, 65)])
def test_pieces_of_different_lengths_are_refused(first, then):
    """All sequences of an Engine stand at one position: a piece of another length is refused, and nothing is written. Of
    one length, pieces give what one prefill gives."""
    m = _model("llama")
    ids = _ids(4, 160)
    eng = exactkv.Engine(m, 4, 64, layer_kernels=True, budget=exactkv.Budget(30, **KEEP))
    eng.prefill(ids[:2, :first])
    before = [(c.T, _held(c, c.T).clone()) for c in eng._caches()]
    mass, dropped = [x.clone() for x in eng.mass], eng.dropped
    with pytest.raises(AssertionError, match="position"):
        eng.prefill(ids[2:, :then], b0=2)
    assert eng.dropped == dropped and all(torch.equal(a, b) for a, b in zip(mass, eng.mass))
    assert all(c.T == T and same_bits(_held(c, T), x) for c, (T, x) in zip(eng._caches(), before))
    eng.prefill(ids[2:, :first], b0=2)
    whole = exactkv.Engine(m, 4, 64, layer_kernels=True, budget=exactkv.Budget(30, **KEEP))
    whole.prefill(ids[:, :first])
    rows = [c.T for c in eng._caches()]
    assert eng.dropped == whole.dropped and rows == [c.T for c in whole._caches()]
    for a, b in zip(eng._caches(), whole._caches()):
        assert same_bits(_held(a, a.T), _held(b, b.T))
    eng.prefill(ids[:2, :then])                                                # slot 0 starts over
    eng.prefill(ids[2:, :then], b0=2)
    assert eng.dropped + eng.kv[0][0].T == then


def test_a_piece_after_steps_is_refused():
    m = _model("llama")
    ids = _ids(3, 100)
    eng = exactkv.Engine(m, 3, 64, layer_kernels=True, budget=exactkv.Budget(30, **KEEP))
    eng.prefill(ids[:, :40])
    _run(eng, ids[:, :80], 40)                                                 # over an eviction
    for n in (40, 80, eng.kv[0][0].T):
        with pytest.raises(AssertionError, match="position"):
            eng.prefill(ids[2:, :n], b0=2)


@pytest.mark.parametrize("fails_at", [1, 2, 3])
def test_an_eviction_that_fails_halfway_is_noticed(fails_at, monkeypatch):
    """Two layers; memory runs out (as far as the caches know) at one of the four replacements. The step raises, and so does the
    next one, until a prefill starts over."""
    m = _model("llama")
    ids = _ids(2, 90)
    eng = exactkv.Engine(m, 2, 64, layer_kernels=True, budget=exactkv.Budget(30, **KEEP))
    eng.prefill(ids[:, :60])
    want = _run(eng, ids, 60)
    eng.prefill(ids[:, :60])
    _run(eng, ids[:, :64], 60)
    real, calls = exactkv.CompressedKV.replace, []

    def replace(self, x):
        calls.append(x)
        if len(calls) == fails_at + 1:
            raise torch.cuda.OutOfMemoryError("no memory")
        return real(self, x)
    monkeypatch.setattr(exactkv.CompressedKV, "replace", replace)
    with pytest.raises(torch.cuda.OutOfMemoryError):
        eng.step(ids[:, 64])
    monkeypatch.undo()
    for _ in range(2):
        with pytest.raises(RuntimeError, match="cut"):
            eng.step(ids[:, 64])
    eng.prefill(ids[:, :60])
    assert same_bits(_run(eng, ids, 60), want)


def test_what_is_wrong_with_a_later_layer_is_said_before_the_first_is_cut():
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(1, 40, 2, 64, generator=g, device=DEV).bfloat16()
    layers = [[exactkv.BF16KV(1, 48, 2, 64, device=d) for _ in "kv"] for d in (DEV, DEV, "cpu")]
    for pair in layers:
        for c in pair:
            c.prefill_slot(0, x.to(c.buf.device))
    mass = [torch.rand(1, 2, 48, generator=g, device=DEV) for _ in range(3)]
    keys, values = ([p[i] for p in layers] for i in (0, 1))
    with pytest.raises(ValueError, match="GPU"):
        exactkv.evict(keys, values, mass, 20)
    for m in ([mass[0], mass[0]], [mass[0], mass[0].view(-1)[:96].view(1, 2, 48)]):
        with pytest.raises(ValueError, match="mass"):
            exactkv.evict(keys[:2], values[:2], m, 20)
    assert all(c.T == 40 for p in layers for c in p) and same_bits(_held(keys[0], 40), x)
    exactkv.evict(keys[:2], values[:2], mass[:2], 20.0)
    assert all(c.T == 20 for p in layers[:2] for c in p)
