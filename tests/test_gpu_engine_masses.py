"""What an Engine under a budget evicts by: the attention that its tokens have received, against softmaxes in 64 bits over
the rows that its caches hold, of the queries that its layers ask with.

Tolerances of a weight are those of tests/test_gpu_mass.py; sums over steps add up their bounds and 2^-24 of the sum a step.
A token that stays has no less than one that goes, to those bounds.

No counterpart in the reference, which keeps no weights and every token."""
import pytest
import torch

import exactkv_amd as exactkv
from exactkv_amd import engine as engines
from tests.conftest import same_bits
from tests.test_gpu_budget import KEEP, _gathered, _held
from tests.test_gpu_engine_layers import _ids, _model
from tests.test_gpu_mass import _weights

pytestmark = pytest.mark.gpu
DEV = "cuda"
SINKS, RECENT = KEEP["sinks"], KEEP["recent"]


def _place(rows, all_rows):
    """Of rows [n, D] each one's index among all_rows [T, D], by their bits."""
    same = (rows[:, None].view(torch.int16) == all_rows[None].view(torch.int16)).all(-1)
    assert same.any(1).all()
    return same.float().argmax(1)


def _by_mass(kept, mass, bound, keep):
    """kept (ascending): the first ones, the latest ones, and between them none with less than one that went."""
    T = mass.shape[0]
    assert kept.shape == (keep,) and (kept.diff() > 0).all()
    assert kept[:SINKS].tolist() == list(range(SINKS)) and kept[-RECENT:].tolist() == list(range(T - RECENT, T))
    went = torch.ones(T, dtype=torch.bool, device=DEV)
    went[kept] = False
    middle = kept[SINKS:-RECENT]
    assert (mass + bound)[middle].min() >= (mass - bound)[went].max()
    assert mass[middle].min() > 0 and mass[middle].mean() > mass[went].mean()     # (they tell tokens apart)


@pytest.mark.parametrize("kind", ["llama", "qwen3"])
@pytest.mark.parametrize("last", [0, 32])
@pytest.mark.parametrize("backend", ["exactkv", "bf16"])
def test_a_prompt_is_cut_by_what_its_queries_give(kind, last, backend, monkeypatch):
    m = _model(kind)
    B, T, keep = 2, 200, 50
    ids = _ids(B, T)
    asked = []
    real = engines.prompt_attention

    def prompt_attention(q, k, v, cu, **kw):
        asked.append((q.clone(), k.clone(), v.clone()))
        return real(q, k, v, cu, **kw)
    monkeypatch.setattr(engines, "prompt_attention", prompt_attention)
    eng = exactkv.Engine(m, B, 64, backend=backend, layer_kernels=True, budget=exactkv.Budget(keep, last=last, **KEEP))
    eng.prefill(ids)
    assert len(asked) == eng.L
    for (q, k, v), (kc, vc), got in zip(asked, eng.kv, eng.mass):
        rows, values = _held(kc, keep), _held(vc, keep)
        for b in range(B):
            at = slice(b * T, (b + 1) * T)
            queries = torch.arange(T - last if last else 0, T, device=DEV)
            w, err = (x.view(eng.Hkv, -1, T).sum(1) for x in _weights(q[at][queries], k[at], queries, 0))
            for h in range(eng.Hkv):
                kept = _place(rows[b, :, h], k[at][:, h])
                assert same_bits(values[b, :, h], v[at][kept, h])
                _by_mass(kept, w[h], err[h], keep)
                assert ((got[b, h, :keep].double() - w[h, kept]).abs() <= err[h, kept]).all()
        assert (got[..., keep:] == 0).all()


@pytest.mark.parametrize("kind", ["llama", "qwen3"])
@pytest.mark.parametrize("backend", ["exactkv", "bf16"])
def test_steps_add_what_their_queries_give(kind, backend):
    """Masses after each step, and the rows that the next eviction keeps; a captured engine beside it agrees bit for bit."""
    m = _model(kind)
    B, T, keep, room = 2, 50, 30, 64
    ids = _ids(B, T + 60)

    def engine(graph):
        e = exactkv.Engine(m, B, room, backend=backend, graph=graph, layer_kernels=True, budget=exactkv.Budget(keep, **KEEP))
        e.prefill(ids[:, :T])
        return e
    eng, captured = engine(False), engine(True)
    asked = []
    real = eng._attend

    def attend(q, kc, vc, window=0):
        asked.append(q.clone())
        return real(q, kc, vc, window)
    eng._attend = attend
    want = [x.double() for x in eng.mass]
    bound = [torch.zeros_like(x) for x in want]
    cuts = 0
    for t in range(T, T + 60):
        held = [(_held(kc, kc.T).clone(), _held(vc, vc.T).clone()) for kc, vc in eng.kv]
        full = eng.kv[0][0].T == room
        asked.clear()
        assert same_bits(eng.step(ids[:, t]), captured.step(ids[:, t]))
        assert len(asked) == eng.L
        n = eng.kv[0][0].T
        for i, ((kc, vc), q) in enumerate(zip(eng.kv, asked)):
            rows = _held(kc, n)
            if full:                                   # cut to the budget before this step's token
                assert n == keep + 1
                at = torch.stack([torch.stack([_place(rows[b, :keep, h], held[i][0][b, :, h]) for h in range(eng.Hkv)]) for b in range(B)])
                assert same_bits(_held(vc, keep), _gathered(held[i][1], at))
                for b in range(B):
                    for h in range(eng.Hkv):
                        _by_mass(at[b, h], want[i][b, h, :room], bound[i][b, h, :room], keep)
                for x in (want, bound):
                    kept = x[i].gather(2, at)
                    x[i] = torch.zeros_like(x[i])
                    x[i][..., :keep] = kept
            for b in range(B):
                w, err = (x.view(eng.Hkv, -1, n).sum(1) for x in _weights(q[b:b + 1], rows[b], torch.tensor([n - 1], device=DEV), 0))
                want[i][b, :, :n] += w
                bound[i][b, :, :n] += err + 2.0 ** -24 * want[i][b, :, :n]
            assert ((eng.mass[i].double() - want[i]).abs() <= bound[i]).all(), (t, i)
            assert torch.equal(eng.mass[i], captured.mass[i])
        cuts += full
    assert cuts >= 1 and captured.captures > 0
