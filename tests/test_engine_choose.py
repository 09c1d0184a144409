"""A choose= that fails: the prompts that were added for it are taken out again.

No counterpart in the reference, whose engine has no choice to make (exactkv/engine.py:93-95)."""
import pytest
import torch

import exactkv_amd as exactkv
from tests.test_engine_host import _tiny


def _fails(logits):
    raise ValueError("choose")


def test_add_on_the_host():
    """Through the model's own modules, and a prompt that the model refuses."""
    eng = exactkv.PagedEngine(_tiny("llama").bfloat16(), 2, 64, backend="bf16", graph=False)
    ids = torch.arange(20)
    free = eng.table.free_pages()
    with pytest.raises(ValueError, match="choose"):
        eng.add(ids, choose=_fails)
    assert eng.table.live_slots() == [] and eng.table.free_pages() == free
    with pytest.raises(Exception):
        eng.add(torch.full((20,), 10 ** 6))            # no such token
    assert eng.table.live_slots() == [] and eng.table.free_pages() == free
    slot, token = eng.add(ids)
    assert slot == 0 and 0 <= int(token) < 256


@pytest.mark.gpu
@pytest.mark.parametrize("layer_kernels", [False, True])
def test_add_and_add_many(layer_kernels):
    m = _tiny("llama").to("cuda").bfloat16()
    eng = exactkv.PagedEngine(m, 4, 64, layer_kernels=layer_kernels)
    ids = torch.arange(20, device="cuda")
    kept, _ = eng.add(ids)
    free = eng.table.free_pages()
    wrong = exactkv.Sampler(temperature=torch.ones(3, device="cuda"))          # settings of three rows
    for call in (lambda: eng.add(ids, choose=wrong), lambda: eng.add_many([ids, ids[:5]], choose=wrong), lambda: eng.add(ids, choose=_fails)):
        with pytest.raises(ValueError):
            call()
        assert eng.table.live_slots() == [kept] and eng.table.free_pages() == free
    slots, tokens = eng.add_many([ids, ids[:5], ids[:7]], choose=wrong)
    assert slots == [1, 2, 3] and tokens.shape == (3,)
    assert eng.step(torch.cat([tokens[:1], tokens])).shape == (4, 256)
