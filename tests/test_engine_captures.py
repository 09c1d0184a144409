"""Engines that went: their memory, and their graphs while another engine captures its step, where no garbage may be collected.

No counterpart in the reference, whose steps are not captured (exactkv/engine.py:66-91)."""
import contextlib
import gc
import weakref

import pytest
import torch

import exactkv_amd as exactkv
from exactkv_amd import engine as engines
from tests.conftest import same_bits
from tests.test_engine_host import _tiny


@pytest.mark.parametrize("collects", [True, False])
def test_no_collection_in_a_capture(collects, monkeypatch):
    """Nor is a graph kept that was not captured to its end; the collector is left as it was."""
    seen = []

    @contextlib.contextmanager
    def graph(g, stream=None):
        seen.append((g, stream, gc.isenabled()))
        yield
    monkeypatch.setattr(torch.cuda, "graph", graph)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: "graph")
    was = gc.isenabled()
    try:
        (gc.enable if collects else gc.disable)()
        with engines._captured("stream") as g:
            assert g == "graph" and not gc.isenabled()
        assert gc.isenabled() == collects
        with pytest.raises(ValueError):
            with engines._captured("stream"):
                raise ValueError
        assert gc.isenabled() == collects
    finally:
        (gc.enable if was else gc.disable)()
    assert seen == [("graph", "stream", False)] * 2


@pytest.mark.parametrize("paged", [False, True])
def test_an_engine_goes_with_its_last_name(paged):
    """Its caches are most of a GPU's memory: they wait for no collection."""
    m = _tiny("llama").bfloat16()
    if paged:
        eng = exactkv.PagedEngine(m, 2, 64, backend="bf16", graph=False, layer_kernels=True)
    else:
        eng = exactkv.Engine(m, 2, 64, backend="bf16", graph=False, layer_kernels=True)
    gone = [weakref.ref(eng), weakref.ref(eng.kv[0][0])]
    gc.disable()
    try:
        del eng
        assert [r() for r in gone] == [None, None]
    finally:
        gc.enable()


@pytest.mark.gpu
@pytest.mark.parametrize("paged", [False, True])
def test_engines_that_went_while_another_captures(paged):
    """Engines with captured steps in cycles, nobody's any more, and so many objects made during a capture that the collector,
    did it not rest, would run there and find them."""
    from tests.test_gpu_engine_layers import _ids, _model
    m = _model("llama")
    ids = _ids(2, 30)
    gone = []

    def run(made):
        if paged:
            eng = exactkv.PagedEngine(m, 2, 64, layer_kernels=True)
            eng.add_many(list(ids[:, :20]))
        else:
            eng = exactkv.Engine(m, 2, 64, layer_kernels=True)
            eng.prefill(ids[:, :20])
        forward, seen = eng._forward, []

        def with_objects(*args, **kw):
            seen.append(torch.cuda.is_current_stream_capturing())
            held = [[i] for i in range(made if seen[-1] else 0)]
            assert not held or all(r() is not None for r in gone)
            return forward(*args, **kw)
        eng._forward = with_objects                    # (and a cycle: only the collector finds this engine)
        out = torch.stack([eng.step(ids[:, t]) for t in range(20, 30)])
        assert eng.captures == 1 and seen == [False, True]
        return eng, out
    was = gc.get_threshold()
    gc.collect()
    try:
        gc.disable()
        want = None
        for _ in range(3):
            eng, out = run(0)
            gone.append(weakref.ref(eng))
            del eng
            assert want is None or same_bits(out, want)
            want = out
        assert all(r() is not None for r in gone)
        gc.set_threshold(100000)
        gc.enable()
        assert same_bits(run(200000)[1], want)
        gc.collect()
        assert all(r() is None for r in gone)
    finally:
        gc.set_threshold(*was)
        gc.enable()
