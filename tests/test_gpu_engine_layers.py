"""The engines with layer_kernels: prompts packed through prompt attention, decode steps with the
rotation, appends and norms of this package -- the operators together, as they are used.

  * the compressed and the bf16 cache still give the same tokens and the same bits;
  * logits against the same model in 64 bits: a layer rounds about 14 times on its way to bf16
    (norm, q, k, v, rotations, weights and output of the attention, projection, stream, norm, gate,
    up, product, down, stream), each at most 2^-8 of what it rounds, so two layers and the head
    stay within 30 x 2^-8 = 0.12 in the 2-norm if nothing amplifies, and the engine's own module
    walk, which rounds more often, is held to the same;
  * a captured step equals an eager one, bit for bit, over page ends;
  * PagedEngine.add_many equals adding one by one, to those roundings.

No counterpart in the reference (engine.py:42-95 leaves all of it to the model's modules)."""
import copy

import pytest
import torch

import exactkv_amd as exactkv

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOUND = 30 * 2.0 ** -8


def _model(kind, window=0):
    from transformers import (LlamaConfig, LlamaForCausalLM, Qwen2Config, Qwen2ForCausalLM, Qwen3Config,
                              Qwen3ForCausalLM)
    common = dict(vocab_size=1024, hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4,
                  num_key_value_heads=2, max_position_embeddings=4096, attn_implementation="eager")
    if window:
        common.update(use_sliding_window=True, sliding_window=window, max_window_layers=1)
    cfg, cls = {"llama": (LlamaConfig, LlamaForCausalLM), "qwen2": (Qwen2Config, Qwen2ForCausalLM),
                "qwen3": (Qwen3Config, Qwen3ForCausalLM)}[kind]
    if kind == "qwen3":
        common["head_dim"] = 128
    torch.manual_seed(0)
    m = cls(cfg(**common)).eval()
    for name, p in m.named_parameters():               # norms and biases that are not ones and zeros
        if "norm" in name or name.endswith("bias"):
            p.data.add_(0.1 * torch.randn_like(p))
    return m.to(DEV).to(torch.bfloat16)


def _exact_logits(m, ids):
    """Logits of every position of ids [B, T] in 64 bits, of the bf16 weights."""
    with torch.no_grad():
        return copy.deepcopy(m).double()(ids).logits


def _far(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


def _ids(B, T, seed=1):
    return torch.randint(0, 1024, (B, T), generator=torch.Generator().manual_seed(seed)).to(DEV)


def _teacher(eng, ids, T):
    """Step logits [B, len - T, vocab] with ids' own tokens fed."""
    eng.prefill(ids[:, :T])
    out = [eng.step(ids[:, t]) for t in range(T, ids.shape[1])]
    return torch.stack(out, dim=1)


@pytest.mark.parametrize("kind,window", [("llama", 0), ("qwen2", 0), ("qwen3", 0), ("qwen2", 24)])
def test_logits_against_64_bits_and_across_caches(kind, window):
    m, B, T, N = _model(kind, window), 3, 37, 30
    ids = _ids(B, T + N)
    print("[case]", kind, window, flush=True)
    exact = _exact_logits(m, ids)[:, T:]
    got = {}
    for backend in ("bf16", "exactkv"):
        for own in (False, True):
            eng = exactkv.Engine(m, B, T + N, backend=backend, layer_kernels=own)
            got[backend, own] = _teacher(eng, ids, T)
    assert torch.equal(got["bf16", True].view(torch.int16), got["exactkv", True].view(torch.int16))
    far = {own: _far(got["exactkv", own], exact) for own in (False, True)}
    print("[far]", far, flush=True)
    assert far[True] <= BOUND and far[False] <= BOUND


def test_generate_and_the_prefill_token():
    m, B, T, N = _model("llama"), 2, 50, 20
    toks = {}
    for backend in ("bf16", "exactkv"):
        eng = exactkv.Engine(m, B, T + N, backend=backend, layer_kernels=True)
        toks[backend], logits = eng.generate(_ids(B, T), N)
        assert torch.isfinite(logits.float()).all() and eng.captures >= 1
    assert torch.equal(toks["bf16"], toks["exactkv"])


def test_prompts_in_several_passes(monkeypatch):
    """Prompts that one pass does not take are walked in several, with the same cache contents to
    the projections' rounding."""
    from exactkv_amd import engine
    m, B, T = _model("llama"), 5, 33
    ids = _ids(B, T)
    k = []
    for pack in (16384, 70, 1):
        monkeypatch.setattr(engine._LayerKernels, "PACK", pack)
        eng = exactkv.Engine(m, B, 64, backend="bf16", layer_kernels=True)
        eng.prefill(ids)
        k.append(eng.kv[1][0].buf[:, :T].clone())
    for other in k[1:]:
        assert _far(other, k[0].double()) <= BOUND


@pytest.mark.parametrize("backend", ["bf16", "exactkv"])
def test_graph_equals_eager(backend):
    m, B, T, N = _model("qwen3"), 3, 30, 24
    ids = _ids(B, T + N)
    a = _teacher(exactkv.Engine(m, B, T + N, backend=backend, layer_kernels=True), ids, T)
    b = _teacher(exactkv.Engine(m, B, T + N, backend=backend, layer_kernels=True, graph=False), ids, T)
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("backend", ["bf16", "exactkv"])
@pytest.mark.parametrize("own", [False, True])
def test_add_many(backend, own):
    m = _model("qwen2")
    lens = [20, 1, 47, 16, 31]
    seqs = [_ids(1, n + 12, seed=n)[0] for n in lens]
    eng = exactkv.PagedEngine(m, 8, 96, backend=backend, layer_kernels=own)
    one = exactkv.PagedEngine(m, 8, 96, backend=backend, layer_kernels=own)
    slots, toks = eng.add_many([s[:n] for s, n in zip(seqs, lens)])
    assert slots == [0, 1, 2, 3, 4] and toks.shape == (5,)
    assert [eng.table.length(s) for s in slots] == lens
    for s, n in zip(seqs, lens):
        one.add(s[:n])
    exact = [_exact_logits(m, s[None])[0] for s in seqs]
    for i in range(12):
        tok = torch.stack([s[n + i] for s, n in zip(seqs, lens)])
        got, other = eng.step(tok), one.step(tok)
        want = torch.stack([e[n + i] for e, n in zip(exact, lens)])
        assert _far(got, want) <= BOUND and _far(other, want) <= BOUND
    eng.release(2)
    (again,), _ = eng.add_many([seqs[0]])
    assert again == 2
    got = eng.step(torch.stack([s[-1] for s in seqs]), [0, 1, 3, 4, 2])
    assert torch.isfinite(got.float()).all()


def test_add_many_adds_all_or_none():
    m = _model("llama")
    eng = exactkv.PagedEngine(m, 4, 64, num_pages=6)
    free = eng.table.free_pages()
    with pytest.raises(RuntimeError, match="exhausted"):
        eng.add_many([_ids(1, 30)[0], _ids(1, 30)[0], _ids(1, 60)[0]])
    assert eng.table.free_pages() == free and eng.table.live_slots() == []
    with pytest.raises(ValueError):
        eng.add_many([_ids(1, 70)[0]])
    with pytest.raises(ValueError):
        eng.add_many([_ids(1, 5)[0], _ids(1, 5)[0][:0]])
    assert eng.table.live_slots() == []


def test_prompts_that_the_model_refuses_leave_no_slot():
    eng = exactkv.PagedEngine(_model("llama"), 4, 64, layer_kernels=True)
    free = eng.table.free_pages()
    with pytest.raises(RuntimeError):
        eng.add_many([_ids(1, 30)[0].cpu(), _ids(1, 20)[0].cpu()])
    with pytest.raises(RuntimeError):
        eng.add(_ids(1, 30)[0].cpu())
    assert eng.table.free_pages() == free and eng.table.live_slots() == []
    slot, tok = eng.add(_ids(1, 30)[0])
    (again,), (tok2,) = eng.add_many([_ids(1, 30)[0]])
    assert tok == tok2 and eng.table.live_slots() == sorted([slot, again])


def test_engines_refuse_what_the_kernels_do_not_do():
    m = _model("llama")
    with pytest.raises(AssertionError, match="bf16"):
        exactkv.Engine(copy.deepcopy(m).float(), 1, 64, layer_kernels=True)
    other = copy.deepcopy(m)
    other.model.rotary_emb.rope_type = "dynamic"
    with pytest.raises(AssertionError, match="tables"):
        exactkv.Engine(other, 1, 64, layer_kernels=True)
    with pytest.raises(AssertionError, match="fit"):
        exactkv.Engine(m, 1, 64, layer_kernels=True).prefill(_ids(2, 5))
