"""Batched greedy decoding for Hugging Face Llama-3 / Qwen2 / Qwen2.5 / Qwen3 models over
the compressed (or bf16) KV cache -- drop-in for the reference's exactkv/engine.py:18-95.

The model's own weights and modules are used; only the KV cache and decode attention
are replaced, so two engines that differ only in the cache produce identical tokens and
logits wherever the cache is lossless (here: always, bit for bit).

MI355X specifics:
  * a decode step depends on no host value: the position comes from the cache's device
    token count, appends read it there, and attention gets it through `lens`. The first
    decode step runs eagerly on the engine's stream (it sets up BLAS handles and the
    attention workspaces there); the next one is captured in a HIP graph, and every
    later step replays it. A pool growth at a page boundary changes the raw-pool
    buffers, so the graph is captured again on the next step;
  * prefill runs one sequence at a time through the model's own forward pass, with SDPA
    restricted to its fused (flash / memory-efficient) kernels;
  * layer_kernels=True (PagedEngine.add_many: always) walks the layers here instead, with this
    package's kernels between the model's projections: rotation and appends in one launch, each
    residual add with the norm behind it in one, and prompts packed, several sequences in one
    pass of prompt attention. It rounds less often than the model's modules (once per kernel),
    so its logits are near theirs, not their bits; the two caches agree bit for bit either way.
"""
import importlib

import torch

from .cache import BF16KV, CompressedKV, check_overflow
from .attention import decode_attention
from .kernels import HEAD_DIMS, attention_compressed, attention_reference, P
from .layer import add_norm, launch_rope_append, prompt_attention, rope_append, rotate_prompt

BACKENDS = {"exactkv": CompressedKV, "bf16": BF16KV}


def _fused_sdpa():
    """Context restricting scaled_dot_product_attention to its fused kernels (it raises
    instead of falling back to the unfused math path)."""
    from torch.nn.attention import SDPBackend, sdpa_kernel
    return sdpa_kernel([SDPBackend.FLASH_ATTENTION, SDPBackend.EFFICIENT_ATTENTION])


_WRITE_THROUGH = None
_FAMILIES = ("llama", "qwen2", "qwen3")


def _describe(engine, model):
    """Set the attention geometry the engines need from a Hugging Face decoder: layers, query
    and KV heads, head dim, the family's RoPE helper, whether keys and queries are normed
    (Qwen3), and each layer's sliding window (0: full attention). Qwen2/Qwen3 mark sliding
    layers with use_sliding_window / sliding_window / layer_types (the reference rejects
    them, engine.py:26-28)."""
    cfg = model.config
    if cfg.model_type not in _FAMILIES:
        raise AssertionError(f"model family {cfg.model_type!r} is not one of {_FAMILIES}")
    attn0 = model.model.layers[0].self_attn
    engine.m = model
    engine.L = cfg.num_hidden_layers
    engine.Hq, engine.Hkv = cfg.num_attention_heads, cfg.num_key_value_heads
    engine.D = getattr(cfg, "head_dim", None) or cfg.hidden_size // cfg.num_attention_heads
    if engine.D not in HEAD_DIMS:       # the reference asserts 128 (engine.py:28)
        raise AssertionError(f"the kernels store head dims {HEAD_DIMS} (the model has {engine.D})")
    engine.rope = getattr(importlib.import_module(type(attn0).__module__), "apply_rotary_pos_emb")
    engine.qk_norm = hasattr(attn0, "k_norm")
    window = int(getattr(cfg, "sliding_window", 0) or 0) if getattr(cfg, "use_sliding_window", False) else 0
    kinds = getattr(cfg, "layer_types", None) or ()     # no per-layer list: no sliding layer
    engine.windows = [window if i < len(kinds) and kinds[i] == "sliding_attention" else 0
                      for i in range(engine.L)]
    engine.dev = next(model.parameters()).device


def _project(eng, att, x, B, cos, sin):
    """One token's q [B, Hq, 1, D] (RoPE'd), k [B, Hkv, 1, D] (RoPE'd) and v [B, 1, Hkv, D]
    through the model's own attention projections (Qwen3: with its q/k norms)."""
    q = att.q_proj(x).view(B, 1, eng.Hq, eng.D)
    k = att.k_proj(x).view(B, 1, eng.Hkv, eng.D)
    v = att.v_proj(x).view(B, 1, eng.Hkv, eng.D)
    if eng.qk_norm:
        q, k = att.q_norm(q), att.k_norm(k)
    q, k = eng.rope(q.transpose(1, 2), k.transpose(1, 2), cos, sin)
    return q, k, v


class _LayerKernels:
    """A decoder's layers with this package's kernels between its projections."""

    PACK = 16384                                # prompt tokens of one pass

    def __init__(self, eng, positions):
        m = eng.m.model
        kind = getattr(m.rotary_emb, "rope_type", "default")
        if kind in ("dynamic", "longrope"):
            raise AssertionError(f"layer kernels take fixed rotary tables (the model's are {kind!r})")
        if next(m.parameters()).dtype != torch.bfloat16:
            raise AssertionError("layer kernels take a bf16 model")
        self.eng = eng
        # the model's own tables, in fp32
        like = torch.zeros(1, dtype=torch.float32, device=eng.dev)
        cos, sin = m.rotary_emb(like, torch.arange(positions, device=eng.dev)[None])
        half = eng.D // 2
        if cos.shape[-1] != eng.D or not torch.equal(cos[..., :half], cos[..., half:]):
            raise AssertionError("layer kernels rotate half-split over the whole head")
        self.cos, self.sin = (t[0, :, :half].float().contiguous() for t in (cos, sin))

    def _norm(self, x, residual, norm):
        return add_norm(x, residual, norm.weight, eps=norm.variance_epsilon)

    def _head_norms(self, att):
        if not self.eng.qk_norm:
            return {}
        return dict(q_norm=att.q_norm.weight, k_norm=att.k_norm.weight, eps=att.q_norm.variance_epsilon)

    def _walk(self, tok, attend):
        """tok: token ids [n]; attend(i, q, k, v, norms) gives layer i's attention [n, Hq, D] from
        its projections. Returns the normed hidden state [n, C]."""
        eng, m = self.eng, self.eng.m.model
        n = tok.shape[0]
        h, x = self._norm(m.embed_tokens(tok), None, m.layers[0].input_layernorm)
        for i, layer in enumerate(m.layers):
            att = layer.self_attn
            q = att.q_proj(x).view(n, eng.Hq, eng.D)
            k = att.k_proj(x).view(n, eng.Hkv, eng.D)
            v = att.v_proj(x).view(n, eng.Hkv, eng.D)
            o = attend(i, q, k, v, self._head_norms(att))
            h, x = self._norm(att.o_proj(o.view(n, eng.Hq * eng.D)), h, layer.post_attention_layernorm)
            after = m.layers[i + 1].input_layernorm if i + 1 < eng.L else m.norm
            h, x = self._norm(layer.mlp(x), h, after)
        return x

    def step(self, tok, attend, device_only):
        """Logits of one decode step: attend(i, q) over layer i's caches, its token appended."""
        append = launch_rope_append if device_only else rope_append

        def layer(i, q, k, v, norms):
            return attend(i, append(q, k, v, self.cos, self.sin, *self.eng.kv[i], **norms))
        return self.eng.m.lm_head(self._walk(tok, layer))

    def prompts(self, prompts, slots):
        """Prompts (1-D token ids) into the caches' slots, packed: the normed hidden state of each
        prompt's last token [len(prompts), C]."""
        eng, last, i = self.eng, [], 0
        while i < len(prompts):
            j, total = i, 0                        # as many as one pass takes, one at least
            while j < len(prompts) and (j == i or total + prompts[j].numel() <= self.PACK):
                total += prompts[j].numel()
                j += 1
            ends = [0]
            for p in prompts[i:j]:
                ends.append(ends[-1] + p.numel())
            cu = torch.tensor(ends, dtype=torch.int32).to(eng.dev)

            def layer(li, q, k, v, norms):
                q, k = rotate_prompt(q, k, self.cos, self.sin, cu, **norms)
                kc, vc = eng.kv[li]
                for slot, a, e in zip(slots[i:j], ends, ends[1:]):
                    kc.prefill_slot(slot, k[None, a:e])
                    vc.prefill_slot(slot, v[None, a:e])
                return prompt_attention(q, k, v, cu, window=eng.windows[li])
            x = self._walk(torch.cat([p.reshape(-1) for p in prompts[i:j]]), layer)
            last.append(x[torch.tensor(ends[1:]).to(eng.dev) - 1])
            i = j
        return torch.cat(last)


def _write_through(engine, b):
    """A prefill-only transformers cache whose update() encodes the layer's keys and values
    into sequence slot b of the engine's caches and keeps nothing, so the model's forward
    pass holds one layer's K/V at a time. Its layer list stays empty: the model reads a
    sequence length of 0 and masks for the prompt alone, as for a fresh DynamicCache."""
    global _WRITE_THROUGH
    if _WRITE_THROUGH is None:
        from transformers.cache_utils import DynamicCache

        class WriteThrough(DynamicCache):
            def __init__(self, eng, slot):
                super().__init__()
                self.eng, self.slot = eng, slot

            def update(self, key_states, value_states, layer_idx, *args, **kwargs):
                kc, vc = self.eng.kv[layer_idx]
                kc.prefill_slot(self.slot, key_states.transpose(1, 2))     # [1, T, H, D] view, no copy
                vc.prefill_slot(self.slot, value_states.transpose(1, 2))
                return key_states, value_states

        _WRITE_THROUGH = WriteThrough
    return _WRITE_THROUGH(engine, b)


def _layer_kv(pkv, i):
    """Layer i's keys and values [1, H, T, D] from a transformers cache (its layers list, or
    the key_cache / value_cache lists of older versions)."""
    layers = getattr(pkv, "layers", None)
    if layers is not None:
        return layers[i].keys, layers[i].values
    return pkv.key_cache[i], pkv.value_cache[i]


class Engine:
    def __init__(self, model, B, T_max, backend="exactkv", attn=None, before_step=None, graph=True,
                 layer_kernels=False):
        """backend: 'exactkv' / 'bf16', or a cache class with the same interface.
        attn(q, k_cache, v_cache) and before_step(engine, T) let benchmarks plug in other
        kernels (reference engine.py:30-33); with either plug-in the step runs eagerly.
        graph: capture the decode step in a HIP graph (default).
        layer_kernels: rotation, norms and prompt attention by this package's kernels (its own
        caches only)."""
        # sliding-window layers: decode attention reads each sequence's last `window` tokens,
        # the keys the model's own mask admits (positions > p - window)
        _describe(self, model)
        assert attn is None or not any(self.windows), "attention plug-ins do not take a sliding window"
        self.B, self.TS = B, -(-T_max // P) * P
        cls = BACKENDS.get(backend, backend)
        kw = {"device": self.dev} if isinstance(cls, type) and issubclass(cls, (CompressedKV, BF16KV)) else {}
        self.kv = [(cls(B, self.TS, self.Hkv, self.D, **kw), cls(B, self.TS, self.Hkv, self.D, **kw))
                   for _ in range(self.L)]
        self.attn = attn
        self.before_step = before_step
        self.grows = 0
        ours = isinstance(cls, type) and issubclass(cls, (CompressedKV, BF16KV))
        if layer_kernels and not ours:
            raise AssertionError("layer kernels append to this package's caches only")
        self._layers = _LayerKernels(self, self.TS) if layer_kernels else None
        self.use_graph = bool(graph) and attn is None and before_step is None and ours
        self._stream = torch.cuda.Stream(device=self.dev) if self.use_graph else None
        self._graph = None
        self._graph_key = None
        self.captures = 0                       # HIP-graph captures of the decode step
        self._warm = False
        self._tok = torch.zeros(B, dtype=torch.long, device=self.dev)
        self._pos = torch.zeros(1, 1, dtype=torch.long, device=self.dev)
        self._logits = None

    # ---------------------------------------------------------------- prefill
    @torch.no_grad()
    def prefill(self, ids, b0=0, fused=True):
        """ids: [B, T] token ids. Returns the greedy next token of each sequence, [B].
        b0 (additive): fill sequence slots b0.. with ids' rows, so a long prefill can be
        done in pieces (slot 0 first).
        fused (additive): each layer's RoPE'd keys and values go straight from the
        attention module into the page encoder, read in place through strides ([1, H, T, D]
        as a [1, T, H, D] view), so the model's DynamicCache never holds the prompt's K/V
        (reference engine.py:42-49 builds it, then cache.py:87-98 copies each layer out of
        it). fused=False keeps that order (the K/V of all layers live until the forward
        pass ends); both give the same cache bytes.
        With layer_kernels the prompts go through packed, several at a time (fused is not used)."""
        if self._layers is not None:
            if ids.shape[1] == 0 or b0 + ids.shape[0] > self.B or ids.shape[1] > self.TS:
                raise AssertionError(f"{ids.shape[0]} prompts of {ids.shape[1]} tokens do not fit slots {b0} to {self.B - 1} "
                                     f"of {self.TS}")
            hidden = self._layers.prompts(list(ids), list(range(b0, b0 + ids.shape[0])))
            self._graph = None                  # buffers may have grown
            return self._prefill_next(hidden[:, None])
        nxt = []
        with _fused_sdpa():
            for i0 in range(ids.shape[0]):
                b = b0 + i0
                if fused:
                    out = self.m.model(ids[i0:i0 + 1], use_cache=True, past_key_values=_write_through(self, b))
                else:
                    out = self.m.model(ids[i0:i0 + 1], use_cache=True)
                    pkv = out.past_key_values
                    for i, (kc, vc) in enumerate(self.kv):
                        keys, values = _layer_kv(pkv, i)             # [1, H, T, D] each
                        kc.prefill_slot(b, keys.transpose(1, 2))
                        vc.prefill_slot(b, values.transpose(1, 2))
                    del pkv
                nxt.append(self._prefill_next(out.last_hidden_state))
                del out
        self._graph = None                      # buffers may have grown
        return torch.cat(nxt)

    def _prefill_next(self, hidden):
        """Greedy next token from the prompt's last hidden state. The final norm is applied
        to the model's output once more, as the reference prefill does (engine.py:50), so
        both backends and the reference pick the same first token."""
        last = self.m.model.norm(hidden[:, -1])
        return self.m.lm_head(last).argmax(dim=-1)

    def _caches(self):
        return [c for pair in self.kv for c in pair]

    # ---------------------------------------------------------------- decode step
    def _attend(self, q, kc, vc, window=0):
        if self.attn is not None:
            return self.attn(q, kc, vc)
        lens = kc.state[:1]                     # token count on the device (after this step's append)
        if isinstance(kc, CompressedKV):
            return attention_compressed(q, kc, vc, kc.TS, lens=lens, window=window)
        return attention_reference(q, kc.buf, vc.buf, kc.TS, lens=lens, window=window)

    def _forward(self, tok, device_only):
        """One decode step: tok [B] -> logits [B, vocab]. device_only: appends launch their
        kernels only (the host counts advance after the step), so the step reads no host
        state that changes between steps and can be captured; otherwise each append also
        advances its cache's host count, as the reference does, so an attention plug-in
        sees the current length."""
        m, B, Hq, Hkv, D = self.m, self.B, self.Hq, self.Hkv, self.D
        if self._layers is not None:
            return self._layers.step(tok, lambda i, q: self._attend(q, *self.kv[i], self.windows[i]), device_only)
        h = m.model.embed_tokens(tok.view(B, 1))
        self._pos.copy_(self.kv[0][0].state[:1].view(1, 1))                 # position = tokens so far
        cos, sin = m.model.rotary_emb(h, self._pos)
        for i, layer in enumerate(m.model.layers):
            att = layer.self_attn
            q, k, v = _project(self, att, layer.input_layernorm(h), B, cos, sin)
            kc, vc = self.kv[i]
            if device_only:
                kc._check_token(k[:, :, 0])
                vc._check_token(v[:, 0])
                kc._launch_append(k[:, :, 0])
                vc._launch_append(v[:, 0])
            else:
                kc.append(k[:, :, 0])
                vc.append(v[:, 0])
            o = self._attend(q[:, :, 0].contiguous(), kc, vc, self.windows[i])
            h = h + att.o_proj(o.reshape(B, 1, Hq * D))
            h = h + layer.mlp(layer.post_attention_layernorm(h))
        return m.lm_head(m.model.norm(h))[:, 0]

    def _buffers_key(self):
        """What a captured step depends on beyond its inputs: every raw pool's address and
        size, and the tail offset (cap) its launches were recorded with. A pool can grow twice
        between steps and land at its old address, so the address alone does not identify it."""
        return tuple((c.raw.data_ptr(), c.cap, c.raw.shape[0]) for kv in self.kv for c in kv
                     if isinstance(c, CompressedKV))

    def _advance(self):
        for kv in self.kv:
            for c in kv:
                c._advance()

    @torch.no_grad()
    def step(self, tok):
        """tok: [B] current tokens. Returns logits [B, vocab] (bf16) for the next token."""
        T = self.kv[0][0].T
        if self.use_graph:
            for kv in self.kv:
                for c in kv:
                    c._check_can_append()
        if self.before_step:
            self.before_step(self, T + 1)
        if not self.use_graph:
            logits = self._forward(tok, device_only=False)
        else:
            cur = torch.cuda.current_stream(self.dev)
            self._stream.wait_stream(cur)
            with torch.cuda.stream(self._stream):
                self._tok.copy_(tok)
                if not self._warm:                       # first step: eager, on the graph's stream
                    logits = self._forward(self._tok, device_only=True)
                    self._warm = True
                else:
                    key = self._buffers_key()
                    if self._graph is None or key != self._graph_key:
                        self._graph = torch.cuda.CUDAGraph()
                        with torch.cuda.graph(self._graph, stream=self._stream):
                            self._logits = self._forward(self._tok, device_only=True)
                        self._graph_key = key
                        self.captures += 1
                    self._graph.replay()
                    logits = self._logits.clone()
            cur.wait_stream(self._stream)
            self._advance()
        if (T + 1) % P == 0:                   # a page filled in every cache: one counter read
            self.grows += check_overflow(self._caches())
        return logits

    @torch.no_grad()
    def generate(self, ids, n_new):
        """Greedy decoding of n_new tokens per sequence, the first from the prefill: returns
        (tokens [B, n_new], the logits of the n_new - 1 decode steps [B, n_new - 1, vocab])."""
        tokens = [self.prefill(ids)]
        step_logits = []
        while len(tokens) < n_new:
            step_logits.append(self.step(tokens[-1]))
            tokens.append(step_logits[-1].argmax(dim=-1))
        return torch.stack(tokens, dim=1), torch.stack(step_logits, dim=1)

    def kv_bytes(self):
        """Device bytes held by every layer's K and V caches."""
        total = 0
        for kc, vc in self.kv:
            total += kc.nbytes() + vc.nbytes()
        return total


class PagedEngine:
    """Greedy decoding over paged caches: sequences of different lengths share one pool of
    16-token pages through a PageTable, join with add() and leave with release().

    No counterpart in the reference, whose engine keeps every sequence at one length in
    contiguous caches (engine.py:18-95); paged KV is its future work (README.md:121-123).
    The model, projections, write-through prefill and sliding-window handling are the
    Engine's. Steps run eagerly: the block table and lengths change on the host between
    steps (begin_step claims a page whenever a token fills one)."""

    def __init__(self, model, max_seqs, T_max, backend="exactkv", num_pages=None, graph=True, layer_kernels=False):
        """graph: replay the step from a HIP graph when the step's slots are 0..n-1 (default);
        the graph is captured again when n or a raw pool's buffer changes.
        layer_kernels: steps and add() by this package's kernels around the projections, as in
        Engine (add_many always)."""
        from .paged import PageTable, PagedBF16KV, PagedCompressedKV
        _describe(self, model)
        max_pages = -(-T_max // P)
        self.table = PageTable(num_pages or max_seqs * max_pages, max_seqs, max_pages, device=self.dev)
        cls = {"exactkv": PagedCompressedKV, "bf16": PagedBF16KV}[backend]
        self.kv = [(cls(self.table, self.Hkv, D=self.D), cls(self.table, self.Hkv, D=self.D)) for _ in range(self.L)]
        self.grows = 0
        self.use_graph = bool(graph)
        self._stream = torch.cuda.Stream(device=self.dev) if self.use_graph else None
        self._graph, self._graph_key, self._warm = None, None, set()
        self._tok = torch.zeros(max_seqs, dtype=torch.long, device=self.dev)
        self._logits = None
        self.captures = 0
        self._positions = P * max_pages
        self._own_layers = bool(layer_kernels)
        self._layers = _LayerKernels(self, self._positions) if layer_kernels else None

    @torch.no_grad()
    def add_many(self, prompts):
        """Prefill several prompts (1-D token ids of any lengths) into new sequence slots, packed:
        one pass over the model's layers for about 16K tokens of them. Returns (slots, the greedy
        next tokens [len(prompts)]). Where a prompt does not fit, or the model refuses one, none is added."""
        if self._layers is None:
            self._layers = _LayerKernels(self, self._positions)
        prompts = list(prompts)
        if not prompts or any(p.numel() == 0 for p in prompts):
            raise ValueError("add_many takes one or more prompts of at least one token")
        slots = []
        try:
            for p in prompts:
                slots.append(self.table.add(int(p.numel())))
            hidden = self._layers.prompts(prompts, slots)
        except Exception:                       # no room, or no prompts the model takes
            for s in slots:
                self.table.release(s)
            raise
        return slots, self.m.lm_head(self.m.model.norm(hidden)).argmax(-1)

    @torch.no_grad()
    def add(self, ids, slot=None):
        """Prefill one prompt (1-D token ids) into a new sequence slot. Returns (slot, the
        greedy next token)."""
        if self._own_layers:
            if ids.numel() == 0:
                raise ValueError("a prompt of no tokens")
            s = self.table.add(int(ids.numel()), slot)
            try:
                hidden = self._layers.prompts([ids.view(-1)], [s])
            except Exception:
                self.table.release(s)
                raise
            return s, self.m.lm_head(self.m.model.norm(hidden)).argmax(-1)[0]
        s = self.table.add(int(ids.numel()), slot)
        with _fused_sdpa():
            out = self.m.model(ids.view(1, -1), use_cache=True, past_key_values=_write_through(self, s))
        return s, self.m.lm_head(self.m.model.norm(out.last_hidden_state[:, -1])).argmax(-1)[0]

    def release(self, slot):
        self.table.release(slot)

    def _forward(self, tok, n):
        """The step's kernels for n rows (appends, attention, the model): no host state."""
        m = self.m
        if self._own_layers:
            return self._layers.step(tok, lambda i, q: decode_attention(q, *self.kv[i], window=self.windows[i]), True)
        _, _, lens = self.table.step_rows()
        pos = (lens - 1).view(n, 1).long()                                   # each sequence's position
        h = m.model.embed_tokens(tok.view(n, 1))
        cos, sin = m.model.rotary_emb(h, pos)
        for i, layer in enumerate(m.model.layers):
            att = layer.self_attn
            q, k, v = _project(self, att, layer.input_layernorm(h), n, cos, sin)
            kc, vc = self.kv[i]
            kc._launch_append(k[:, :, 0])
            vc._launch_append(v[:, 0])
            o = decode_attention(q[:, :, 0].contiguous(), kc, vc, window=self.windows[i])
            h = h + att.o_proj(o.reshape(n, 1, self.Hq * self.D))
            h = h + layer.mlp(layer.post_attention_layernorm(h))
        return m.lm_head(m.model.norm(h))[:, 0]

    @torch.no_grad()
    def step(self, tok, slots=None):
        """tok: [n] the current token of each slot in `slots` (default: every live slot, in
        order). Returns logits [n, vocab] for their next tokens."""
        slots = self.table.begin_step(slots)
        n = len(slots)
        caches = [c for kv in self.kv for c in kv]
        for c in caches:
            c._check_append((n, self.Hkv, self.D))
        dense = self.table.step_rows()[0] is None
        if not (self.use_graph and dense):
            logits = self._forward(tok, n)
        else:
            cur = torch.cuda.current_stream(self.dev)
            self._stream.wait_stream(cur)
            with torch.cuda.stream(self._stream):
                self._tok[:n].copy_(tok)
                key = (n, tuple((c.raw.data_ptr(), c.cap, c.raw.shape[0]) for c in caches if hasattr(c, "raw")))
                if n not in self._warm:                  # first step at this n: eager, on the graph's stream
                    logits = self._forward(self._tok[:n], n)
                    self._warm.add(n)
                else:
                    if self._graph is None or key != self._graph_key:
                        self._graph = torch.cuda.CUDAGraph()
                        with torch.cuda.graph(self._graph, stream=self._stream):
                            self._logits = self._forward(self._tok[:n], n)
                        self._graph_key = key
                        self.captures += 1
                    self._graph.replay()
                    logits = self._logits.clone()
            cur.wait_stream(self._stream)
        for c in caches:
            c._advance()
        if self.table.filled_in_step():
            self.grows += check_overflow(caches)
        return logits

    def kv_bytes(self):
        """Device bytes held by every layer's paged K and V caches."""
        total = 0
        for kc, vc in self.kv:
            total += kc.nbytes() + vc.nbytes()
        return total
