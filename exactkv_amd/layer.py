"""What a decoder layer does around its caches: attention of whole prompts, the rotation on the
way into the caches, and the residual stream with its norms.

  prompt_attention    causal attention of packed prompts (the prefill counterpart of
                      decode_attention)
  rotate_prompt       a packed prompt's queries and keys rotated at their positions
  rope_append         a decode step's queries rotated, keys rotated and appended, values
                      appended, in one launch, into whichever caches hold them
  rope_append_paged   the same on plain tensors: bf16 pools or a compressed cache's arrays
  add_norm            a block's output onto the residual stream, and the next block's norm

No counterpart in the reference, whose engine leaves all of this to the model's own modules
(exactkv/engine.py:42-49,75-91). Everything is bf16 in and out and fp32 inside, rounded once.
The tensors of a call are on one GPU; the work goes to that GPU's current stream, allocates
nothing but the outputs, waits for nothing, and can be captured in a HIP graph.
"""
import torch

from . import _lib
from .cache import BF16KV, CompressedKV
from .kernels import HEAD_DIMS, P, _QK_SCALE
from .paged import PagedBF16KV, PagedCompressedKV

BF16 = torch.bfloat16


def _rows(t, what):
    """(tokens, heads, D, token stride, head stride) of bf16 rows [n, H, D] on the GPU."""
    if t.dim() != 3 or t.dtype != BF16 or not t.is_cuda:
        raise ValueError(f"{what} must be a bf16 [tokens, heads, D] GPU tensor")
    n, H, D = t.shape
    s_t, s_h, s_d = t.stride()
    if s_d != 1 and D > 1:
        raise ValueError(f"{what}: rows (the last axis) must be contiguous")
    return n, H, D, (s_t if n > 1 else H * D), (s_h if H > 1 else D)


def _check_heads(Hq, Hkv, D):
    if D not in HEAD_DIMS:
        raise ValueError(f"head dim must be one of {HEAD_DIMS} (got {D})")
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads do not divide over {Hkv} KV heads")


def _offsets(cu, what):
    if cu.dtype != torch.int32 or cu.dim() != 1 or cu.numel() < 1 or not cu.is_cuda or not cu.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 [sequences + 1] GPU tensor")
    return cu.numel() - 1


def _one_device(dev, *tensors):
    for t in tensors:
        if t is not None and t.device != dev:
            raise ValueError(f"all tensors of a call must be on {dev} (got one on {t.device})")


def _vector(w, n, what):
    """Pointer of a bf16 [n] weight, or None."""
    if w is None:
        return None
    if w.dtype != BF16 or w.shape != (n,) or not w.is_contiguous():
        raise ValueError(f"{what} must be a contiguous bf16 [{n}] GPU tensor")
    return _lib.ptr(w, 16, what)


def _tables(cos, sin, D):
    """(cos pointer, sin pointer, rows) of fp32 tables [positions, D / 2]."""
    if (cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.dim() != 2 or cos.shape[1] != D // 2
            or cos.shape != sin.shape or cos.shape[0] < 1 or not cos.is_contiguous() or not sin.is_contiguous()):
        raise ValueError(f"cos and sin must be contiguous fp32 [positions, {D // 2}] GPU tensors of one shape")
    return _lib.ptr(cos, 16, "cos"), _lib.ptr(sin, 16, "sin"), cos.shape[0]


def _overlap(a, b):
    """Whether the memory that a and b span meets."""
    def span(t):
        first = t.data_ptr()
        return first, first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _elsewhere(dev):
    """Whether dev is not the current device (calls then make it so: its current stream may be the
    null stream, which is the current device's)."""
    return dev.index != torch.cuda.current_device()


def prompt_attention(q, k, v, cu_seqlens, *, cu_seqlens_k=None, window=0, out=None):
    """Causal attention of packed prompts: q bf16 [N, Hq, D] (D = 64, 128 or 256), k and v bf16
    [N, Hkv, D], rotated already, sequence s in rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1
    (int32 [S + 1] on the GPU, ascending from 0; sequences may be empty). Every query attends to
    its own sequence's keys up to its own token, with window > 0 to the last `window` of those
    (the tokens decode_attention's window admits). Query heads share KV heads in order: head h
    reads KV head h // (Hq / Hkv). Returns bf16 [N, Hq, D].

    cu_seqlens_k: the keys' own offsets into k and v [NK, Hkv, D], where a sequence has more keys
    than queries: its queries are then its last tokens (the next piece of a prompt whose earlier
    keys are held). A query that sees no key (fewer keys than queries) gets 0.

    Keys and values that a query does not attend to never reach it, be they infinite or NaN. q, k
    and v may be strided views (of a fused projection, of [1, H, N, D]): rows contiguous, 16-byte
    aligned. out: a contiguous tensor shaped like q that overlaps no input; its rows behind the
    last sequence are left as they were (without out they are 0)."""
    N, Hq, D, sq_t, sq_h = _rows(q, "q")
    NK, Hkv, Dk, sk_t, sk_h = _rows(k, "k")
    NV, Hv, Dv, sv_t, sv_h = _rows(v, "v")
    _check_heads(Hq, Hkv, D)
    if Dk != D or (NV, Hv, Dv) != (NK, Hkv, D):
        raise ValueError(f"k and v must be of one shape [keys, heads, {D}] (got {tuple(k.shape)}, {tuple(v.shape)})")
    S = _offsets(cu_seqlens, "cu_seqlens")
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens
        if NK != N:
            raise ValueError(f"{NK} keys for {N} queries: give cu_seqlens_k")
    elif _offsets(cu_seqlens_k, "cu_seqlens_k") != S:
        raise ValueError("cu_seqlens and cu_seqlens_k must hold as many sequences")
    window = int(window or 0)
    if window < 0 or window > 0x7FFFFFFF:
        raise ValueError(f"window must be >= 0 (got {window})")
    dev = q.device
    _one_device(dev, k, v, cu_seqlens, cu_seqlens_k, out)
    fresh = out is None
    if fresh:
        out = torch.empty((N, Hq, D), dtype=BF16, device=dev)
    else:
        if out.shape != q.shape or out.dtype != BF16 or not out.is_contiguous():
            raise ValueError("out must be a contiguous bf16 tensor shaped like q")
        if any(_overlap(out, t) for t in (q, k, v)):
            raise ValueError("out overlaps an input")
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            prompt_attention(q, k, v, cu_seqlens, cu_seqlens_k=cu_seqlens_k, window=window, out=out.zero_() if fresh else out)
        return out
    # a call with few rows splits its keys: partial results, this call's own (in a graph: the graph's)
    need = _lib.load().exkv_prompt_workspace(S, N, NK, Hq, Hkv, D, window)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _lib.call("exkv_prompt_attention", q.data_ptr(), sq_t, sq_h, k.data_ptr(), sk_t, sk_h, v.data_ptr(), sv_t, sv_h,
              out.data_ptr(), cu_seqlens.data_ptr(), cu_seqlens_k.data_ptr(), S, N, NK, Hq, Hkv, D, window, int(fresh),
              _QK_SCALE[D], None if ws is None else ws.data_ptr(), need, _lib.stream(dev.index))
    return out


def rotate_prompt(q, k, cos, sin, cu_seqlens, *, start=None, q_norm=None, k_norm=None, eps=1e-6):
    """A packed prompt's queries and keys rotated (half-split rotary embedding): q bf16 [N, Hq, D],
    k bf16 [N, Hkv, D], strided views allowed, sequences as in prompt_attention; token i of
    sequence s stands at position i, or start[s] + i (start: int32 [S] on the GPU), whose row of
    cos and sin (fp32 [positions, D / 2]) turns it. q_norm, k_norm (bf16 [D]): the heads are
    RMS-normed with these weights and eps first (Qwen3). Returns the two, contiguous, ready for
    prompt_attention and the caches' prefill; rows that no sequence holds are 0.

    A position outside the tables is clamped to them and sets an error bit (kernels.check_errors)."""
    N, Hq, D, sq_t, sq_h = _rows(q, "q")
    NK, Hkv, Dk, sk_t, sk_h = _rows(k, "k")
    if D not in HEAD_DIMS or Dk != D or NK != N or Hq == 0 or Hkv == 0:
        raise ValueError(f"q and k must be [N, heads, D] with D in {HEAD_DIMS} (got {tuple(q.shape)}, {tuple(k.shape)})")
    S = _offsets(cu_seqlens, "cu_seqlens")
    dev = q.device
    _one_device(dev, k, cos, sin, cu_seqlens, start, q_norm, k_norm)
    if start is not None and (start.dtype != torch.int32 or start.shape != (S,) or not start.is_contiguous()):
        raise ValueError(f"start must be a contiguous int32 [{S}] GPU tensor")
    cp, sp, rows = _tables(cos, sin, D)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return rotate_prompt(q, k, cos, sin, cu_seqlens, start=start, q_norm=q_norm, k_norm=k_norm, eps=eps)
    qo = torch.empty((N, Hq, D), dtype=BF16, device=dev)
    ko = torch.empty((N, Hkv, D), dtype=BF16, device=dev)
    _lib.call("exkv_rotate_prompt", q.data_ptr(), sq_t, sq_h, k.data_ptr(), sk_t, sk_h, cp, sp, rows,
              _vector(q_norm, D, "q_norm"), _vector(k_norm, D, "k_norm"), eps, qo.data_ptr(), ko.data_ptr(),
              cu_seqlens.data_ptr(), None if start is None else start.data_ptr(), S, N, Hq, Hkv, D, _lib.stream(dev.index))
    return qo, ko


def _token_rows(q, k, v, cos, sin, q_norm, k_norm, eps, out):
    """The rows' arguments of a rotated append, and (out, n, Hkv, D)."""
    n, Hq, D, sq_n, sq_h = _rows(q, "q")
    nk, Hkv, Dk, sk_n, sk_h = _rows(k, "k")
    nv, Hv, Dv, sv_n, sv_h = _rows(v, "v")
    if D not in HEAD_DIMS or (nk, Dk) != (n, D) or (nv, Hv, Dv) != (n, Hkv, D) or Hq == 0 or Hkv == 0:
        raise ValueError(f"q [n, Hq, D], k and v [n, Hkv, D] with D in {HEAD_DIMS} expected (got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)})")
    _one_device(q.device, k, v, cos, sin, q_norm, k_norm, out)
    cp, sp, rows = _tables(cos, sin, D)
    if out is None:
        out = torch.empty((n, Hq, D), dtype=BF16, device=q.device)
    elif out.shape != q.shape or out.dtype != BF16 or not out.is_contiguous():
        raise ValueError("out must be a contiguous bf16 tensor shaped like q")
    elif any(_overlap(out, t) for t in (q, k, v)):
        raise ValueError("out overlaps an input")
    return (q.data_ptr(), sq_n, sq_h, k.data_ptr(), sk_n, sk_h, v.data_ptr(), sv_n, sv_h, cp, sp, rows,
            _vector(q_norm, D, "q_norm"), _vector(k_norm, D, "k_norm"), eps, _lib.ptr(out, 16, "out"), n, Hq, Hkv), out, n, Hkv, D


_ARRAYS = ("sm", "code", "base", "rowmask", "rowoff", "raw")


def _compressed_args(buf, n, H, D, dev, what):
    """A compressed cache's arrays and counters (its encoder view) as a call takes them, checked."""
    raw = buf["raw"]
    if (buf["H"], buf["D"]) != (H, D) or buf["sm"].shape[-1] != D or raw.shape[-1] != D:
        raise ValueError(f"{what} holds {buf['H']} heads of {buf['D']}, the rows {H} of {D}")
    for name in _ARRAYS:
        if not buf[name].is_contiguous():
            raise ValueError(f"{what}: {name} must be contiguous")
    _one_device(dev, *(buf[name] for name in _ARRAYS))
    return ([_lib.ptr(buf[name], 16, name) for name in _ARRAYS]
            + [_lib.ptr(buf["cnt"], 4, "cnt"), _lib.ptr(buf["before"], 4, "before")], int(buf["cap"]), raw.shape[0])


def rope_append_paged(q, k, v, cos, sin, kbuf, vbuf, lens, block_table, slots=None, *, q_norm=None, k_norm=None,
                      eps=1e-6, out=None):
    """One token of each of n sequences into pages, the rotation on the way: q bf16 [n, Hq, D], k
    and v bf16 [n, Hkv, D] (not rotated; strided views allowed). Row i belongs to sequence slot
    slots[i] (int32 [n], distinct; default: i), which has lens[slot] tokens, this one included: its
    position, whose row of cos and sin (fp32 [positions, D / 2]) turns it, is lens[slot] - 1, and
    its page block_table[slot, position // 16] (int32). kbuf, vbuf: bf16 pools [1, 16 * pages,
    Hkv, D], or the encoder views of two compressed caches (PagedCompressedKV._buf()). Norms as in
    rotate_prompt. Returns the rotated queries [n, Hq, D], ready for decode_attention; everything
    in one launch. A slot whose lens is 0 or past the table is left alone.

    This is rope_append on tensors: it changes no host state."""
    rows, out, n, H, D = _token_rows(q, k, v, cos, sin, q_norm, k_norm, eps, out)
    dev = q.device
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1:
        raise ValueError("block_table must be an int32 [sequences, pages] tensor with contiguous rows")
    if lens.dtype != torch.int32 or lens.dim() != 1 or not lens.is_contiguous() or lens.shape[0] < block_table.shape[0]:
        raise ValueError("lens must be a contiguous int32 [sequences] tensor")
    if slots is not None and (slots.dtype != torch.int32 or slots.shape != (n,) or not slots.is_contiguous()):
        raise ValueError("slots must be a contiguous int32 tensor with one entry per row")
    _one_device(dev, lens, block_table, slots)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return rope_append_paged(q, k, v, cos, sin, kbuf, vbuf, lens, block_table, slots, q_norm=q_norm,
                                     k_norm=k_norm, eps=eps, out=out)
    seqs, max_pages = block_table.shape
    table = (None if slots is None else slots.data_ptr(), lens.data_ptr(), block_table.data_ptr(),
             block_table.stride(0) if seqs > 1 else max_pages, seqs, max_pages)
    st = _lib.stream(dev.index)
    if isinstance(kbuf, dict):
        (*kp, kcap, krows), (*vp, vcap, vrows) = _flat(kbuf, n, H, D, dev, "kbuf"), _flat(vbuf, n, H, D, dev, "vbuf")
        arrivals = kbuf.get("arrivals")
        if arrivals is None:
            raise ValueError("kbuf has no arrival word ('arrivals', int32, zero between calls)")
        pages = kbuf["TS"] // P
        if vbuf["TS"] != kbuf["TS"] or kbuf["sm"].shape[0] * kbuf["sm"].shape[1] != kbuf["TS"]:
            raise ValueError("kbuf and vbuf must be pools of as many pages")
        _lib.call("exkv_rope_append_paged", *rows, *kp, _lib.ptr(arrivals, 4, "arrivals"), kcap, krows, *vp, vcap, vrows,
                  *table, pages, D, st)
        return out
    for t in (kbuf, vbuf):
        if t.dtype != BF16 or t.dim() != 4 or t.shape[2:] != (H, D) or not t.is_contiguous() or t.shape[1] % P:
            raise ValueError(f"kbuf and vbuf must be contiguous bf16 [1, {P} * pages, {H}, {D}] tensors")
    _one_device(dev, kbuf, vbuf)
    pages = kbuf.shape[0] * kbuf.shape[1] // P
    if vbuf.shape != kbuf.shape or pages < 1:
        raise ValueError("kbuf and vbuf must be pools of as many pages")
    _lib.call("exkv_rope_append_paged_bf16", *rows, _lib.ptr(kbuf), _lib.ptr(vbuf), *table, pages, D, st)
    return out


def _flat(buf, n, H, D, dev, what):
    ptrs, cap, rows = _compressed_args(buf, n, H, D, dev, what)
    return [*ptrs, cap, rows]


def launch_rope_append(q, k, v, cos, sin, kc, vc, *, q_norm=None, k_norm=None, eps=1e-6, out=None):
    """rope_append's kernel alone, without the host's checks of the step and its counts (a captured
    step replays it; the host then advances the caches)."""
    if isinstance(kc, (PagedCompressedKV, PagedBF16KV)):
        t = kc.table
        slots = t.step_rows()[0]
        kb, vb = (kc._buf(), vc._buf()) if isinstance(kc, PagedCompressedKV) else (kc.buf, vc.buf)
        return rope_append_paged(q, k, v, cos, sin, kb, vb, t.lens, t.block_table, slots, q_norm=q_norm, k_norm=k_norm,
                                 eps=eps, out=out)
    if _elsewhere(q.device):
        with torch.cuda.device(q.device):
            return launch_rope_append(q, k, v, cos, sin, kc, vc, q_norm=q_norm, k_norm=k_norm, eps=eps, out=out)
    rows, out, n, H, D = _token_rows(q, k, v, cos, sin, q_norm, k_norm, eps, out)
    st = _lib.stream(q.device.index)
    if isinstance(kc, CompressedKV):
        _one_device(q.device, kc.sm, vc.sm)
        _lib.call("exkv_rope_append", *rows, *kc._ptrs(), kc.cap, kc.raw.shape[0], *vc._ptrs(), vc.cap, vc.raw.shape[0],
                  kc.TS, D, st)
    else:
        _one_device(q.device, kc.buf, vc.buf)
        _lib.call("exkv_rope_append_bf16", *rows, _lib.ptr(kc.buf), _lib.ptr(kc.state, 4), _lib.ptr(vc.buf),
                  _lib.ptr(vc.state, 4), kc.TS, D, st)
    return out


def rope_append(q, k, v, cos, sin, k_cache, v_cache, *, q_norm=None, k_norm=None, eps=1e-6, out=None):
    """A decode step's token into a pair of caches with the rotation on the way: what

        k_cache.append(rotated k); v_cache.append(v)

    leaves, and the rotated queries [n, Hq, D] for decode_attention, in one launch. q bf16 [n, Hq,
    D], k and v bf16 [n, Hkv, D], not rotated (strided views allowed), one row per sequence, or per
    slot of the current step (begin_step) for paged caches; the position of each is the number of
    tokens its cache holds, and cos, sin (fp32 [positions, D / 2]) must reach it. k_cache, v_cache:
    two different caches of one kind -- CompressedKV, BF16KV, PagedCompressedKV or PagedBF16KV (of
    one PageTable) -- holding the same tokens. check_overflow follows at page ends as after append.
    q_norm, k_norm, eps: as in rotate_prompt. out: a contiguous tensor shaped like q."""
    if type(k_cache) is not type(v_cache) or not isinstance(k_cache, (CompressedKV, BF16KV, PagedCompressedKV, PagedBF16KV)):
        raise TypeError(f"rope_append takes two caches of one kind (got {type(k_cache).__name__}, {type(v_cache).__name__})")
    if k_cache is v_cache:
        raise ValueError("keys and values need a cache each")
    if (k_cache.H, k_cache.D) != (v_cache.H, v_cache.D):
        raise ValueError("k and v caches differ in shape")
    if k.dim() != 3 or v.shape != k.shape or q.dim() != 3:
        raise ValueError("q [n, Hq, D], k and v [n, Hkv, D] expected")
    if isinstance(k_cache, (PagedCompressedKV, PagedBF16KV)):
        t = k_cache.table
        if v_cache.table is not t:
            raise ValueError("k and v caches belong to two page tables")
        for c in (k_cache, v_cache):
            c._check_append(tuple(k.shape))
        last = max((t.length(s) for s in t._step_slots), default=1) - 1
    else:
        if (k_cache.B, k_cache.TS, k_cache.T) != (v_cache.B, v_cache.TS, v_cache.T):
            raise ValueError("k and v caches differ in shape or in the tokens they hold")
        for c in (k_cache, v_cache):
            c._check_can_append()
        if k.shape != (k_cache.B, k_cache.H, k_cache.D):
            raise ValueError(f"append expects [{k_cache.B}, {k_cache.H}, {k_cache.D}] rows (got {tuple(k.shape)})")
        last = k_cache.T
    if q.shape[0] != k.shape[0]:
        raise ValueError(f"{q.shape[0]} query rows for {k.shape[0]} key rows")
    if last >= cos.shape[0]:
        raise ValueError(f"position {last} is outside the tables of {cos.shape[0]} rows")
    out = launch_rope_append(q, k, v, cos, sin, k_cache, v_cache, q_norm=q_norm, k_norm=k_norm, eps=eps, out=out)
    k_cache._advance()
    v_cache._advance()
    return out


def add_norm(x, residual, weight, *, eps=1e-6, post_weight=None, gate=None, scale=1.0):
    """The residual stream between two blocks: a block's output x onto it, and the RMS norm that
    feeds the next block. x bf16 [..., C] (C up to 16384); residual of x's shape, or None (the
    stream starts with x); weight bf16 [C]. Returns (h, y), contiguous, of x's shape:

        u = x, or x rsqrt(mean(x^2) + eps) post_weight     (post_weight: a norm behind the block)
        u = u gate                                         (gate: bf16 [C], or of x's shape)
        h = residual + scale u
        y = h rsqrt(mean(h^2) + eps) weight

    fp32 inside; h and y are rounded once each, y from the unrounded h. Rows (the last axis)
    contiguous; x, residual and gate may have a stride between rows. With nothing to add, gate,
    norm or scale, h is x itself."""
    if x.dim() < 1 or x.dtype != BF16 or not x.is_cuda:
        raise ValueError("x must be a bf16 GPU tensor [..., C]")
    C = x.shape[-1]
    if not 1 <= C <= 16384:
        raise ValueError(f"add_norm takes 1 to 16384 channels (got {C})")
    dev = x.device
    _one_device(dev, residual, weight, post_weight, gate)
    _vec(weight, C, "weight")
    _vec(post_weight, C, "post_weight")
    scale = float(scale)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return add_norm(x, residual, weight, eps=eps, post_weight=post_weight, gate=gate, scale=scale)
    xr, sx = _row_view(x, "x")
    N = xr.shape[0]
    rr = gr = None
    sr = sg = 0
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != BF16:
            raise ValueError("residual must be a bf16 tensor of x's shape")
        rr, sr = _row_view(residual, "residual")
    if gate is not None:
        if gate.dtype != BF16 or (gate.shape != x.shape and gate.shape != (C,)):
            raise ValueError(f"gate must be a bf16 tensor of x's shape or [{C}]")
        if gate.shape == (C,) and x.dim() > 1:
            gr = _vec(gate, C, "gate")
        else:
            gr, sg = _row_view(gate, "gate")
            gr = gr.data_ptr()
    plain = residual is None and post_weight is None and gate is None and scale == 1.0
    h = x if plain else torch.empty(x.shape, dtype=BF16, device=dev)
    y = torch.empty(x.shape, dtype=BF16, device=dev)
    _lib.call("exkv_add_norm", xr.data_ptr(), sx, None if rr is None else rr.data_ptr(), sr, weight.data_ptr(),
              None if post_weight is None else post_weight.data_ptr(), gr, sg, scale, eps, None if plain else h.data_ptr(),
              y.data_ptr(), N, C, _lib.stream(dev.index))
    return h, y


def _vec(w, C, what):
    """Pointer of a bf16 [C] vector, or None."""
    if w is None:
        return None
    if w.dtype != BF16 or w.shape != (C,) or (C > 1 and w.stride(0) != 1):
        raise ValueError(f"{what} must be a contiguous bf16 [{C}] GPU tensor")
    return w.data_ptr()


def _row_view(t, what):
    """t [..., C] as rows [N, C] and their stride."""
    C = t.shape[-1]
    if C > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}: rows (the last axis) must be contiguous")
    if t.dim() != 2:
        try:
            t = t.view(-1, C) if t.numel() else t.reshape(0, C)
        except RuntimeError:
            raise ValueError(f"{what}: the axes before the last must have one stride") from None
    return t, (t.stride(0) if t.shape[0] > 1 else C)
