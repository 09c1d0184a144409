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
(exactkv/engine.py:42-49,75-91). Everything is bf16 in and out and fp32 inside, rounded once, but
for the weights of prompt_attention's softmax, which are rounded to bf16 for the matrix product with
the values (at most 2^-8 of each; the sum they are divided by is not).
The tensors of a call are on one GPU; the work goes to that GPU's current stream, allocates
nothing but the outputs (and a split prompt's partial results), waits for nothing, and can be
captured in a HIP graph. No gradients are recorded.
"""
import operator

import torch

from . import _lib
from .cache import BF16KV, CompressedKV
from .kernels import HEAD_DIMS, P, _QK_SCALE
from .paged import PagedBF16KV, PagedCompressedKV

BF16 = torch.bfloat16


# The checks below run in every call of a decode step, so each reads an attribute once and names
# what is wrong only when something is.

def _rows(t, dev, what):
    """(tokens, heads, D, token stride, head stride) of bf16 rows [n, H, D] on GPU `dev` (an index)."""
    if t.dtype is not BF16 or t.dim() != 3 or t.get_device() != dev or dev < 0:
        _bad_tensor(t, dev, what, "a bf16 [tokens, heads, D] GPU tensor", t.dtype is BF16 and t.dim() == 3)
    n, H, D = t.shape
    s_t, s_h, s_d = t.stride()
    if s_d != 1 and D > 1:
        raise ValueError(f"{what}: rows (the last axis) must be contiguous")
    return n, H, D, (s_t if n > 1 else H * D), (s_h if H > 1 else D)


def _bad_tensor(t, dev, what, kind, form):
    if form and t.is_cuda and dev >= 0:
        raise ValueError(f"all tensors of a call must be on one GPU: {what} is on {t.device}, the first on cuda:{dev}")
    raise ValueError(f"{what} must be {kind}")


def _check_heads(Hq, Hkv, D):
    if D not in HEAD_DIMS:
        raise ValueError(f"head dim must be one of {HEAD_DIMS} (got {D})")
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads do not divide over {Hkv} KV heads")


def _int32(t, dims, dev, what, kind):
    """Pointer of a contiguous int32 tensor on GPU `dev`."""
    if t.dtype is not torch.int32 or t.dim() != dims or t.get_device() != dev or not t.is_contiguous():
        _bad_tensor(t, dev, what, kind, t.dtype is torch.int32 and t.dim() == dims and t.is_contiguous())
    return t.data_ptr()


def _offsets(cu, dev, what):
    """(pointer, sequences) of packed sequences' offsets."""
    p = _int32(cu, 1, dev, what, "a contiguous int32 [sequences + 1] GPU tensor")
    n = cu.shape[0]
    if n < 1:
        raise ValueError(f"{what} must be a contiguous int32 [sequences + 1] GPU tensor")
    return p, n - 1


def _vector(w, n, dev, what):
    """Pointer of a bf16 [n] weight, or None."""
    if w is None:
        return None
    if w.dtype is not BF16 or w.get_device() != dev or w.shape != (n,) or not w.is_contiguous():
        _bad_tensor(w, dev, what, f"a contiguous bf16 [{n}] GPU tensor",
                    w.dtype is BF16 and w.shape == (n,) and w.is_contiguous())
    return w.data_ptr()


def _tables(cos, sin, D, dev):
    """(cos pointer, sin pointer, rows) of fp32 tables [positions, D / 2]."""
    shape = cos.shape
    f32 = torch.float32
    if (cos.dtype is not f32 or sin.dtype is not f32 or cos.get_device() != dev or sin.get_device() != dev
            or len(shape) != 2 or shape[1] != D // 2 or sin.shape != shape or shape[0] < 1
            or not cos.is_contiguous() or not sin.is_contiguous()):
        raise ValueError(f"cos and sin must be contiguous fp32 [positions, {D // 2}] tensors of one shape on the call's GPU")
    return cos.data_ptr(), sin.data_ptr(), shape[0]


def _out_like(out, q, shape, *inputs):
    """out, checked, or a new tensor of q's shape."""
    if out is None:
        return torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    if out.shape != shape or out.dtype is not BF16 or out.get_device() != q.get_device() or not out.is_contiguous():
        raise ValueError("out must be a contiguous bf16 tensor shaped like q, on its GPU")
    if _overlap(out, q) or any(_overlap(out, t) for t in inputs):
        raise ValueError("out overlaps an input")
    return out


def _overlap(a, b):
    """Whether the memory that a and b span meets."""
    def span(t):
        first = t.data_ptr()
        return first, first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _on(dev):
    """The context in which a call on GPU `dev` launches when that is not the current device: its
    current stream may be the null stream, which is the current device's."""
    return torch.cuda.device(dev)


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
    dev = q.get_device()
    if dev >= 0 and dev != _lib.current_device():
        with _on(dev):
            return prompt_attention(q, k, v, cu_seqlens, cu_seqlens_k=cu_seqlens_k, window=window, out=out)
    N, Hq, D, sq_t, sq_h = _rows(q, dev, "q")
    NK, Hkv, Dk, sk_t, sk_h = _rows(k, dev, "k")
    NV, Hv, Dv, sv_t, sv_h = _rows(v, dev, "v")
    _check_heads(Hq, Hkv, D)
    if Dk != D or NV != NK or Hv != Hkv or Dv != D:
        raise ValueError(f"k and v must be of one shape [keys, heads, {D}] (got {tuple(k.shape)}, {tuple(v.shape)})")
    cu, S = _offsets(cu_seqlens, dev, "cu_seqlens")
    if cu_seqlens_k is None:
        cu_k = cu
        if NK != N:
            raise ValueError(f"{NK} keys for {N} queries: give cu_seqlens_k")
    else:
        cu_k, Sk = _offsets(cu_seqlens_k, dev, "cu_seqlens_k")
        if Sk != S:
            raise ValueError("cu_seqlens and cu_seqlens_k must hold as many sequences")
    window = int(window or 0)
    if window < 0 or window > 0x7FFFFFFF:
        raise ValueError(f"window must be >= 0 (got {window})")
    fresh = out is None
    out = _out_like(out, q, (N, Hq, D), k, v)
    # a call with few rows splits its keys: partial results, this call's own (in a graph: the graph's)
    need = _lib.load().exkv_prompt_workspace(S, N, NK, Hq, Hkv, D, window)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _lib.call("exkv_prompt_attention", q.data_ptr(), sq_t, sq_h, k.data_ptr(), sk_t, sk_h, v.data_ptr(), sv_t, sv_h,
              out.data_ptr(), cu, cu_k, S, N, NK, Hq, Hkv, D, window, fresh, _QK_SCALE[D],
              ws.data_ptr() if need else None, need, _lib.stream(dev))
    return out


def rotate_prompt(q, k, cos, sin, cu_seqlens, *, start=None, q_norm=None, k_norm=None, eps=1e-6):
    """A packed prompt's queries and keys rotated (half-split rotary embedding): q bf16 [N, Hq, D],
    k bf16 [N, Hkv, D], strided views allowed (rows 4-byte aligned), sequences as in prompt_attention; token i of
    sequence s stands at position i, or start[s] + i (start: int32 [S] on the GPU), whose row of
    cos and sin (fp32 [positions, D / 2]) turns it. q_norm, k_norm (bf16 [D]): the heads are
    RMS-normed with these weights and eps first (Qwen3). Returns the two, contiguous, ready for
    prompt_attention and the caches' prefill; rows that no sequence holds are 0.

    A position outside the tables is clamped to them and sets an error bit (kernels.check_errors)."""
    dev = q.get_device()
    if dev >= 0 and dev != _lib.current_device():
        with _on(dev):
            return rotate_prompt(q, k, cos, sin, cu_seqlens, start=start, q_norm=q_norm, k_norm=k_norm, eps=eps)
    N, Hq, D, sq_t, sq_h = _rows(q, dev, "q")
    NK, Hkv, Dk, sk_t, sk_h = _rows(k, dev, "k")
    if D not in HEAD_DIMS or Dk != D or NK != N or Hq == 0 or Hkv == 0:
        raise ValueError(f"q and k must be [N, heads, D] with D in {HEAD_DIMS} (got {tuple(q.shape)}, {tuple(k.shape)})")
    cu, S = _offsets(cu_seqlens, dev, "cu_seqlens")
    first = None
    if start is not None:
        first = _int32(start, 1, dev, "start", f"a contiguous int32 [{S}] GPU tensor")
        if start.shape[0] != S:
            raise ValueError(f"start must be a contiguous int32 [{S}] GPU tensor")
    cp, sp, rows = _tables(cos, sin, D, dev)
    qw, kw = _vector(q_norm, D, dev, "q_norm"), _vector(k_norm, D, dev, "k_norm")
    qo, ko = _out_like(None, q, (N, Hq, D)), _out_like(None, k, (N, Hkv, D))
    _lib.call("exkv_rotate_prompt", q.data_ptr(), sq_t, sq_h, k.data_ptr(), sk_t, sk_h, cp, sp, rows, qw, kw, eps,
              qo.data_ptr(), ko.data_ptr(), cu, first, S, N, Hq, Hkv, D, _lib.stream(dev))
    return qo, ko


def _token_rows(q, k, v, cos, sin, q_norm, k_norm, eps, out, dev):
    """The rows' arguments of a rotated append, and (out, n, Hkv, D)."""
    n, Hq, D, sq_n, sq_h = _rows(q, dev, "q")
    nk, Hkv, Dk, sk_n, sk_h = _rows(k, dev, "k")
    nv, Hv, Dv, sv_n, sv_h = _rows(v, dev, "v")
    if D not in HEAD_DIMS or nk != n or Dk != D or nv != n or Hv != Hkv or Dv != D or Hq == 0 or Hkv == 0:
        raise ValueError(f"q [n, Hq, D], k and v [n, Hkv, D] with D in {HEAD_DIMS} expected (got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)})")
    cp, sp, rows = _tables(cos, sin, D, dev)
    qw, kw = _vector(q_norm, D, dev, "q_norm"), _vector(k_norm, D, dev, "k_norm")
    out = _out_like(out, q, (n, Hq, D), k, v)
    return (q.data_ptr(), sq_n, sq_h, k.data_ptr(), sk_n, sk_h, v.data_ptr(), sv_n, sv_h, cp, sp, rows, qw, kw, eps,
            out.data_ptr(), n, Hq, Hkv), out, n, Hkv, D


_ARRAYS = operator.itemgetter("sm", "code", "base", "rowmask", "rowoff", "raw")
_WORDS = operator.itemgetter("cnt", "before", "cap", "TS")


def _pool_args(buf, H, D, dev, what):
    """A paged compressed cache's arrays and counters (its encoder view) as a call takes them, with the
    arrival word last if it has one, its cap, raw rows and pages, checked: the kernel writes them by
    address."""
    arrays = sm, code, base, rowmask, rowoff, raw = _ARRAYS(buf)
    cnt, before, cap, TS = _WORDS(buf)
    arrivals = buf.get("arrivals")                     # (the keys' serves both)
    u8, i32 = torch.uint8, torch.int32
    if (sm.dtype is not u8 or code.dtype is not u8 or base.dtype is not u8 or rowmask.dtype is not i32
            or rowoff.dtype is not i32 or raw.dtype is not BF16):
        raise ValueError(f"{what}: sm, code and base must be uint8, rowmask and rowoff int32, raw bfloat16")
    shape = raw.shape
    if len(shape) != 2 or shape[1] != D or buf["H"] != H or buf["D"] != D:
        raise ValueError(f"{what} holds {buf['H']} heads of {buf['D']} and raw rows {tuple(shape)}, the rows {H} of {D}")
    pages = TS // P
    units = pages * H
    if (TS % P or cap < 0 or sm.numel() != units * P * D or code.numel() * 2 != units * P * D or base.numel() != units * D
            or rowmask.numel() != units or rowoff.numel() != units):
        raise ValueError(f"{what}: the arrays are not those of {pages} pages")
    low, ptrs = 0, []
    for t in arrays:
        if t.get_device() != dev or not t.is_contiguous():
            raise ValueError(f"{what}: the arrays must be contiguous, on the rows' GPU")
        p = t.data_ptr()
        low |= p
        ptrs.append(p)
    for t in (cnt, before) if arrivals is None else (cnt, before, arrivals):
        if t.dtype is not i32 or t.get_device() != dev or t.numel() < 1:
            raise ValueError(f"{what}: cnt, before and arrivals must be int32 words on the rows' GPU")
        p = t.data_ptr()
        low |= p << 2
        ptrs.append(p)
    if low & 15:
        raise ValueError(f"{what}: the arrays must be 16-byte aligned, the counters 4-byte")
    return ptrs, int(cap), shape[0], pages


def rope_append_paged(q, k, v, cos, sin, kbuf, vbuf, lens, block_table, slots=None, *, q_norm=None, k_norm=None,
                      eps=1e-6, out=None):
    """One token of each of n sequences into pages, the rotation on the way: q bf16 [n, Hq, D], k
    and v bf16 [n, Hkv, D] (not rotated; strided views allowed, rows 4-byte aligned). Row i belongs to sequence slot
    slots[i] (int32 [n], distinct; default: i), which has lens[slot] tokens, this one included: its
    position, whose row of cos and sin (fp32 [positions, D / 2]) turns it, is lens[slot] - 1, and
    its page block_table[slot, position // 16] (int32). kbuf, vbuf: bf16 pools [1, 16 * pages,
    Hkv, D], or the encoder views of two compressed caches (PagedCompressedKV._buf()). Norms as in
    rotate_prompt. Returns the rotated queries [n, Hq, D], ready for decode_attention; everything
    in one launch.

    In compressed pools a token that fills its page (position % 16 == 15) also opens the next one in
    both caches, so entry position // 16 + 1, where the table has it, must be the slot's own by then
    (PageTable.begin_step claims it). An entry outside the pool opens nothing and sets an error bit
    (kernels.check_errors).

    A slot whose lens is 0 or past the table appends nothing and its pages stay as they are; its query
    row is written, rotated at position 0, and an error bit is set.

    This is rope_append on tensors: it changes no host state."""
    dev = q.get_device()
    if dev >= 0 and dev != _lib.current_device():
        with _on(dev):
            return rope_append_paged(q, k, v, cos, sin, kbuf, vbuf, lens, block_table, slots, q_norm=q_norm,
                                     k_norm=k_norm, eps=eps, out=out)
    rows, out, n, H, D = _token_rows(q, k, v, cos, sin, q_norm, k_norm, eps, out, dev)
    if block_table.dtype is not torch.int32 or block_table.dim() != 2 or block_table.get_device() != dev or block_table.stride(1) != 1:
        raise ValueError("block_table must be an int32 [sequences, pages] tensor with contiguous rows, on the rows' GPU")
    seqs, max_pages = block_table.shape
    lp = _int32(lens, 1, dev, "lens", "a contiguous int32 [sequences] GPU tensor")
    if lens.shape[0] < seqs:
        raise ValueError(f"lens has {lens.shape[0]} entries for {seqs} sequences")
    sp = None
    if slots is not None:
        sp = _int32(slots, 1, dev, "slots", "a contiguous int32 GPU tensor with one entry per row")
        if slots.shape[0] != n:
            raise ValueError("slots must be a contiguous int32 GPU tensor with one entry per row")
    table = (sp, lp, block_table.data_ptr(), block_table.stride(0) if seqs > 1 else max_pages, seqs, max_pages)
    st = _lib.stream(dev)
    if isinstance(kbuf, dict):
        kp, kcap, krows, pages = _pool_args(kbuf, H, D, dev, "kbuf")
        vp, vcap, vrows, vpages = _pool_args(vbuf, H, D, dev, "vbuf")
        if len(kp) < 9:
            raise ValueError("kbuf has no arrival word ('arrivals', int32, zero between calls)")
        if vpages != pages:
            raise ValueError("kbuf and vbuf must be pools of as many pages")
        _lib.call("exkv_rope_append_paged", *rows, *kp, kcap, krows, *vp[:8], vcap, vrows, *table, pages, D, st)
        return out
    shape = kbuf.shape
    for t in (kbuf, vbuf):
        if (t.dtype is not BF16 or t.shape != shape or len(shape) != 4 or shape[2] != H or shape[3] != D or shape[1] % P
                or t.get_device() != dev or not t.is_contiguous()):
            raise ValueError(f"kbuf and vbuf must be contiguous bf16 [1, {P} * pages, {H}, {D}] tensors on the rows' GPU")
    _lib.call("exkv_rope_append_paged_bf16", *rows, _lib.ptr(kbuf), _lib.ptr(vbuf), *table, shape[0] * shape[1] // P, D, st)
    return out


def launch_rope_append(q, k, v, cos, sin, kc, vc, *, q_norm=None, k_norm=None, eps=1e-6, out=None):
    """rope_append's kernel alone, without the host's checks of the step and its counts (a captured
    step replays it; the host then advances the caches)."""
    if isinstance(kc, (PagedCompressedKV, PagedBF16KV)):
        t = kc.table
        slots = t.step_rows()[0]
        kb, vb = (kc._buf(), vc._buf()) if isinstance(kc, PagedCompressedKV) else (kc.buf, vc.buf)
        return rope_append_paged(q, k, v, cos, sin, kb, vb, t.lens, t.block_table, slots, q_norm=q_norm, k_norm=k_norm,
                                 eps=eps, out=out)
    dev = q.get_device()
    if dev >= 0 and dev != _lib.current_device():
        with _on(dev):
            return launch_rope_append(q, k, v, cos, sin, kc, vc, q_norm=q_norm, k_norm=k_norm, eps=eps, out=out)
    rows, out, n, H, D = _token_rows(q, k, v, cos, sin, q_norm, k_norm, eps, out, dev)
    if (kc.B, kc.H, kc.D, kc.TS) != (n, H, D, vc.TS) or (vc.B, vc.H, vc.D) != (n, H, D):
        raise ValueError(f"the caches do not hold {n} sequences of {H} heads of {D}")
    st = _lib.stream(dev)
    if isinstance(kc, CompressedKV):
        if kc.raw.get_device() != dev or vc.raw.get_device() != dev:
            raise ValueError("the caches must be on the rows' GPU")
        _lib.call("exkv_rope_append", *rows, *kc._ptrs(), kc.cap, kc.raw.shape[0], *vc._ptrs(), vc.cap, vc.raw.shape[0],
                  kc.TS, D, st)
    else:
        if kc.buf.get_device() != dev or vc.buf.get_device() != dev:
            raise ValueError("the caches must be on the rows' GPU")
        _lib.call("exkv_rope_append_bf16", *rows, _lib.ptr(kc.buf), _lib.ptr(kc.state, 4), _lib.ptr(vc.buf),
                  _lib.ptr(vc.state, 4), kc.TS, D, st)
    return out


def rope_append(q, k, v, cos, sin, k_cache, v_cache, *, q_norm=None, k_norm=None, eps=1e-6, out=None):
    """A decode step's token into a pair of caches with the rotation on the way: what

        k_cache.append(rotated k); v_cache.append(v)

    leaves, and the rotated queries [n, Hq, D] for decode_attention, in one launch. q bf16 [n, Hq,
    D], k and v bf16 [n, Hkv, D], not rotated (strided views allowed), one row per sequence, or per
    slot of the current step (begin_step) for paged caches; the row of cos and sin (fp32
    [positions, D / 2], which must reach it) that turns each is the number of tokens its cache
    holds. (After an eviction that is its position less the tokens cut: the tables then begin at
    these, and slots cut by different numbers of tokens are refused.) k_cache, v_cache:
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
        if t._cut and len({t.dropped(s) for s in t._step_slots}) > 1:
            raise RuntimeError("the step's slots were cut by different numbers of tokens (evict): no table of angles serves them all")
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
    stream starts with x; fewer than 2^31 rows); weight bf16 [C]. Returns (h, y), contiguous, of x's shape:

        u = x, or x rsqrt(mean(x^2) + eps) post_weight     (post_weight: a norm behind the block)
        u = u gate                                         (gate: bf16 [C], or of x's shape)
        h = residual + scale u
        y = h rsqrt(mean(h^2) + eps) weight

    fp32 inside; h and y are rounded once each, y from the unrounded h. Rows (the last axis)
    contiguous; x, residual and gate may have a stride between rows. With nothing to add, gate,
    norm or scale, h is x itself."""
    shape, dev = x.shape, x.get_device()
    if not shape or x.dtype is not BF16 or dev < 0:
        raise ValueError("x must be a bf16 GPU tensor [..., C]")
    if dev != _lib.current_device():
        with _on(dev):
            return add_norm(x, residual, weight, eps=eps, post_weight=post_weight, gate=gate, scale=scale)
    C = shape[-1]
    if not 1 <= C <= 16384:
        raise ValueError(f"add_norm takes 1 to 16384 channels (got {C})")
    wp, pp = _vector(weight, C, dev, "weight"), _vector(post_weight, C, dev, "post_weight")
    if wp is None:
        raise ValueError("add_norm needs the norm's weight")
    xp, N, sx = _row_view(x, shape, dev, "x")
    if N > 0x7FFFFFFF:
        raise ValueError(f"add_norm takes fewer than 2^31 rows (got {N})")
    rp = gp = None
    sr = sg = 0
    if residual is not None:
        rp, _, sr = _row_view(residual, shape, dev, "residual")
    if gate is not None:
        if gate.dim() == 1 and len(shape) > 1:
            gp = _vector(gate, C, dev, "gate")
        else:
            gp, _, sg = _row_view(gate, shape, dev, "gate")
    y = torch.empty_like(x) if x.is_contiguous() else x.new_empty(shape)
    if rp is None and pp is None and gp is None and scale == 1.0:
        h, hp = x, None
    else:
        h = torch.empty_like(y)
        hp = h.data_ptr()
    _lib.call("exkv_add_norm", xp, sx, rp, sr, wp, pp, gp, sg, scale, eps, hp, y.data_ptr(), N, C, _lib.stream(dev))
    return h, y


def _row_view(t, shape, dev, what):
    """(pointer, rows, row stride) of a bf16 tensor of this shape [..., C], seen as rows."""
    if t.dtype is not BF16 or t.shape != shape or t.get_device() != dev:
        _bad_tensor(t, dev, what, f"a bf16 tensor of x's shape {tuple(shape)}", t.dtype is BF16 and t.shape == shape)
    C = shape[-1]
    n = t.numel() // C
    if t.is_contiguous():
        return t.data_ptr(), n, C
    if C > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}: rows (the last axis) must be contiguous")
    if t.dim() != 2:
        try:
            t = t.view(-1, C)
        except RuntimeError:
            raise ValueError(f"{what}: the axes before the last must have one stride") from None
    return t.data_ptr(), n, (t.stride(0) if n > 1 else C)
