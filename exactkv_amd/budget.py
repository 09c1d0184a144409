"""Caches that hold no more than a budget of tokens: the attention that cached tokens receive, and the eviction of those
that receive the least.

  attention_mass   a decode step's attention weights over its cached keys, added to what they had
  prompt_mass      the same for the queries of packed prompts
  select_tokens    which tokens of each KV head a budget keeps
  gather_tokens    their keys and values out of a pair of caches
  evict            the three parts of an eviction in place: selected, gathered, encoded again

No counterpart in the reference, whose caches keep every token (exactkv/cache.py). Keys are cached with their rotation, so
tokens that stay keep their positions wherever they are stored, and each KV head keeps its own. The tensors of a call are
on one GPU; but for evict, the work goes to that GPU's current stream, waits for nothing and can be captured in a HIP
graph."""
import functools

import torch

from . import _lib
from .cache import BF16KV, CompressedKV
from .kernels import _QK_SCALE, P, _block_table_arg, _cache_args, _cache_dim, _check_q, _lens_arg, _window_arg, read_words
from .layer import _check_heads, _offsets, _on, _rows
from .paged import PagedBF16KV, PagedCompressedKV

F32 = torch.float32


# bytes of the calls' workspaces (16 at least), which the sizes alone determine
@functools.lru_cache(maxsize=4096)
def _mass_workspace(*sizes):
    return max(16, _lib.load().exkv_mass_workspace(*sizes))


@functools.lru_cache(maxsize=4096)
def _prompt_workspace(*sizes):
    return max(16, _lib.load().exkv_prompt_mass_workspace(*sizes))


def _is_bf16(c):
    return isinstance(c, (BF16KV, PagedBF16KV, torch.Tensor))


def _bf16_rows(c, dev, what):
    """The tensor [B, TS, H, D] of a bf16 cache."""
    t = c if isinstance(c, torch.Tensor) else c.buf
    if t.dtype is not torch.bfloat16 or t.dim() != 4 or not t.is_contiguous() or t.get_device() != dev:
        raise ValueError(f"{what} must be a contiguous bf16 [B, TS, H, D] tensor on the call's GPU")
    _lib.ptr(t, what=what)
    return t


def _compressed(c, dev, what):
    """(pointers and raw rows, TS, H, B, D) of a compressed cache on GPU `dev`."""
    args, TS, H, B = _cache_args(c)
    raw = c["raw"] if isinstance(c, dict) else c.raw
    if raw.get_device() != dev:
        raise ValueError(f"{what} must be on the call's GPU")
    return args, TS, H, B, _cache_dim(c)


def _table(block_table, B, dev):
    """(pointer, stride, capacity) of a block table, or (None, 0, None)."""
    if block_table is None:
        return None, 0, None
    if block_table.get_device() != dev:
        raise ValueError("block_table must be on the call's GPU")
    return _block_table_arg(block_table, B)


def _lens_on(lens, B, dev):
    if lens is not None and lens.get_device() != dev:
        raise ValueError("lens must be on the call's GPU")
    return _lens_arg(lens, B)


def _tokens(T, TS, lens, what):
    """The token count of a call without lens."""
    if lens is not None:
        return TS
    if T is None:
        raise ValueError(f"{what} needs T or lens")
    if not 0 <= int(T) <= TS:
        raise ValueError(f"{int(T)} tokens of a capacity of {TS}")
    return int(T)


def _mass_rows(t, shape, dev, what):
    if t.dtype is not F32 or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous fp32 {list(shape)} tensor on the call's GPU")
    return t.data_ptr()


def attention_mass(q, k_cache, T=None, *, mass=None, lens=None, block_table=None, window=0, out=None):
    """The attention that cached tokens receive from one query token of each sequence, added to what they had:

        out[b, h, j] = mass[b, h, j] + sum of softmax_j(q[b, g] . k[b, j, h] / sqrt(D)) over the query heads g of KV head h

    q bf16 [B, Hq, D] as decode_attention takes it. k_cache: the keys' cache, any of the four kinds (paged: rows as in
    decode_attention's current step), or a buffers() dict, or a bf16 tensor [B, TS, Hkv, D]; T, lens (int32, one entry or one
    per sequence), block_table and window as in attention_compressed. The softmax is over the tokens the window admits; the
    others get nothing. mass: fp32 [B, Hkv, TS], TS the cache's capacity in tokens (16 per entry of a block table's row), or
    None for 0. Returns out, new, or the one given, which may be mass itself; its entries behind a sequence's tokens are
    left as they are (0 in a new one).

    While it runs, the call holds 4 bytes a query head and token of workspace: T tokens a sequence, with lens as many as the
    cache's capacity (whatever the window), since its host does not know them."""
    dev = q.get_device()
    if dev >= 0 and dev != _lib.current_device():
        with _on(dev):
            return attention_mass(q, k_cache, T, mass=mass, lens=lens, block_table=block_table, window=window, out=out)
    B, Hq, D = _check_q(q)
    if isinstance(k_cache, (PagedCompressedKV, PagedBF16KV)) and block_table is None:
        if lens is not None or T is not None:
            raise ValueError("a paged cache's step has its own lengths: give block_table with T or lens")
        _, block_table, lens = k_cache.table.step_rows()
    elif T is None and lens is None and isinstance(k_cache, (CompressedKV, BF16KV)):
        T = k_cache.T
    bt, stride, capacity = _table(block_table, B, dev)
    if _is_bf16(k_cache):
        t = _bf16_rows(k_cache, dev, "k_cache")
        held, TS, Hkv, Dk = t.shape
        name, cache = "exkv_attention_mass_bf16", (t.data_ptr(),)
    else:
        cache, TS, Hkv, held, Dk = _compressed(k_cache, dev, "k_cache")
        name = "exkv_attention_mass"
    _check_heads(Hq, Hkv, D)
    if Dk != D:
        raise ValueError(f"cache head dim {Dk} differs from q's {D}")
    if block_table is None:
        if held < B:
            raise ValueError(f"the cache holds {held} sequences, q {B}")
        pages = 0
    else:
        pages, TS = held * TS // P, capacity
    T = _tokens(T, TS, lens, "attention_mass")
    lp, lstride = _lens_on(lens, B, dev)
    if window:
        window = _window_arg(window)
        if window > 0x7FFFFFFF:
            raise ValueError(f"window must be >= 0 (got {window})")
    else:
        window = 0
    shape = (B, Hkv, TS)
    mp = None if mass is None else _mass_rows(mass, shape, dev, "mass")
    fresh = out is None
    if fresh:
        out = torch.empty(shape, dtype=F32, device=q.device)
        op = out.data_ptr()
    else:
        op = _mass_rows(out, shape, dev, "out")
        if mass is not None and op != mp and abs(op - mp) < out.numel() * 4:
            raise ValueError("out overlaps mass")
    need = _mass_workspace(B, Hq, Hkv, T, TS, lens is not None, window)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    _lib.call(name, q.data_ptr(), *cache, bt, stride, pages, B, Hq, Hkv, D, T, TS, lp, lstride, window, _QK_SCALE[D], mp, op, fresh,
              ws.data_ptr(), need, _lib.stream(dev))
    return out


def prompt_mass(q, k, cu_seqlens, *, cu_seqlens_k=None, window=0, last=0):
    """The attention that the keys of packed prompts receive from their queries: q, k, cu_seqlens, cu_seqlens_k and window
    as in prompt_attention. Returns fp32 [Hkv, NK]: for each key and KV head the sum of the weights (softmax over the
    keys each query sees) of its sequence's queries, or with last > 0 of its last `last` ones, over the query heads of the
    KV head; 0 for keys that no sequence holds. A query that sees no key gives nothing."""
    dev = q.get_device()
    if dev >= 0 and dev != _lib.current_device():
        with _on(dev):
            return prompt_mass(q, k, cu_seqlens, cu_seqlens_k=cu_seqlens_k, window=window, last=last)
    N, Hq, D, sq_t, sq_h = _rows(q, dev, "q")
    NK, Hkv, Dk, sk_t, sk_h = _rows(k, dev, "k")
    _check_heads(Hq, Hkv, D)
    if Dk != D:
        raise ValueError(f"k must be [keys, heads, {D}] (got {tuple(k.shape)})")
    cu, S = _offsets(cu_seqlens, dev, "cu_seqlens")
    if cu_seqlens_k is None:
        cu_k = cu
        if NK != N:
            raise ValueError(f"{NK} keys for {N} queries: give cu_seqlens_k")
    else:
        cu_k, Sk = _offsets(cu_seqlens_k, dev, "cu_seqlens_k")
        if Sk != S:
            raise ValueError("cu_seqlens and cu_seqlens_k must hold as many sequences")
    window, last = int(window or 0), int(last or 0)
    if not 0 <= window <= 0x7FFFFFFF or not 0 <= last <= 0x7FFFFFFF:
        raise ValueError(f"window and last must be >= 0 (got {window}, {last})")
    out = torch.empty(Hkv, NK, dtype=F32, device=q.device)
    need = _prompt_workspace(S, N, NK, Hq, Hkv, D, window, last)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    _lib.call("exkv_prompt_mass", q.data_ptr(), sq_t, sq_h, k.data_ptr(), sk_t, sk_h, cu, cu_k, S, N, NK, Hq, Hkv, D, window, last,
              _QK_SCALE[D], out.data_ptr(), ws.data_ptr(), need, _lib.stream(dev))
    return out


def select_tokens(mass, keep, T=None, *, lens=None, sinks=0, recent=0):
    """Which `keep` tokens each KV head of each sequence keeps, by mass fp32 [B, H, TS] (rows contiguous): the first `sinks`,
    the latest `recent`, and of those between the ones with the most mass, of equal ones the first (NaN counts as
    the least). A sequence has T tokens, or lens[b] (int32, one entry or one per sequence). Returns (index int32 [B, H,
    keep], their mass fp32 [B, H, keep]), tokens ascending; of a sequence of fewer tokens all, then -1 and 0."""
    dev = mass.get_device()
    if dev >= 0 and dev != _lib.current_device():
        with _on(dev):
            return select_tokens(mass, keep, T, lens=lens, sinks=sinks, recent=recent)
    if mass.dtype is not F32 or mass.dim() != 3 or dev < 0:
        raise ValueError("mass must be an fp32 [B, H, TS] GPU tensor")
    B, H, TS = mass.shape
    if TS > 1 and mass.stride(2) != 1:
        raise ValueError("mass: rows (the last axis) must be contiguous")
    keep, sinks, recent = int(keep), int(sinks), int(recent)
    if keep < 1 or sinks < 0 or recent < 0 or sinks + recent > keep:
        raise ValueError(f"{sinks} first and {recent} latest tokens of {keep} kept")
    T = _tokens(T, TS, lens, "select_tokens")
    lp, lstride = _lens_on(lens, B, dev)
    index = torch.empty(B, H, keep, dtype=torch.int32, device=mass.device)
    kept = torch.empty(B, H, keep, dtype=F32, device=mass.device)
    _lib.call("exkv_select_tokens", mass.data_ptr(), mass.stride(0) if B > 1 else 0, mass.stride(1) if H > 1 else 0, lp, lstride, T, B, H,
              TS, keep, sinks, recent, index.data_ptr(), kept.data_ptr(), _lib.stream(dev))
    return index, kept


def gather_tokens(k_cache, v_cache, index, *, block_table=None):
    """Tokens of each KV head out of a pair of caches of one kind (cache objects, buffers() dicts, or bf16 tensors [B, TS, H,
    D]): row i of head h of sequence b is token index[b, h, i] (int32 [B, H, n]). block_table: the caches are pools of pages,
    as in attention_compressed (of paged cache objects their table's, a row for each slot, where none is given). Returns
    two bf16 tensors [B, n, H, D], with zeros where the index is -1; any other index outside the cache counts as -1 and sets
    an error bit (kernels.check_errors)."""
    dev = index.get_device()
    if dev >= 0 and dev != _lib.current_device():
        with _on(dev):
            return gather_tokens(k_cache, v_cache, index, block_table=block_table)
    if index.dtype is not torch.int32 or index.dim() != 3 or not index.is_contiguous() or dev < 0:
        raise ValueError("index must be a contiguous int32 [B, H, n] GPU tensor")
    B, H, n = index.shape
    if block_table is None and isinstance(k_cache, (PagedCompressedKV, PagedBF16KV)):
        block_table = k_cache.table.block_table
    bt, stride, capacity = _table(block_table, B, dev)
    if _is_bf16(k_cache) != _is_bf16(v_cache):
        raise ValueError("k_cache and v_cache must be of one kind")
    if _is_bf16(k_cache):
        k, v = _bf16_rows(k_cache, dev, "k_cache"), _bf16_rows(v_cache, dev, "v_cache")
        held, TS, Hc, D = k.shape
        other = v.shape
        name, caches = "exkv_gather_tokens_bf16", (k.data_ptr(), v.data_ptr())
    else:
        ka, TS, Hc, held, D = _compressed(k_cache, dev, "k_cache")
        va, *other = _compressed(v_cache, dev, "v_cache")
        other = (other[2], other[0], other[1], other[3])
        name, caches = "exkv_gather_tokens", (*ka, *va)
    if tuple(other) != (held, TS, Hc, D):
        raise ValueError(f"the caches differ in shape ({(held, TS, Hc, D)} and {tuple(other)})")
    if Hc != H or (block_table is None and held < B):
        raise ValueError(f"index is for {B} sequences of {H} heads, the caches hold {held} of {Hc}")
    pages = 0
    if block_table is not None:
        pages, TS = held * TS // P, capacity
    out = [torch.empty(B, n, H, D, dtype=torch.bfloat16, device=index.device) for _ in range(2)]
    _lib.call(name, *caches, bt, stride, pages, B, H, TS, D, index.data_ptr(), n, out[0].data_ptr(), out[1].data_ptr(), _lib.stream(dev))
    return tuple(out)


class Budget:
    """How many tokens each KV head keeps, and which (Engine's budget=): the first `sinks`, the latest `recent` (default:
    a quarter of keep) and otherwise those that have received the most attention. last: of a prompt's queries only the last
    `last` count (0: all)."""

    def __init__(self, keep, sinks=4, recent=None, last=0):
        recent = keep // 4 if recent is None else recent
        if keep < 1 or sinks < 0 or recent < 0 or sinks + recent > keep or last < 0:
            raise ValueError(f"{sinks} first and {recent} latest tokens of {keep} kept, last {last}")
        self.keep, self.sinks, self.recent, self.last = int(keep), int(sinks), int(recent), int(last)


def evict(k_cache, v_cache, mass, keep, *, sinks=0, recent=0, slots=None):
    """An eviction in place: of each KV head of each sequence the `keep` tokens that select_tokens chooses by mass stay, in
    their order, and are stored as the caches' first ones; their mass moves with them and what is behind them is 0. Caches
    of one kind that hold the same tokens:

      * contiguous ones: mass fp32 [B, H, TS]; the cache's token count becomes keep;
      * paged ones of one PageTable: mass fp32 [max_seqs, H, capacity], a row for each slot; slots (host ints, default all
        live ones) are cut, the pages behind go back to the pool (raw rows of evicted tokens stay in theirs until an eviction
        finds it more than half full, or compact()), and begin_step comes before the next step.

    Of several layers, give lists of equal length: a cache pair and its mass each. Paged layers share their table's lengths,
    so all caches of a table are cut in one call (ValueError otherwise).

    Everything about the arguments is checked before the first cache changes. An eviction that fails all the same (memory runs
    out) leaves caches of different lengths behind, which want a new prefill.

    Sequences of at most `keep` tokens stay as they are. Returns the index that select_tokens gave, a row for each sequence
    (slot); of lists, a list of them. Compressed caches wait for a raw-row count each (as a prefill does), so an eviction is
    not captured.

    The next token's position is from then on its place plus what was cut (the caches' dropped, PageTable.dropped(slot)), and
    rope_append's tables have to begin at that. Engines refuse to go on from evictions that they did not make."""
    many = isinstance(k_cache, (list, tuple))
    keep = int(keep)
    layers = list(zip(k_cache, v_cache, mass)) if many else [(k_cache, v_cache, mass)]
    if many and not (len(k_cache) == len(v_cache) == len(mass) > 0):
        raise ValueError(f"{len(k_cache)} key caches, {len(v_cache)} value caches and {len(mass)} masses")
    kind = type(layers[0][0])
    if any(type(c) is not kind for k, v, _ in layers for c in (k, v)) or not issubclass(kind, (CompressedKV, BF16KV, PagedCompressedKV,
                                                                                               PagedBF16KV)):
        raise TypeError(f"evict takes caches of one kind (got {', '.join(sorted({type(c).__name__ for x in layers for c in x[:2]}))})")
    caches = [c for k, v, _ in layers for c in (k, v)]
    if len({id(c) for c in caches}) != len(caches):
        raise ValueError("keys and values need a cache each")
    if any(getattr(c, "_pending", None) is not None for c in caches):
        raise RuntimeError("a page filled: call check_overflow() before evict()")
    dev = layers[0][2].get_device()
    if dev >= 0 and dev != _lib.current_device():
        with _on(dev):
            return evict(k_cache, v_cache, mass, keep, sinks=sinks, recent=recent, slots=slots)
    paged = issubclass(kind, (PagedCompressedKV, PagedBF16KV))
    if slots is not None and not paged:
        raise ValueError("contiguous caches are cut as a whole (slots are of paged ones)")
    for k, v, m in layers:
        if paged:
            if any(c.table is not layers[0][0].table or (c.H, c.D) != (k.H, k.D) for c in (k, v)):
                raise ValueError("k and v caches differ in shape or belong to two page tables")
            shape = (k.table.max_seqs, k.H, k.table.capacity)
        else:
            if (v.B, v.TS, v.H, v.D, v.T) != (k.B, k.TS, k.H, k.D, k.T):
                raise ValueError("k and v caches differ in shape or in the tokens they hold")
            shape = (k.B, k.H, k.TS)
        _mass_rows(m, shape, dev, "mass")
        if any((c.buf if _is_bf16(c) else c.raw).get_device() != dev for c in (k, v)):
            raise ValueError("the caches must be on the mass's GPU")
    spans = sorted((m.data_ptr(), m.data_ptr() + m.nbytes) for _, _, m in layers)
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError("each layer needs a mass of its own")
    choice = dict(sinks=sinks, recent=recent)
    kept = _evict_paged(layers, keep, choice, slots) if paged else [_evict_rows(*x, keep, choice) for x in layers]
    return kept if many else kept[0]


def _evict_rows(k_cache, v_cache, mass, keep, choice):
    T = k_cache.T
    index, kept = select_tokens(mass, keep, T, **choice)
    if T > keep:
        k, v = gather_tokens(k_cache, v_cache, index)
        dropped = k_cache.dropped + T - keep
        for c, x in ((k_cache, k), (v_cache, v)):
            c.replace(x)
            c.dropped = dropped
        mass[..., :keep] = kept
        mass[..., keep:] = 0
    return index


def _drop_raw_rows(caches, cut):
    """The raw rows of `cut` slots, which are about to be encoded again, out of pools that are more than half full: what
    earlier evictions left in them goes as well, so that a pool grows by what its sequences hold alone."""
    if not isinstance(caches[0], PagedCompressedKV):
        return
    others = [s for s in caches[0].table.live_slots() if s not in cut]
    for c, rows in zip(caches, read_words([c.cnt for c in caches])):
        if 2 * rows > c.cap:
            c._pack(others)


def _evict_paged(layers, keep, choice, slots):
    table = layers[0][0].table
    caches = {id(c) for k, v, _ in layers for c in (k, v)}
    if any(id(c) not in caches for c in table.caches()):
        raise ValueError("other caches share the page table and its lengths: evict from all of them in one call")
    if table.step_open() and any(c._appended != table.step for k, v, _ in layers for c in (k, v)):
        raise RuntimeError("the step's tokens come before evict()")
    slots = table.live_slots() if slots is None else [int(s) for s in slots]
    if len(set(slots)) != len(slots) or any(not 0 <= s < table.max_seqs or table._pages[s] is None for s in slots):
        raise ValueError(f"slots must be distinct and in use (got {slots})")
    dev = layers[0][2].device
    if not slots:
        return [torch.empty(0, k.H, keep, dtype=torch.int32, device=dev) for k, _, _ in layers]
    at = torch.tensor(slots, dtype=torch.int64).to(dev)
    lens = table.lens[at]
    chosen = [select_tokens(mass[at], keep, lens=lens, **choice) for _, _, mass in layers]
    long = [i for i, s in enumerate(slots) if table.length(s) > keep]
    if long:
        rows = torch.tensor(long, dtype=torch.int64).to(at.device)
        pages = table.block_table[at[rows]]
        tokens = [gather_tokens(k, v, index[rows], block_table=pages) for (k, v, _), (index, _) in zip(layers, chosen)]
        for i in long:
            table.cut(slots[i], keep)
        _drop_raw_rows([c for k, v, _ in layers for c in (k, v)], {slots[i] for i in long})
        for (k_cache, v_cache, mass), (_, kept), (k, v) in zip(layers, chosen, tokens):
            for j, i in enumerate(long):
                k_cache.prefill(slots[i], k[j:j + 1])
                v_cache.prefill(slots[i], v[j:j + 1])
            mass[at[rows], :, :keep] = kept[rows]
            mass[at[rows], :, keep:] = 0
    return [index for index, _ in chosen]
