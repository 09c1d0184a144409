"""What a decode loop does behind its logits, and with a cache that may hold no more tokens, as cases to measure.

Each case names an operator (`op`) and its sizes:

  sample       sample: one token a row from logits and given uniform numbers, with temperature, top-k, top-p and min-p,
               and its log-probability
  mass         attention_mass: the attention weights of one new token of each sequence over its cached keys, summed over
               the query heads of each KV head and added to what the tokens have gathered before
  prompt_mass  prompt_mass: the same for the queries of packed prompts, all of each or its last ones
  evict        select_tokens and gather_tokens: the tokens of each KV head that a budget keeps (the first ones, the
               latest ones and those with the most weight), and their keys and values out of the cache

`own` chooses the framework's kernels; otherwise run computes the same in elementary torch operations."""
import math

import torch

DEV = "cuda"
PAGE = 16
own = False
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one chat sequence's next token with the usual cuts: latency
        dict(name="sample_one", op="sample", B=1, V=128256, dtype="bf16", t=0.7, k=50, p=0.9, m=0.0, mixed=False),
        # a serving batch whose rows each have their own settings, greedy ones among them
        dict(name="sample_mixed", op="sample", B=128, V=128256, dtype="bf16", t=1.0, k=0, p=1.0, m=0.0, mixed=True),
        # nucleus sampling over fp32 logits, a vocabulary of odd size
        dict(name="sample_nucleus", op="sample", B=61, V=50257, dtype="fp32", t=1.0, k=0, p=0.95, m=0.0, mixed=False),
        # many samples from the whole distribution, as a rollout draws them: the largest
        dict(name="sample_pure", op="sample", B=256, V=152064, dtype="bf16", t=1.0, k=0, p=1.0, m=0.0, mixed=False),
        # one chat sequence of about a thousand tokens in a plain cache: latency
        dict(name="mass_one", op="mass", cache="bf16", B=1, T=997, Hq=32, Hkv=8, D=128, window=0),
        # the benchmark's headline shape over compressed keys
        dict(name="mass_8x8k", op="mass", cache="compressed", B=8, T=8192, Hq=32, Hkv=8, D=128, window=0),
        # a serving batch of mixed lengths over a pool of pages
        dict(name="mass_paged", op="mass", cache="paged", B=61, T=4339, Hq=28, Hkv=4, D=128, window=0),
        # new prompts of mixed lengths, one empty, a small model's head dim
        dict(name="prompt_mixed", op="prompt_mass", lens="1201,17,640,0,333,1,1024,95", past="0,0,0,0,0,0,0,0", Hq=14,
             Hkv=2, D=64, window=0, last=0),
        # a document of 8K tokens: the largest
        dict(name="prompt_8k", op="prompt_mass", lens="8192", past="0", Hq=32, Hkv=8, D=128, window=0, last=0),
        # what the last 64 tokens of a 16K prompt look at, its earlier pieces already held
        dict(name="prompt_last", op="prompt_mass", lens="512", past="15873", Hq=32, Hkv=8, D=128, window=0, last=64),
        # one sequence's plain cache cut to a quarter
        dict(name="evict_one", op="evict", cache="bf16", B=1, T=2051, keep=512, sinks=4, recent=64, H=8, D=128),
        # the headline shape's compressed caches cut to a quarter
        dict(name="evict_8x8k", op="evict", cache="compressed", B=8, T=8192, keep=2048, sinks=4, recent=512, H=8, D=128),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = [(32, 8), (28, 4), (32, 32), (16, 2), (14, 2), (40, 8), (24, 6), (8, 1), (64, 8)]


def draw(rng):
    op = rng.choice(["sample"] * 4 + ["mass"] * 3 + ["prompt_mass"] * 3 + ["evict"] * 3)
    Hq, Hkv = rng.choice(_HEADS)
    D = rng.choice([128, 128, 64, 256])
    if op == "sample":
        V = rng.choice([_spread(rng, 100, 152064), 32000, 50257, 128256, 152064])
        dtype = rng.choice(["bf16", "bf16", "fp32", "fp16"])
        B = _spread(rng, 1, 256 if dtype != "fp32" else 128)
        return dict(op=op, B=B, V=V, dtype=dtype, t=rng.choice([1.0, 0.7, 1.3, 0.2, 0.0]), k=rng.choice([0, 0, 50, _spread(rng, 1, V)]),
                    p=rng.choice([1.0, 0.9, 0.95, round(rng.uniform(0.05, 0.999), 3)]), m=rng.choice([0.0, 0.0, 0.05, 0.3]),
                    mixed=rng.random() < 0.3)
    if op == "mass":
        T = _spread(rng, 1, 32768)
        most = 61 * 4339 * 4 * 128 // (T * Hkv * D)             # no more than the largest listed one reads
        return dict(op=op, cache=rng.choice(["bf16", "compressed", "paged"]), B=_spread(rng, 1, max(1, min(128, most))), T=T,
                    Hq=Hq, Hkv=Hkv, D=D, window=rng.choice([0, 0, 0, _spread(rng, 1, 4096)]))
    if op == "prompt_mass":
        S = rng.choice([1, 1, 2, 3, 5, 9])
        # the padded batch of the plain form is no larger than the largest listed case's
        top = int(8192 * math.sqrt(32 * 128 / (S * Hq * max(D, 128))))
        longest = _spread(rng, 1, top)
        keys = [longest] + [rng.choice([0, 1, _spread(rng, 1, longest)]) if rng.random() < 0.3 else
                            rng.randint(1, longest) for _ in range(S - 1)]
        chunk = rng.random() < 0.3
        past = [rng.randint(0, n) if chunk else 0 for n in keys]
        lens = [n - p for n, p in zip(keys, past)]
        if sum(lens) == 0:
            lens[0], past[0] = keys[0], 0
        return dict(op=op, lens=",".join(map(str, lens)), past=",".join(map(str, past)), Hq=Hq, Hkv=Hkv, D=D,
                    window=rng.choice([0, 0, 0, _spread(rng, 1, 4096)]), last=rng.choice([0, 0, 1, _spread(rng, 1, 512)]))
    H = min(Hkv, 8)
    T = _spread(rng, 2, 16384)
    B = _spread(rng, 1, max(1, min(64, 8 * 8192 * 8 * 128 // (T * H * D))))
    keep = rng.randint(1, T)
    sinks = min(rng.choice([0, 4, rng.randint(0, keep)]), keep)
    return dict(op=op, cache=rng.choice(["bf16", "compressed", "paged"]), B=B, T=T, keep=keep, sinks=sinks,
                recent=rng.randint(0, keep - sinks), H=H, D=D)


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV)


def _ints(text):
    return [int(n) for n in text.split(",")]


def _offsets(lens):
    return torch.tensor([0] + lens, device=DEV).cumsum(0).int()


def _heads(g, n, H, D, sigma=0.5):
    """Rows of H heads with a scale for each channel, as projections give them."""
    return (_randn(g, n, H, D) * torch.exp(_randn(g, H, D) * sigma)).bfloat16()


def _lengths(c):
    """Lengths of a pool's sequences: from a third of T up to T; of one cache's: T."""
    if c["cache"] != "paged":
        return [c["T"]] * c["B"]
    return [max(1, c["T"] - (i * 7 % c["B"]) * (c["T"] * 2 // 3) // c["B"]) for i in range(c["B"])]


def _encode(x, lens):
    """Rows x [B, TS, H, D] as a compressed cache holds them: a byte of sign and mantissa and a 4-bit exponent code each,
    over one base exponent for 16 tokens of a channel, and as they are where that does not reach or the page is still open."""
    B, TS, H, D = x.shape
    bits = x.view(torch.int16).int() & 0xFFFF
    e = ((bits >> 7) & 0xFF).view(B, TS // PAGE, PAGE, H, D)
    low = (e.amax(2, keepdim=True) - 15).clamp(min=0)
    flag = (e == 0).any(2, keepdim=True) & (low > 0)             # a page with zeros: code 0 is exponent 0
    zero = flag & (e == 0)
    code = torch.where(zero, 0, e - low)
    raw = ((code < (flag & ~zero).int()) | (low >= 128)).any(-1)                      # [B, pages, 16, H]
    opened = torch.arange(TS // PAGE, device=DEV) == torch.tensor(lens, device=DEV)[:, None] // PAGE
    raw |= opened[:, :, None, None]
    code = code.clamp(0, 15).view(B, TS, H, D)
    order = raw.transpose(2, 3)                                                       # [B, pages, H, 16]
    counts = order.sum(-1)
    offset = counts.flatten().cumsum(0).view(counts.shape) - counts
    rows = x.view(B, TS // PAGE, PAGE, H, D).transpose(2, 3)[order]
    return dict(sm=((bits >> 8) & 0x80 | bits & 0x7F).byte(), code=(code[..., : D // 2] | code[..., D // 2:] << 4).byte(),
                base=(low + 128 * flag)[:, :, 0].clamp(max=255).byte(),
                rowmask=(order * (1 << torch.arange(PAGE, device=DEV))).sum(-1).int(), rowoff=offset.int(),
                raw=torch.cat([rows, torch.zeros(1, D, dtype=x.dtype, device=DEV)]), shape=(B, TS, H, D))


def _cache(c, g, x, order=None):
    """Rows x as the case's cache; of a pool the pages stand in the given order."""
    if c["cache"] == "bf16":
        return x
    comp = _encode(x, _lengths(c))
    if c["cache"] == "compressed":
        return comp
    B, TS, H, D = x.shape
    pool = {"raw": comp["raw"], "shape": (1, B * TS, H, D)}
    for name, per in (("sm", PAGE), ("code", PAGE), ("base", 1), ("rowmask", 1), ("rowoff", 1)):
        t = comp[name]
        t = t.reshape(B * TS // PAGE, per, *t.shape[2:])
        pool[name] = t[order].reshape(1, -1, *t.shape[2:])
    return pool


def _table(c, g, pages):
    """(which page of all stands at each place of the pool, block table) of B sequences."""
    order = torch.randperm(c["B"] * pages, generator=g, device=DEV)
    at = torch.empty_like(order)
    at[order] = torch.arange(order.numel(), device=DEV)
    return order, at.view(c["B"], pages).int()


def _prepare_sample(c, g):
    B, V = c["B"], c["V"]
    logits = _randn(g, B, V) * 2.2
    head = torch.randint(V, (B, 40), generator=g, device=DEV)                # a few tokens that the context makes likely
    logits.scatter_(1, head, 6 + 2.5 * _randn(g, B, 40))
    s = dict(logits=logits.to(_TYPES[c["dtype"]]), u=_rand(g, B), t=c["t"], k=c["k"], p=c["p"], m=c["m"])
    if c["mixed"]:
        on = _rand(g, 4, B)
        s["t"] = torch.where(on[0] < 0.15, 0.0, 0.3 + _rand(g, B))
        s["k"] = torch.where(on[1] < 0.4, 0, torch.randint(1, 200, (B,), generator=g, device=DEV)).int()
        s["p"] = torch.where(on[2] < 0.4, 1.0, 0.5 + 0.49 * _rand(g, B))
        s["m"] = torch.where(on[3] < 0.6, 0.0, 0.02 + 0.1 * _rand(g, B))
    return s


def _prepare_mass(c, g):
    lens, H, D = _lengths(c), c["Hkv"], c["D"]
    TS = -(-c["T"] // PAGE) * PAGE
    x = _heads(g, c["B"] * TS, H, D).view(c["B"], TS, H, D)
    order, table = _table(c, g, TS // PAGE) if c["cache"] == "paged" else (None, None)
    mass = _rand(g, c["B"], H, TS) * 3
    return dict(q=_randn(g, c["B"], c["Hq"], D).bfloat16(), x=x, k=_cache(c, g, x, order), table=table, mass=mass,
                lens=torch.tensor(lens, dtype=torch.int32, device=DEV), out=torch.zeros_like(mass))


def _prepare_prompt(c, g):
    lens, past = _ints(c["lens"]), _ints(c["past"])
    keys = [a + b for a, b in zip(lens, past)]
    return dict(q=_randn(g, sum(lens), c["Hq"], c["D"]).bfloat16(), k=_heads(g, sum(keys), c["Hkv"], c["D"]),
                cu_q=_offsets(lens), cu_k=_offsets(keys))


def _prepare_evict(c, g):
    H, D, B = c["H"], c["D"], c["B"]
    TS = -(-c["T"] // PAGE) * PAGE
    order, table = _table(c, g, TS // PAGE) if c["cache"] == "paged" else (None, None)
    s = dict(table=table, lens=torch.tensor(_lengths(c), dtype=torch.int32, device=DEV))
    for name in "kv":
        s["x" + name] = _heads(g, B * TS, H, D).view(B, TS, H, D)
        s[name] = _cache(c, g, s["x" + name], order)
    s["mass"] = torch.exp(2 * _randn(g, B, H, TS))                           # a few tokens gather most of the weight
    return s


def prepare(case, seed):
    return _OPS[case["op"]][0](case, _gen(seed)) | {"case": case}


# ---------------------------------------------------------------- plain forms

def _column(v, n, dtype):
    """A setting as a column of n rows."""
    return torch.as_tensor(v, device=DEV).to(dtype).expand(n)[:, None]


def _plain_sample(s):
    l = s["logits"].double()
    B, V = l.shape
    t, p, m = (_column(s[x], B, torch.float32).double() for x in "tpm")
    k = _column(s["k"], B, torch.int64)
    l, token = l.sort(dim=1, descending=True, stable=True)                   # equal ones keep their order
    rank = torch.arange(V, device=DEV)
    greedy = ~(t > 0)
    w = ((l - l[:, :1]) / torch.where(greedy, 1.0, t)).exp_()
    fit = ((k <= 0) | (rank < k)) & (w >= m)                                 # a beginning of the row, each time
    fit &= ~greedy | (rank == 0)
    total = w.cumsum(1)
    before = total - w
    whole = total.gather(1, fit.sum(1, keepdim=True) - 1)
    fit &= (before < p * whole) | (p >= 1)
    kept = fit.sum(1, keepdim=True)
    whole = total.gather(1, kept - 1)
    r = torch.minimum((total <= s["u"].double()[:, None] * whole).sum(1, keepdim=True), kept - 1)
    return token.gather(1, r)[:, 0], (w.gather(1, r) / whole).log_()[:, 0].float()


def _decode(c, s, name):
    """A cache's rows [B, TS, H, D] in bf16, from the bytes that it holds."""
    k = s[name]
    if c["cache"] == "bf16":
        return k
    H, D = k["shape"][2:]
    pages = k["shape"][0] * k["shape"][1] // PAGE
    at = torch.arange(pages, device=DEV).view(c["B"], -1) if s["table"] is None else s["table"].long()
    sm, code = (k[x].view(pages, PAGE, H, -1)[at] for x in ("sm", "code"))
    base = k["base"].view(pages, 1, H, D)[at]
    code = torch.cat([code & 15, code >> 4], -1)
    e = ((base & 127) + code).masked_fill_((base >= 128) & (code == 0), 0).short()
    sm = sm.short()
    x = ((sm & 0x80) << 8 | e << 7 | sm & 0x7F).view(torch.bfloat16)         # [B, pages, 16, H, D]
    held = (k["rowmask"].view(pages, H)[at][:, :, None] >> torch.arange(PAGE, device=DEV, dtype=torch.int32)[:, None]) & 1
    slot = k["rowoff"].view(pages, H)[at][:, :, None] + held.cumsum(2) - held
    x = torch.where(held.bool()[..., None], k["raw"][slot * held], x)
    return x.view(c["B"], -1, H, D)


def _plain_mass(s):
    c, q = s["case"], s["q"]
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    k = _decode(c, s, "k").float().permute(0, 2, 3, 1).contiguous()          # [B, Hkv, D, TS]
    score = torch.matmul(q.float().view(B, Hkv, Hq // Hkv, D), k).mul_(D ** -0.5)
    n, j = s["lens"][:, None], torch.arange(k.shape[-1], device=DEV)
    seen = j < n
    if c["window"]:
        seen &= j >= n - c["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    w = score.sub_(score.amax(-1, keepdim=True)).exp_()
    w /= w.sum(-1, keepdim=True)
    return torch.where((j < n)[:, None], s["mass"] + w.sum(2), s["out"])


def _rows(cu, n, most, first):
    """Row index [S, most] of every token from `first` on of a padded batch (clamped to the n rows) and whether it is one."""
    at = first[:, None] + torch.arange(most, device=DEV)
    return (cu[:-1, None].long() + at).clamp(max=max(n - 1, 0)), at < (cu[1:] - cu[:-1])[:, None]


def _plain_prompt(s):
    c, q, k = s["case"], s["q"], s["k"]
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    lens, past = _ints(c["lens"]), _ints(c["past"])
    S, Lk = len(lens), max(a + b for a, b in zip(lens, past))
    nk, nq = s["cu_k"].diff(), s["cu_q"].diff()
    first = (nq - c["last"]).clamp(min=0) if c["last"] else torch.zeros_like(nq)
    Lq = min(max(lens), c["last"]) if c["last"] else max(lens)
    qi, q_real = _rows(s["cu_q"], q.shape[0], Lq, first)
    ki, k_real = _rows(s["cu_k"], k.shape[0], Lk, torch.zeros_like(nk))
    qp = q[qi].float().view(S, Lq, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, -1, D)
    kp = k[ki].float().permute(0, 2, 3, 1).contiguous()                      # [S, Hkv, D, Lk]
    score = torch.matmul(qp, kp).view(S, Hkv, Hq // Hkv, Lq, Lk)
    score *= D ** -0.5
    pos = (nk - nq + first)[:, None] + torch.arange(Lq, device=DEV)           # the key a query stands at
    key = torch.arange(Lk, device=DEV)
    seen = (key <= pos[..., None]) & k_real[:, None] & q_real[..., None]
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    w = score.sub_(top.masked_fill(top == -math.inf, 0)).exp_()
    total = w.sum(-1, keepdim=True)
    w /= total.masked_fill(total == 0, 1)
    return w.sum((2, 3)).permute(1, 0, 2)[:, k_real].contiguous()            # [Hkv, keys]


def _plain_evict(s):
    c, mass = s["case"], s["mass"]
    j, n = torch.arange(mass.shape[-1], device=DEV), s["lens"][:, None, None]
    worth = torch.where((j < c["sinks"]) | (j >= n - c["recent"]), math.inf, mass)
    worth = torch.where(j < n, worth, -math.inf)
    best = worth.argsort(stable=True, dim=-1, descending=True)[..., : c["keep"]]   # equal ones keep their order
    at = best.sort(-1).values
    real = torch.arange(c["keep"], device=DEV) < n
    rows = torch.where(real, at, 0).transpose(1, 2)                           # [B, keep, H]
    out = [torch.where(real, at, -1).int(), torch.where(real, mass.gather(-1, at), 0)]
    for name in "kv":
        x = _decode(c, s, name)
        x = x.gather(1, rows[..., None].expand(-1, -1, -1, x.shape[-1]))
        out.append(x.masked_fill(~real.transpose(1, 2)[..., None], 0))
    return tuple(out)


# ---------------------------------------------------------------- the framework's operators

def _own_sample(s):
    import exactkv_amd as exactkv
    return exactkv.sample(s["logits"], s["u"], temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["m"], logprob=True)


def _own_mass(s):
    import exactkv_amd as exactkv
    return exactkv.attention_mass(s["q"], s["k"], lens=s["lens"], block_table=s["table"], window=s["case"]["window"],
                                  mass=s["mass"], out=s["out"])


def _own_prompt(s):
    import exactkv_amd as exactkv
    return exactkv.prompt_mass(s["q"], s["k"], s["cu_q"], cu_seqlens_k=s["cu_k"], window=s["case"]["window"],
                               last=s["case"]["last"])


def _own_evict(s):
    import exactkv_amd as exactkv
    c = s["case"]
    index, mass = exactkv.select_tokens(s["mass"], c["keep"], lens=s["lens"], sinks=c["sinks"], recent=c["recent"])
    k, v = exactkv.gather_tokens(s["k"], s["v"], index, block_table=s["table"])
    return index, mass, k, v


_OPS = {"sample": (_prepare_sample, _plain_sample, _own_sample),
        "mass": (_prepare_mass, _plain_mass, _own_mass),
        "prompt_mass": (_prepare_prompt, _plain_prompt, _own_prompt),
        "evict": (_prepare_evict, _plain_evict, _own_evict)}


def run(state):
    return _OPS[state["case"]["op"]][2 if own else 1](state)


# ---------------------------------------------------------------- what a pass cannot do without

def _seen_keys(n, window):
    return min(n, window) if window else n


def _row_bytes(c, D):
    """Bytes of one token's row of one head in the case's cache."""
    return 2 * D if c["cache"] == "bf16" else D + D // 2 + D / PAGE


def _queries(c):
    """(queries that count, keys before the first of them) of each sequence."""
    out = []
    for n, p in zip(_ints(c["lens"]), _ints(c["past"])):
        m = min(n, c["last"]) if c["last"] else n
        out.append((m, p + n - m))
    return out


def _pairs(c):
    """Visible (query, key) pairs."""
    total = 0
    for n, p in _queries(c):
        if c["window"] == 0:
            total += n * p + n * (n + 1) // 2
        else:                                          # query i sees min(p + i + 1, window) keys
            short = max(0, min(n, c["window"] - p - 1))
            total += short * p + short * (short + 1) // 2 + (n - short) * c["window"]
    return total


def work(case):
    c = case
    if c["op"] == "sample":
        return {"bytes": c["B"] * (c["V"] * (4 if c["dtype"] == "fp32" else 2) + 16), "flops": 4 * c["B"] * c["V"]}
    if c["op"] == "mass":
        keys = sum(_seen_keys(n, c["window"]) for n in _lengths(c))
        return {"bytes": int(keys * c["Hkv"] * _row_bytes(c, c["D"])) + 2 * c["B"] * c["Hq"] * c["D"]
                + 8 * c["Hkv"] * sum(_lengths(c)), "flops": keys * c["Hq"] * (2 * c["D"] + 4)}
    if c["op"] == "prompt_mass":
        queries = _queries(c)
        keys = sum(min(n + p, n + c["window"] - 1) if c["window"] and n else (n + p if n else 0) for n, p in queries)
        held = sum(_ints(c["lens"])) + sum(_ints(c["past"]))
        # the products once for the rows' sums and once for the keys'
        return {"bytes": 2 * c["D"] * (sum(n for n, _ in queries) * c["Hq"] + keys * c["Hkv"]) + 4 * held * c["Hkv"],
                "flops": 4 * c["D"] * c["Hq"] * _pairs(c)}
    kept = sum(min(n, c["keep"]) for n in _lengths(c)) * c["H"]
    return {"bytes": int(2 * kept * _row_bytes(c, c["D"])) + 8 * c["B"] * c["keep"] * c["H"] * (c["D"] // 2 + 1)
            + 4 * c["H"] * sum(_lengths(c)), "flops": 4 * c["H"] * sum(_lengths(c))}


# ---------------------------------------------------------------- the definitions, in 64 bits

def _exact_sample(c, s):
    if c["B"] * c["V"] > 60_000_000:
        return None
    rows = s["logits"].double()
    tokens, logs = [], []
    for b in range(c["B"]):
        t, k, p, m = (float(s[x][b]) if torch.is_tensor(s[x]) else float(torch.tensor(s[x]).float()) for x in "tkpm")
        l = rows[b]
        # by value, equal ones by index: two stable sorts of the row turned round
        order = (c["V"] - 1) - torch.sort(l.flip(0), stable=True).indices.flip(0)
        l = l[order]
        if t <= 0:
            tokens.append(order[0])
            logs.append(torch.zeros((), dtype=torch.float64, device=DEV))
            continue
        if k > 0:
            l = l[: int(k)]
        w = torch.exp(l / t - l[0] / t)
        w = w[w >= m]
        if p < 1:
            heard = torch.cat([torch.zeros(1, dtype=torch.float64, device=DEV), torch.cumsum(w, 0)])
            w = w[: int(torch.searchsorted(heard[:-1].contiguous(), (p * heard[-1]).view(1)))]
        run_up = torch.cumsum(w / w.sum(), 0)
        r = min(int(torch.searchsorted(run_up, s["u"][b].double().view(1), right=True)), w.numel() - 1)
        tokens.append(order[r])
        logs.append(torch.log(w[r]) - torch.log(w.sum()))
    return torch.stack(tokens), torch.stack(logs)


def _exact_mass(c, s):
    out = s["out"].double().clone()
    G = c["Hq"] // c["Hkv"]
    for b, n in enumerate(_lengths(c)):
        a = max(0, n - c["window"]) if c["window"] else 0
        k = s["x"][b, a:n].double()
        out[b, :, :n] = s["mass"][b, :, :n].double()
        for h in range(c["Hkv"]):
            z = s["q"][b, h * G:(h + 1) * G].double() @ k[:, h].T / math.sqrt(c["D"])
            out[b, h, a:n] += torch.softmax(z, dim=1).sum(0)
    return out


def _exact_prompt(c, s):
    q, k = s["q"].double(), s["k"].double()
    G, out, a, b = c["Hq"] // c["Hkv"], torch.zeros(c["Hkv"], s["k"].shape[0], dtype=torch.float64, device=DEV), 0, 0
    for n, p, (m, first) in zip(_ints(c["lens"]), _ints(c["past"]), _queries(c)):
        for h in range(c["Hq"]):
            for i in range(0, m, 2048):
                r = min(2048, m - i)
                end = first + i + r
                at = first + i + torch.arange(r, device=DEV)[:, None]
                j = torch.arange(end, device=DEV)[None]
                hidden = (j > at) | ((j <= at - c["window"]) if c["window"] else (j < 0))
                z = q[a + n - m + i:a + n - m + i + r, h] @ k[b:b + end, h // G].T / math.sqrt(c["D"])
                out[h // G, b:b + end] += torch.softmax(z.masked_fill(hidden, -math.inf), dim=1).sum(0)
        a, b = a + n, b + n + p
    return out


def _exact_evict(c, s):
    B, H, keep, D = c["B"], c["H"], c["keep"], c["D"]
    index = torch.full((B, H, keep), -1, dtype=torch.int32, device=DEV)
    mass = torch.zeros(B, H, keep, dtype=torch.float64, device=DEV)
    out = [torch.zeros(B, keep, H, D, dtype=torch.float64, device=DEV) for _ in "kv"]
    for b, n in enumerate(_lengths(c)):
        for h in range(H):
            m = s["mass"][b, h, :n].double()
            if n <= keep:
                at = torch.arange(n, device=DEV)
            else:
                first, latest = torch.arange(c["sinks"], device=DEV), torch.arange(n - c["recent"], n, device=DEV)
                mid = m[c["sinks"]:n - c["recent"]]
                some = keep - c["sinks"] - c["recent"]
                # by weight, equal ones by index: a stable sort of the row turned round
                order = (mid.numel() - 1) - torch.sort(mid.flip(0), stable=True).indices.flip(0)
                at = torch.cat([first, order[:some].sort().values + c["sinks"], latest])
            r = at.numel()
            index[b, h, :r], mass[b, h, :r] = at.int(), m[at]
            out[0][b, :r, h], out[1][b, :r, h] = s["xk"][b, at, h].double(), s["xv"][b, at, h].double()
    return index, mass, out[0], out[1]


_EXACT = {"sample": _exact_sample, "mass": _exact_mass, "prompt_mass": _exact_prompt, "evict": _exact_evict}


def exact(case, seed):
    return _EXACT[case["op"]](case, prepare(case, seed))
