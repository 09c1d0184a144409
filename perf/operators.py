"""What a decoder layer does around its caches, as cases to measure.

Each case names an operator (`op`) and its sizes:

  attention  prompt_attention: causal attention of packed prompts with grouped heads, each sequence's queries its
             last tokens (`past` keys before them), a whole prompt or a window of it
  append     rope_append_paged: one token of every sequence rotated at its position, keys and values into the pages
             of a bf16 pool or into the open pages of a compressed one, queries handed back
  rotate     rotate_prompt: queries and keys of packed prompts rotated at their positions, with or without the
             per-head norms of Qwen3
  norm       add_norm: a block's output (normed, gated, scaled) onto the residual stream, and the next block's norm

`own` chooses the framework's kernels; otherwise run computes the same in elementary torch operations."""
import math

import torch

DEV = "cuda"
PAGE = 16
EPS = 1e-6
own = False


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # a one-line chat prompt: latency
        dict(name="attention_short", op="attention", lens="97", past="0", Hq=32, Hkv=8, D=128, window=0),
        # a step's new prompts of mixed lengths, one empty, in a 28q/4kv model
        dict(name="attention_mixed", op="attention", lens="1201,17,640,0,333,1,1024,95,511,1500,64,702",
             past="0,0,0,0,0,0,0,0,0,0,0,0", Hq=28, Hkv=4, D=128, window=0),
        # a document of 8K tokens, the benchmark's context length: the largest
        dict(name="attention_8k", op="attention", lens="8192", past="0", Hq=32, Hkv=8, D=128, window=0),
        # the next piece of two long prompts, their earlier tokens already held
        dict(name="attention_chunk", op="attention", lens="512,301", past="4096,1999", Hq=32, Hkv=8, D=128, window=0),
        # a small model's head dim with sliding-window layers
        dict(name="attention_d64_window", op="attention", lens="4093,2048,777", past="0,0,0", Hq=14, Hkv=2, D=64,
             window=1024),
        # the largest head dim, one KV head
        dict(name="attention_d256", op="attention", lens="2051,1000", past="0,0", Hq=8, Hkv=1, D=256, window=0),
        # one chat sequence's token into plain pages: latency
        dict(name="append_one", op="append", cache="bf16", n=1, T=501, Hq=32, Hkv=8, D=128, norm=False),
        # a serving batch's tokens into compressed pages, sequences of mixed lengths, Qwen3's norms
        dict(name="append_batch", op="append", cache="compressed", n=128, T=4339, Hq=32, Hkv=8, D=128, norm=True),
        # the queries and keys of 8K prompt tokens in two sequences
        dict(name="rotate_8k", op="rotate", lens="5001,3191", Hq=32, Hkv=8, D=128, norm=True),
        # one token of one sequence between two blocks: latency
        dict(name="norm_one", op="norm", N=1, C=4096, post=False, gate="none", scale=1.0),
        # a serving batch's step, an odd row count
        dict(name="norm_batch", op="norm", N=621, C=4096, post=False, gate="none", scale=1.0),
        # 8K prompt tokens through norms on both sides of the block, a gate and a residual scale
        dict(name="norm_sandwich_8k", op="norm", N=8191, C=3584, post=True, gate="full", scale=0.22),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = [(32, 8), (28, 4), (32, 32), (16, 2), (14, 2), (40, 8), (24, 6), (8, 1), (64, 8)]


def draw(rng):
    op = rng.choice(["attention"] * 4 + ["append"] * 2 + ["rotate", "norm", "norm"])
    Hq, Hkv = rng.choice(_HEADS)
    D = rng.choice([128, 128, 64, 256])
    if op == "attention":
        S = rng.choice([1, 1, 2, 3, 5, 9, 16])
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
        window = rng.choice([0, 0, 0, _spread(rng, 1, 4096)])
        return dict(op=op, lens=",".join(map(str, lens)), past=",".join(map(str, past)), Hq=Hq, Hkv=Hkv, D=D,
                    window=window)
    if op == "append":
        return dict(op=op, cache=rng.choice(["bf16", "compressed"]), n=_spread(rng, 1, 256), T=_spread(rng, 2, 4339),
                    Hq=Hq, Hkv=min(Hkv, 8), D=D, norm=rng.random() < 0.3) | ({"Hq": 32} if Hkv > 8 else {})
    if op == "rotate":
        N = _spread(rng, 1, 8192 * 32 // max(Hq, 32))
        cut = rng.randint(0, N)
        return dict(op=op, lens="%d,%d" % (cut, N - cut), Hq=Hq, Hkv=Hkv, D=min(D, 128), norm=rng.random() < 0.5)
    C = _spread(rng, 64, 8192) if rng.random() < 0.5 else rng.choice([896, 2048, 3584, 4096, 5120, 8192])
    return dict(op=op, N=_spread(rng, 1, 8191 * 3584 // max(C, 3584)), C=C, post=rng.random() < 0.4,
                gate=rng.choice(["none", "none", "channel", "full"]), scale=rng.choice([1.0, 1.0, 0.22]))


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _ints(text):
    return [int(n) for n in text.split(",")]


def _offsets(lens):
    return torch.tensor([0] + lens, device=DEV).cumsum(0).int()


def _heads(g, n, H, D, sigma=0.5):
    """Rows of H heads with a scale for each channel, as projections give them."""
    return (_randn(g, n, H, D) * torch.exp(_randn(g, H, D) * sigma)).bfloat16()


def _tables(rows, D, theta=5e5):
    """fp32 cosines and sines [rows, D / 2] of a model's positions."""
    inv = theta ** (-torch.arange(D // 2, device=DEV, dtype=torch.float64) / (D // 2))
    ang = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _head_norms(c, g):
    w = [(1 + 0.1 * _randn(g, c["D"])).bfloat16() for _ in range(2)]
    return dict(q_norm=w[0], k_norm=w[1]) if c["norm"] else dict(q_norm=None, k_norm=None)


def _prepare_attention(c, g):
    lens, past = _ints(c["lens"]), _ints(c["past"])
    keys = [a + b for a, b in zip(lens, past)]
    return dict(q=_randn(g, sum(lens), c["Hq"], c["D"]).bfloat16(), k=_heads(g, sum(keys), c["Hkv"], c["D"]),
                v=_heads(g, sum(keys), c["Hkv"], c["D"]), cu_q=_offsets(lens), cu_k=_offsets(keys))


def _lengths(c):
    """Lengths of an append's sequences, the new token included: from a third of T up to T, none of which fills a
    page."""
    lens = [max(1, c["T"] - (i * 7 % c["n"]) * (c["T"] * 2 // 3) // c["n"]) for i in range(c["n"])]
    return [n - (n % PAGE == 0) for n in lens]


def _prepare_append(c, g):
    n, H, D = c["n"], c["Hkv"], c["D"]
    lens = _lengths(c)
    pages = [x // PAGE + 1 for x in lens]
    most, total = max(pages), sum(pages)
    owned = torch.randperm(total, generator=g, device=DEV).int()             # the pool's pages in no order
    first = torch.tensor([0] + pages, device=DEV).cumsum(0)[:-1]
    col = torch.arange(most, device=DEV)
    table = owned[(first[:, None] + col).clamp(max=total - 1)] * (col < torch.tensor(pages, device=DEV)[:, None])
    cos, sin = _tables(c["T"] + 1, D)
    s = dict(q=_heads(g, n, c["Hq"], D), k=_heads(g, n, H, D), v=_heads(g, n, H, D), cos=cos, sin=sin,
             lens=torch.tensor(lens, dtype=torch.int32, device=DEV), table=table.int().contiguous())
    if c["cache"] == "bf16":
        s["kbuf"], s["vbuf"] = (_randn(g, 1, total * PAGE, H, D).bfloat16() for _ in range(2))
    else:
        s["kbuf"], s["vbuf"] = (_compressed_pool(c, g, total, s["lens"], s["table"]) for _ in range(2))
    return s | _head_norms(c, g)


def _compressed_pool(c, g, pages, lens, table):
    """A compressed pool as its cache's encoder view: full pages of zeros, every sequence's open page held raw."""
    n, H, D = c["n"], c["Hkv"], c["D"]
    cap = n * H * PAGE
    raw = torch.zeros(cap + n * H * PAGE, D, dtype=torch.bfloat16, device=DEV)
    raw[cap:] = _randn(g, n * H * PAGE, D).bfloat16()
    u8, i32 = dict(dtype=torch.uint8, device=DEV), dict(dtype=torch.int32, device=DEV)
    mask, off = torch.zeros(1, pages, H, **i32), torch.zeros(1, pages, H, **i32)
    seq = torch.arange(n, device=DEV)
    opened = table[seq, (lens.long() - 1) // PAGE].long()
    mask[0, opened] = 0xFFFF
    off[0, opened] = (cap + torch.arange(n * H, device=DEV).view(n, H) * PAGE).int()
    return dict(sm=torch.zeros(1, pages * PAGE, H, D, **u8), code=torch.zeros(1, pages * PAGE, H, D // 2, **u8),
                base=torch.zeros(1, pages, H, D, **u8), rowmask=mask, rowoff=off, raw=raw, cnt=torch.zeros(1, **i32),
                before=torch.zeros(1, **i32), arrivals=torch.zeros(1, **i32), cap=cap, TS=pages * PAGE, H=H, D=D)


def _prepare_rotate(c, g):
    lens = _ints(c["lens"])
    cos, sin = _tables(max(lens), c["D"])
    return dict(q=_heads(g, sum(lens), c["Hq"], c["D"]), k=_heads(g, sum(lens), c["Hkv"], c["D"]), cos=cos, sin=sin,
                cu=_offsets(lens)) | _head_norms(c, g)


def _prepare_norm(c, g):
    N, C = c["N"], c["C"]
    gates = dict(none=lambda: None, channel=lambda: torch.sigmoid(_randn(g, C)).bfloat16(),
                 full=lambda: torch.sigmoid(_randn(g, N, C)).bfloat16())
    return dict(x=_randn(g, N, C).bfloat16(), r=(2 * _randn(g, N, C)).bfloat16(),
                w=(1 + 0.1 * _randn(g, C)).bfloat16(), pw=(1 + 0.1 * _randn(g, C)).bfloat16() if c["post"] else None,
                gate=gates[c["gate"]]())


def prepare(case, seed):
    return _OPS[case["op"]][0](case, _gen(seed)) | {"case": case}


# ---------------------------------------------------------------- plain forms

def _rows(cu, n, most):
    """Row index [S, most] of every token of a padded batch (clamped to the n rows) and whether it is one."""
    at = torch.arange(most, device=DEV)
    return (cu[:-1, None].long() + at).clamp(max=max(n - 1, 0)), at < (cu[1:] - cu[:-1])[:, None]


def _plain_attention(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    lens, past = _ints(c["lens"]), _ints(c["past"])
    S, Lq, Lk = len(lens), max(lens), max(a + b for a, b in zip(lens, past))
    qi, q_real = _rows(s["cu_q"], q.shape[0], Lq)
    ki, k_real = _rows(s["cu_k"], k.shape[0], Lk)
    qp = q[qi].float().view(S, Lq, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, -1, D)
    kp = k[ki].float().permute(0, 2, 3, 1).contiguous()                      # [S, Hkv, D, Lk]
    vp = v[ki].float().permute(0, 2, 1, 3).contiguous()                      # [S, Hkv, Lk, D]
    score = torch.matmul(qp, kp).view(S, Hkv, Hq // Hkv, Lq, Lk)
    score *= D ** -0.5
    nk, nq = s["cu_k"].diff(), s["cu_q"].diff()
    pos = (nk - nq)[:, None] + torch.arange(Lq, device=DEV)                   # the key a query stands at
    key = torch.arange(Lk, device=DEV)
    seen = (key <= pos[..., None]) & k_real[:, None]
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(top.masked_fill(top == -math.inf, 0)).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(S, Hkv, -1, Lk), vp).view(S, Hkv, Hq // Hkv, Lq, D)
    out /= total.masked_fill(total == 0, 1)
    return out.permute(0, 3, 1, 2, 4).reshape(S, Lq, Hq, D)[q_real].bfloat16()


def _plain_norm_rows(x, w):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _plain_turn(x, w, cos, sin):
    """Rows x [n, H, D], normed if w is given, rotated with the rows cos, sin [n, D / 2]: fp32."""
    x = x.float() if w is None else _plain_norm_rows(x, w)
    a, b = x.chunk(2, dim=-1)
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _plain_append(s):
    c, D = s["case"], s["case"]["D"]
    pos = s["lens"].long() - 1
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _plain_turn(s["q"], s["q_norm"], cos, sin).bfloat16()
    k = _plain_turn(s["k"], s["k_norm"], cos, sin).bfloat16()
    seq = torch.arange(c["n"], device=DEV)
    if c["cache"] == "bf16":
        page = s["table"][seq, pos // PAGE].long()
        row = page * PAGE + pos % PAGE
        s["kbuf"][0, row] = k
        s["vbuf"][0, row] = s["v"]
        return q, s["kbuf"], s["vbuf"]
    kraw, vraw = s["kbuf"]["raw"], s["vbuf"]["raw"]
    unit = seq[:, None] * c["Hkv"] + torch.arange(c["Hkv"], device=DEV)
    row = s["kbuf"]["cap"] + unit * PAGE + (pos % PAGE)[:, None]
    kraw[row] = k
    vraw[row] = s["v"]
    return q, kraw.view(-1, PAGE, D), vraw.view(-1, PAGE, D)


def _plain_rotate(s):
    t = torch.arange(s["q"].shape[0], device=DEV)
    cu = s["cu"].long()
    pos = t - cu[torch.searchsorted(cu[1:].contiguous(), t, right=True)]
    cos, sin = s["cos"][pos], s["sin"][pos]
    return (_plain_turn(s["q"], s["q_norm"], cos, sin).bfloat16(), _plain_turn(s["k"], s["k_norm"], cos, sin).bfloat16())


def _plain_norm(s):
    u = s["x"].float() if s["pw"] is None else _plain_norm_rows(s["x"], s["pw"])
    if s["gate"] is not None:
        u = u * s["gate"].float()
    h = s["r"].float() + s["case"]["scale"] * u
    return h.bfloat16(), _plain_norm_rows(h, s["w"]).bfloat16()


# ---------------------------------------------------------------- the framework's operators

def _own_attention(s):
    import exactkv_amd as exactkv
    return exactkv.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], cu_seqlens_k=s["cu_k"],
                                    window=s["case"]["window"])


def _own_append(s):
    import exactkv_amd as exactkv
    q = exactkv.rope_append_paged(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["kbuf"], s["vbuf"], s["lens"],
                                  s["table"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
    if s["case"]["cache"] == "bf16":
        return q, s["kbuf"], s["vbuf"]
    D = s["case"]["D"]
    return q, s["kbuf"]["raw"].view(-1, PAGE, D), s["vbuf"]["raw"].view(-1, PAGE, D)


def _own_rotate(s):
    import exactkv_amd as exactkv
    return exactkv.rotate_prompt(s["q"], s["k"], s["cos"], s["sin"], s["cu"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                                 eps=EPS)


def _own_norm(s):
    import exactkv_amd as exactkv
    return exactkv.add_norm(s["x"], s["r"], s["w"], eps=EPS, post_weight=s["pw"], gate=s["gate"],
                            scale=s["case"]["scale"])


_OPS = {"attention": (_prepare_attention, _plain_attention, _own_attention),
        "append": (_prepare_append, _plain_append, _own_append),
        "rotate": (_prepare_rotate, _plain_rotate, _own_rotate),
        "norm": (_prepare_norm, _plain_norm, _own_norm)}


def run(state):
    return _OPS[state["case"]["op"]][2 if own else 1](state)


# ---------------------------------------------------------------- what a pass cannot do without

def _pairs(lens, past, window):
    """Visible (query, key) pairs."""
    total = 0
    for n, p in zip(lens, past):
        if window == 0:
            total += n * p + n * (n + 1) // 2
        else:                                          # query i sees min(p + i + 1, window) keys
            short = max(0, min(n, window - p - 1))      # queries whose window is not yet full
            total += short * p + short * (short + 1) // 2 + (n - short) * window
    return total


def work(case):
    c = case
    if c["op"] == "attention":
        lens, past = _ints(c["lens"]), _ints(c["past"])
        keys = sum(min(n + p, n + c["window"] - 1) if c["window"] and n else (n + p if n else 0)
                   for n, p in zip(lens, past))
        return {"bytes": 2 * c["D"] * (2 * sum(lens) * c["Hq"] + 2 * keys * c["Hkv"]) + 8 * (len(lens) + 1),
                "flops": 4 * c["D"] * c["Hq"] * _pairs(lens, past, c["window"])}
    if c["op"] == "append":
        rows, D = c["n"] * (c["Hq"] + 2 * c["Hkv"]), c["D"]
        return {"bytes": 4 * D * rows + 4 * D * c["n"] + 8 * c["n"],
                "flops": c["n"] * D * (c["Hq"] + c["Hkv"]) * (7 if c["norm"] else 3)}
    if c["op"] == "rotate":
        lens, D = _ints(c["lens"]), c["D"]
        return {"bytes": 4 * D * sum(lens) * (c["Hq"] + c["Hkv"]) + 4 * D * max(lens),
                "flops": sum(lens) * D * (c["Hq"] + c["Hkv"]) * (7 if c["norm"] else 3)}
    full = c["gate"] == "full"
    return {"bytes": 2 * c["N"] * c["C"] * (4 + full) + 2 * c["C"] * (1 + c["post"] + (c["gate"] == "channel")),
            "flops": c["N"] * c["C"] * (6 + 4 * c["post"] + (c["gate"] != "none"))}


# ---------------------------------------------------------------- the definitions, in 64 bits

def _exact_attention(c, s):
    q, k, v = (s[x].double() for x in "qkv")
    G, out, a, b = c["Hq"] // c["Hkv"], torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV), 0, 0
    for n, p in zip(_ints(c["lens"]), _ints(c["past"])):
        for h in range(c["Hq"]):
            for i in range(0, n, 2048):
                m = min(2048, n - i)
                at = p + i + torch.arange(m, device=DEV)[:, None]
                j = torch.arange(p + i + m, device=DEV)[None]
                hidden = (j > at) | ((j <= at - c["window"]) if c["window"] else (j < 0))
                z = q[a + i:a + i + m, h] @ k[b:b + p + i + m, h // G].T / math.sqrt(c["D"])
                z = torch.softmax(z.masked_fill(hidden, -math.inf), dim=1)
                out[a + i:a + i + m, h] = z @ v[b:b + p + i + m, h // G]
        a, b = a + n, b + n + p
    return out


def _exact_turn(x, w, cos, sin, pos):
    x = x.double()
    if w is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
    z = torch.complex(x[..., : x.shape[-1] // 2], x[..., x.shape[-1] // 2:])
    z = z * torch.complex(cos.double(), sin.double())[pos][:, None]
    return torch.cat([z.real, z.imag], dim=-1)


def _exact_append(c, s):
    pos = torch.tensor([n - 1 for n in _lengths(c)], device=DEV)
    q = _exact_turn(s["q"], s["q_norm"], s["cos"], s["sin"], pos)
    new = {"kbuf": _exact_turn(s["k"], s["k_norm"], s["cos"], s["sin"], pos), "vbuf": s["v"].double()}
    out = [q]
    for name in ("kbuf", "vbuf"):
        if c["cache"] == "bf16":
            pool = s[name].double()
            for i, p in enumerate(pos.tolist()):
                pool[0, int(s["table"][i, p // PAGE]) * PAGE + p % PAGE] = new[name][i]
        else:
            pool = s[name]["raw"].double().view(-1, PAGE, c["D"])
            for i, p in enumerate(pos.tolist()):
                first = s[name]["cap"] // PAGE + i * c["Hkv"]
                pool[first:first + c["Hkv"], p % PAGE] = new[name][i]
        out.append(pool)
    return tuple(out)


def _exact_rotate(c, s):
    pos = torch.cat([torch.arange(n, device=DEV) for n in _ints(c["lens"])])
    return tuple(_exact_turn(s[x], s[x + "_norm"], s["cos"], s["sin"], pos) for x in "qk")


def _exact_norm(c, s):
    def unit(z):
        return z / (z.pow(2).sum(-1, keepdim=True) / c["C"] + EPS).sqrt()
    u = s["x"].double()
    if c["post"]:
        u = unit(u) * s["pw"].double()
    if c["gate"] != "none":
        u = u * s["gate"].double()
    h = s["r"].double() + c["scale"] * u
    return h, unit(h) * s["w"].double()


_EXACT = {"attention": _exact_attention, "append": _exact_append, "rotate": _exact_rotate, "norm": _exact_norm}


def exact(case, seed):
    return _EXACT[case["op"]](case, prepare(case, seed))
