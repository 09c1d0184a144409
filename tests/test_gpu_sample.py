"""sample against its definition in 64 bits, row by row on the CPU: sizes around the kernel's pieces and lists, each cut
and all of them, ties, hidden and non-finite logits, strides, streams and graphs.

Tokens have to be equal: the kernel's weights are within 2^-44 + 2^-50 of the definition's, so that a cut moves only
where a sum comes within 2^-24 of its bound, of which the cases with random logits have none. The log-probability
is a double rounded to fp32 once, from weights of at least 2^-44 with 2^-44 of error: cases whose chosen tokens weigh 2^-20
at least are within 2^-23 absolute and 2^-24 relative.

No counterpart in the reference (greedy decoding, exactkv/engine.py:93-95)."""
import math

import pytest
import torch

import exactkv_amd as exactkv
from exactkv_amd import _lib, kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _row(l, u, t, k, p, m):
    """(token, log-probability) of one row of logits [V] in fp64 on the CPU."""
    l = torch.where(torch.isnan(l), -math.inf, l)
    order = torch.sort(l, descending=True, stable=True).indices
    if not t > 0:
        return int(order[0]), 0.0
    top = l[order[0]]
    z = torch.where(l[order] == top, 0.0, (l[order] - top) / t)
    w = torch.where(l[order] == -math.inf, 0.0, torch.exp(z))
    n = int(((w >= m) & (w > 0)).sum())
    if k > 0:
        n = min(n, k)
    w = w[:n]
    total = torch.cumsum(w, 0)
    if p < 1:
        n = max(1, int((total - w < p * total[-1]).sum()))
        w, total = w[:n], total[:n]
    r = min(int((total <= u * total[-1]).sum()), n - 1)
    return int(order[r]), math.log(w[r] / total[-1])


def _check(logits, u, t=1.0, k=0, p=1.0, m=0.0):
    token, lp = exactkv.sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=m, logprob=True)
    assert token.dtype == torch.int64 and lp.dtype == torch.float32
    assert torch.equal(token, exactkv.sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=m))
    B = logits.shape[0]
    rows = [torch.as_tensor(v).to(torch.float32).double().expand(B) if not torch.is_tensor(v) else v.double().cpu() for v in (t, p, m)]
    ks = torch.as_tensor(k).expand(B) if not torch.is_tensor(k) else k.cpu()
    x, us = logits.double().cpu(), u.double().cpu()
    for b in range(B):
        want, wlp = _row(x[b], float(us[b]), float(rows[0][b]), int(ks[b]), float(rows[1][b]), float(rows[2][b]))
        assert int(token[b]) == want, (b, int(token[b]), want)
        if wlp > -13.8:
            assert abs(float(lp[b]) - wlp) <= 2.0 ** -23 + 2.0 ** -24 * abs(wlp), (b, float(lp[b]), wlp)
    return token


def _logits(B, V, seed, dtype=torch.bfloat16, sigma=2.2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(B, V, generator=g, device=DEV) * sigma
    x[:, torch.randint(V, (min(V, 20),), generator=g, device=DEV)] += 6
    return x.to(dtype), torch.rand(B, generator=g, device=DEV)


SIZES = [1, 2, 3, 7, 8, 9, 63, 64, 65, 1000, 2047, 2048, 2049, 4096, 4097, 8191, 8192, 8193, 16385, 32003, 50257, 65537, 128256, 152064]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("V", SIZES)
def test_sizes(V, dtype):
    print("[case]", V, dtype, flush=True)
    x, u = _logits(3, V, V, dtype)
    _check(x, u)
    _check(x, u, t=0.7, k=50, p=0.9)
    _check(x, u, p=0.95)


@pytest.mark.parametrize("m", [0.0, 0.05, 1.0])
@pytest.mark.parametrize("p", [1.0, 0.999, 0.5, 1e-6, 0.0])
@pytest.mark.parametrize("k", [0, 1, 2, 64, 2048, 2049, 7000, 10 ** 9])
@pytest.mark.parametrize("t", [0.0, 0.05, 1.0, 30.0])
def test_cuts(t, k, p, m):
    print("[case]", t, k, p, m, flush=True)
    x, u = _logits(2, 9001, 5)
    _check(x, u, t, k, p, m)


@pytest.mark.parametrize("B", [1, 2, 5, 33, 200])
def test_settings_of_each_row(B):
    x, u = _logits(B, 20011, B)
    g = torch.Generator(device=DEV).manual_seed(B + 1)

    def r():
        return torch.rand(B, generator=g, device=DEV)
    t = torch.where(r() < 0.2, 0.0, 0.2 + r())
    k = torch.where(r() < 0.4, 0, torch.randint(1, 5000, (B,), generator=g, device=DEV)).int()
    p = torch.where(r() < 0.4, 1.0, r())
    m = torch.where(r() < 0.5, 0.0, 0.1 * r())
    _check(x, u, t, k, p, m)


@pytest.mark.parametrize("V", [5, 4096, 5000, 100000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_equal_logits(V, dtype):
    """Every cut falls among ties, which go by index; their sums are whole numbers, exact in any order."""
    x = torch.full((7, V), -3.25, device=DEV, dtype=dtype)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 0.125, 0.3], device=DEV)
    assert int(_check(x, u)[0]) == 0
    _check(x, u, p=0.5)
    _check(x, u, k=3)
    _check(x, u, k=min(V, 4500), p=0.25)
    _check(x, u, m=1.0)


@pytest.mark.parametrize("k", [0, 40, 3000])
def test_few_distinct_logits(k):
    """Thousands of ties at each of a few values, more than one list holds, in mixed order."""
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randint(0, 4, (4, 60001), generator=g, device=DEV).bfloat16() * 0.5
    x[1] *= -1
    u = torch.rand(4, generator=g, device=DEV)
    _check(x, u, k=k)
    _check(x, u, p=0.37, k=k)
    _check(x, u, t=0.5, p=0.9, m=0.2, k=k)


@pytest.mark.parametrize("V", [5000, 20001])
@pytest.mark.parametrize("n", [1, 5, 63, 64, 65, 255, 256, 257, 300, 511, 512, 513, 640, 1000, 1023, 1024, 1025, 1500, 2048, 2049, 3000, 4096])
def test_near_ones_of_every_number(V, n):
    """n logits so near each other that no bin tells them apart, anywhere in the row and in any order; u and the cuts take
    places all over them. (Weights within 2^-9 of each other: n <= 2^12 of them leave no sum within 2^-24 of a bound but
    by chance, which seeds decide for both sides alike.)"""
    print("[case]", V, n, flush=True)
    g = torch.Generator(device=DEV).manual_seed(n)
    x = torch.full((4, V), -9.0, device=DEV)
    at = torch.stack([torch.randperm(V, generator=g, device=DEV)[:n] for _ in range(4)])
    near = 2.0 + torch.rand(4, n, generator=g, device=DEV) * 2.0 ** -9
    near[2:] = (near[2:] * 2.0 ** 14).round() * 2.0 ** -14                    # 32 values: ties
    x.scatter_(1, at, near)
    u = torch.tensor([0.03, 0.98, 0.51, 0.7], device=DEV)
    _check(x, u, m=0.5)
    _check(x, u, p=0.6, m=0.5)
    _check(x, u, k=(n + 1) // 2)
    _check(x, u, k=n, p=0.9)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_hidden_logits(dtype):
    """Masked tokens at -infinity, the type's lowest value and NaN, most of a row or all but one."""
    low = torch.finfo(dtype).min
    x, u = _logits(6, 10007, 11, dtype)
    x[0, 100:] = -math.inf
    x[1, :-1] = -math.inf
    x[2, 50:] = low
    x[3, ::2] = math.nan
    x[4, :5000] = -math.inf
    x[4, 5000:] = low
    x[5, 1:] = math.nan
    for kw in ({}, dict(k=50), dict(p=0.9), dict(t=0.0), dict(t=0.3, k=4000, p=0.5, m=0.01)):
        _check(x, u, **kw)


def test_infinite_logits():
    x, u = _logits(2, 3001, 12, torch.float32)
    x[0, [5, 77, 2000]] = math.inf
    x[1] = 3e38
    x[1, 9] = -3e38
    _check(x, u)
    _check(x, u, k=2)
    _check(x, u, t=0.0)


def test_signed_zeros_tie():
    x = torch.zeros(1, 4097, device=DEV)
    x[0, ::2] = -0.0
    for u in (0.0, 0.3, 0.9):
        _check(x, torch.tensor([u], device=DEV))


def test_far_logits_and_temperatures():
    x, u = _logits(3, 5003, 13, torch.float32)
    _check(x * 1e4, u, p=0.9)
    _check(x * 1e-5, u, p=0.9)                         # all in one bin
    _check(x, u, t=1e-6)
    _check(x, u, t=1e6, k=4500)
    _check(x + 1e5, u, p=0.8)


@pytest.mark.parametrize("V", [5003, 20011])
def test_far_logits_and_temperatures_of_every_path(V):
    """Temperatures from fp32's least to infinity, logits up to its ends, one row's largest infinite."""
    x, u = _logits(3, V, 15, torch.float32)
    for t in (1e-45, 1e-30, 1e-6, 1e6, 1e30, 3e38, math.inf):
        _check(x, u, t=t)
        _check(x, u, t=t, p=0.7)
        _check(x, u, t=t, k=700, p=0.9)
    for y in (x * 1e4, x * 1e-5, x + 1e5, x * 1e-38, x * 1e37):
        _check(y, u, p=0.9)
        _check(y, u, k=900)
        _check(y, u, t=1e37, p=0.6, k=3000)
    x[0, [5, 77, V - 1]] = math.inf
    x[1] = 3e38
    x[1, 9] = -3e38
    _check(x, u)
    _check(x, u, k=2)
    _check(x, u, t=0.0)
    _check(x, u, t=1e38, p=0.5)


def test_nothing_to_draw():
    x, u = _logits(3, 999, 14)
    x[1] = -math.inf
    x[2] = math.nan
    token, lp = exactkv.sample(x, u, logprob=True)
    assert token[1:].tolist() == [0, 0] and lp[1:].tolist() == [-math.inf] * 2
    assert int(token[0]) == int(exactkv.sample(x[:1], u[:1])[0])
    assert kernels.error_bits(clear=True) == 0x400 and "logit" in _lib.describe_errors(0x400)


@pytest.mark.parametrize("V", [999, 9000])
def test_entries_out_of_range(V):
    """Settings given as tensors, and u, beyond their ranges count as the nearest value in them; NaN draws some token."""
    x, u = _logits(6, V, 16)

    def row(v, dtype=torch.float32):
        return torch.full((6,), v, device=DEV, dtype=dtype)
    for bad, ok in ((dict(temperature=row(-1.0)), dict(temperature=0.0)), (dict(temperature=row(-math.inf)), dict(temperature=0.0)),
                    (dict(top_k=row(-3, torch.int32)), {}), (dict(top_p=row(1.5)), {}), (dict(top_p=row(-0.5)), dict(top_p=0.0)),
                    (dict(min_p=row(-1.0)), {}), (dict(min_p=row(7.0)), dict(min_p=1.0))):
        got, want = (exactkv.sample(x, u, logprob=True, **kw) for kw in (bad, ok))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for name in ("temperature", "top_p", "min_p"):
        got = exactkv.sample(x, u, **{name: row(math.nan)})
        assert ((got >= 0) & (got < V)).all()
    for v, w in ((-1.0, 0.0), (2.0, 1 - 2.0 ** -24), (math.inf, 1 - 2.0 ** -24)):
        assert torch.equal(exactkv.sample(x, row(v)), exactkv.sample(x, row(w)))


@pytest.mark.parametrize("V", [8192, 8193, 70000])
def test_rows_with_nothing_to_draw_among_others(V):
    x, u = _logits(4, V, 17)
    x[1] = -math.inf
    x[2] = math.nan
    token, lp = exactkv.sample(x, u, logprob=True)
    assert kernels.error_bits(clear=True) == 0x400
    assert token[1:3].tolist() == [0, 0] and torch.isneginf(lp[1:3]).all()
    _check(x[::3], u[::3].contiguous())


def test_u_out_of_range_is_clamped():
    x, _ = _logits(4, 2000, 15)
    x[:] = x[0]
    u = torch.tensor([-1.0, 1.0, 2.0, math.nan], device=DEV)
    same = torch.tensor([0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.0], device=DEV)
    assert torch.equal(exactkv.sample(x, u), exactkv.sample(x, same))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_strided_and_unaligned_rows(dtype):
    x, u = _logits(4, 12000, 16, dtype)
    for a, z in ((1, 11000), (3, 9002), (5, 5006)):
        _check(x[:, a:z], u, p=0.9)
    _check(x[::2, 7:], u[:2].contiguous(), k=20)
    _check(x[:1].expand(4, -1), u)


def test_no_rows():
    assert exactkv.sample(torch.zeros(0, 10, device=DEV), torch.zeros(0, device=DEV)).shape == (0,)


def test_another_stream_and_two_at_once():
    x, u = _logits(64, 50257, 17)
    y, v = _logits(3, 128256, 18)
    want, other = exactkv.sample(x, u, top_p=0.9), exactkv.sample(y, v)
    s = [torch.cuda.Stream() for _ in range(2)]
    for i in s:
        i.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(s[0]):
            a = exactkv.sample(x, u, top_p=0.9)
        with torch.cuda.stream(s[1]):
            b = exactkv.sample(y, v)
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, other)


@pytest.mark.parametrize("B,V", [(1, 128256), (40, 32000)])
def test_graph_replays_follow_their_inputs(B, V):
    x, u = _logits(B, V, 19)
    t = torch.ones(B, device=DEV)
    k = torch.zeros(B, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        exactkv.sample(x, u, temperature=t, top_k=k, top_p=0.9)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = exactkv.sample(x, u, temperature=t, top_k=k, top_p=0.9)
    for seed in range(4):
        nx, nu = _logits(B, V, 20 + seed)
        x.copy_(nx)
        u.copy_(nu)
        t.fill_(0.5 + 0.2 * seed)
        k.fill_([0, 50, 5000, 1][seed])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, exactkv.sample(x, u, temperature=t, top_k=k, top_p=0.9))
        _check(x, u, t, k, 0.9)


def test_refusals():
    x, u = _logits(4, 100, 30)
    ok = dict(temperature=1.0)
    for bad in (dict(temperature=-1.0), dict(top_k=-1), dict(top_k=1.5), dict(top_p=1.1), dict(top_p=-0.1), dict(min_p=2.0), dict(min_p=math.nan),
                dict(temperature=torch.ones(3, device=DEV)), dict(temperature=torch.ones(4)), dict(top_k=torch.ones(4, device=DEV)),
                dict(top_p=torch.ones(4, device=DEV, dtype=torch.float64)), dict(min_p="a"), dict(top_k=2 ** 31), dict(temperature=True)):
        with pytest.raises(ValueError):
            exactkv.sample(x, u, **(ok | bad))
    for a, b in ((x.double(), u), (x[0], u), (x.t(), torch.rand(100, device=DEV)), (x, u[:3]), (x, u.double()), (x, u.cpu()), (x.cpu(), u),
                 (torch.zeros(2, 0, device=DEV), u[:2]), (torch.zeros(1, 2 ** 19 + 1, device=DEV), u[:1])):
        with pytest.raises(ValueError):
            exactkv.sample(a, b)
