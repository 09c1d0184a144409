"""prompt_attention against the formula in 64 bits: packed sequences of every length around the
tiles' edges, empty ones, continued prompts, windows, rows that see no key, head layouts and head
dims, strided inputs, infinities and NaN where a row does not look, graphs and streams.

Tolerance, per value: the store rounds by at most 2^-8 of it; each weight is rounded to bf16, at
most 2^-8 of it, so the sum is off by at most 2^-8 of sum_j p_j |v_j| =: A; what is left is fp32:
a score of D products is off by at most D 2^-24 sum_i |q_i k_i| / sqrt(D) (256 x 2^-24 x 170 / 16 =
2^-12.6 for normal q, k at D = 256), a weight by that, the exponential's 2^-22 and 2^-23 of its
argument (below 2^5), the sums by 2^-24 per key (a few hundred here): below 2^-11 of A together.

No counterpart in the reference (its prefill is the model's own forward pass, engine.py:42-49)."""
import math

import pytest
import torch

import exactkv_amd as exactkv
from exactkv_amd import kernels
from tests.conftest import same_bits

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(lens, keys, Hq, Hkv, D, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rows(n, H):
        return torch.randn(n, H, D, generator=g, device=DEV).bfloat16()
    return rows(sum(lens), Hq), rows(sum(keys), Hkv), rows(sum(keys), Hkv)


def _cu(lens):
    return torch.tensor([0] + list(lens), device=DEV).cumsum(0).int()


def _formula(q, k, v, lens, keys, window):
    """(out, sum_j p_j |v_j|) in 64 bits."""
    Hq, D, G = q.shape[1], q.shape[2], q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(out)
    a = b = 0
    for n, m in zip(lens, keys):
        if n and m:
            kk = k[b:b + m].double().repeat_interleave(G, dim=1).permute(1, 2, 0).contiguous()
            vv = v[b:b + m].double().repeat_interleave(G, dim=1).transpose(0, 1).contiguous()
            s = torch.matmul(q[a:a + n].double().transpose(0, 1).contiguous(), kk) / math.sqrt(D)
            p = torch.arange(n, device=DEV)[:, None] + (m - n)
            j = torch.arange(m, device=DEV)[None]
            seen = (j <= p) & ((j > p - window) if window else (j >= 0))
            s = s.masked_fill(~seen, -math.inf)
            w = torch.softmax(s, dim=-1).masked_fill(~seen.any(1)[None, :, None], 0)
            out[a:a + n] = torch.matmul(w, vv).transpose(0, 1)
            mag[a:a + n] = torch.matmul(w, vv.abs()).transpose(0, 1)
        a, b = a + n, b + m
    return out, mag


def _check(got, want, mag):
    err = (got.double() - want).abs()
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -11) * mag + 1e-30
    assert torch.isfinite(got).all()
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"error {worst:.2f} times the bound"


def _run(lens, Hq, Hkv, D, window=0, keys=None, seed=0):
    past = keys is not None
    keys = lens if keys is None else keys
    q, k, v = _inputs(lens, keys, Hq, Hkv, D, seed)
    print("[case]", lens, keys, Hq, Hkv, D, window, flush=True)
    got = exactkv.prompt_attention(q, k, v, _cu(lens), cu_seqlens_k=_cu(keys) if past else None, window=window)
    assert got.shape == q.shape and got.dtype == torch.bfloat16 and got.is_contiguous()
    _check(got, *_formula(q, k, v, lens, keys, window))
    return got


LENS = [[1], [2], [31], [32], [33], [63], [64], [65], [127, 1], [128, 129], [255, 0, 257], [0, 0, 5, 0], [1] * 20,
        [300, 17, 1, 64, 500]]


@pytest.mark.parametrize("lens", LENS, ids=str)
def test_lengths_around_the_tiles(lens):
    _run(lens, 8, 2, 128)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (4, 4), (8, 1), (14, 2), (28, 4), (24, 6), (40, 8), (34, 2)])
def test_head_layouts(Hq, Hkv, D):
    _run([70, 1, 129], Hq, Hkv, D, seed=Hq)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 2, 31, 63, 64, 65, 100, 1000])
def test_windows(window, D):
    _run([1, 64, 200, 333], 8, 2, D, window=window, seed=window)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,keys", [([1], [500]), ([5, 70], [5, 300]), ([100, 3, 0], [129, 400, 50]), ([64], [64]),
                                       ([17, 33], [1000, 77])], ids=str)
@pytest.mark.parametrize("window", [0, 50])
def test_continued_prompts(lens, keys, window, D):
    _run(lens, 8, 4, D, window=window, keys=keys, seed=3)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_that_see_no_key_are_zero(D):
    """Fewer keys than queries: the first queries stand before the first key; no keys at all."""
    got = _run([40, 9, 64], 8, 2, D, keys=[10, 0, 3])
    assert (got[:30] == 0).all() and (got[40:49] == 0).all() and (got[49:110] == 0).all()


SPLIT = [([1], [3000], 8, 8, 0), ([40, 1, 200], [2500, 40, 900], 8, 2, 0), ([17, 0, 130], [1500, 0, 130], 14, 2, 700),
         ([700], [700], 4, 1, 0), ([3, 5, 2, 8], [5, 1000, 2, 700], 32, 8, 0), ([1] * 70, list(range(600, 670)), 4, 1, 0),
         ([64, 30], [20, 1200], 8, 2, 0), ([17, 0, 130], [3500, 0, 130], 14, 2, 2000)]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,keys,Hq,Hkv,window", SPLIT, ids=lambda x: str(x)[:24])
def test_few_rows_split_their_keys(lens, keys, Hq, Hkv, window, D):
    """Calls with few rows and many keys take a workspace and split the keys; rows without a key
    among them are 0, rows that no sequence holds as without a split."""
    from exactkv_amd import _lib
    # at head dim 64 and 128, 700 keys (all, or a window's) are too few tiles to split
    if max(keys) > 700 and window != 700:
        assert _lib.load().exkv_prompt_workspace(len(lens), sum(lens), sum(keys), Hq, Hkv, D, window) > 0
    got = _run(lens, Hq, Hkv, D, window=window, keys=keys, seed=41)
    q, k, v = _inputs(lens, keys, Hq, Hkv, D, 41)
    tail = torch.cat([q, q[:3]])
    assert same_bits(exactkv.prompt_attention(tail, k, v, _cu(lens), cu_seqlens_k=_cu(keys), window=window)[:sum(lens)], got)
    out = torch.full_like(tail, 7.0)
    exactkv.prompt_attention(tail, k, v, _cu(lens), cu_seqlens_k=_cu(keys), window=window, out=out)
    assert (out[sum(lens):] == 7).all() and same_bits(out[:sum(lens)], got)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (2, 2)])
@pytest.mark.parametrize("window", [897, 961, 993, 1024, 1090, 1921, 2017])
def test_split_windows_that_begin_within_a_tile(window, Hq, Hkv, D):
    """A window of a whole number of key tiles that begins within one reaches into one more."""
    _run([64, 5, 33], Hq, Hkv, D, window=window, keys=[3001, 2500, 1800], seed=45)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq", [3, 5, 7])
@pytest.mark.parametrize("extra", [0, 24, 40, 56])
def test_split_windows_where_groups_begin_within_a_tile(extra, Hq, D):
    """Row tiles of 128 rows hold parts of a token's heads at both ends, one token more than whole ones."""
    _run([37, 28, 280], Hq, 1, D, window=432 + extra, keys=[37, 14, 709], seed=50)
    _run([37, 28, 280], Hq, 1, D, window=1008 + extra, keys=[37, 14, 2709], seed=51)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,keys,Hq,Hkv", [([700, 1, 300], [700, 3000, 1999], 8, 4), ([1] * 40, [1500] * 40, 8, 2),
                                              ([513], [4000], 16, 4), ([2051, 90], [2051, 1500], 8, 1),
                                              ([1] * 64, list(range(900, 964)), 4, 1)], ids=lambda x: str(x)[:24])
def test_split_tiles_of_many_lengths(lens, keys, Hq, Hkv, D):
    _run(lens, Hq, Hkv, D, keys=keys, seed=46)


@pytest.mark.parametrize("lens,Hq,Hkv", [([2048], 16, 4), ([1000, 900, 1100, 17], 16, 4), ([600] * 7, 4, 4), ([2500], 16, 8)],
                         ids=lambda x: str(x)[:24])
def test_head_dim_256_at_one_and_two_workgroups_a_cu(lens, Hq, Hkv):
    _run(lens, Hq, Hkv, 256, seed=47)


@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("lens", [[1100], [500, 1, 0, 620]], ids=str)
def test_head_dim_256_two_workgroups_a_cu(lens, window):
    """Calls of many row tiles take the other instance; a bad value reaches the rows that see it."""
    _run(lens, 64, 64, 256, window=window, seed=49)
    q, k, v = _inputs(lens, lens, 64, 64, 256, 49)
    at = lens[0] - 40
    v[at, 3] = math.nan
    got = exactkv.prompt_attention(q, k, v, _cu(lens), window=window)
    assert got[at:lens[0], 3].isnan().all()
    got[at:lens[0], 3] = 0
    v[at, 3] = 0
    want, mag = _formula(q, k, v, lens, lens, window)
    want[at:lens[0], 3] = 0
    _check(got, want, mag)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_split_rows_with_bad_values(D):
    """The joined result of split keys is checked for the rows that must not see a bad value, too."""
    lens, keys = [30], [2000]
    q, k, v = _inputs(lens, keys, 4, 2, D, 43)
    v[1985, 1] = float("nan")                          # seen by the queries from key 1985 on, of KV head 1
    got = exactkv.prompt_attention(q, k, v, _cu(lens), cu_seqlens_k=_cu(keys))
    seen = torch.zeros(30, 4, dtype=torch.bool, device=DEV)
    seen[15:, 2:] = True
    v[1985, 1] = 0
    want, mag = _formula(q, k, v, lens, keys, 0)
    assert got[seen].isnan().all() and torch.isfinite(got[~seen]).all()
    err = (got.double() - want).abs() - (2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -11) * mag)
    assert (err[~seen] <= 0).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("lens,keys", [([300, 40], [200, 25]), ([700, 33, 500], [0, 33, 100]), ([257] * 5, [1, 257, 0, 300, 60]),
                                       ([900, 5], [100, 4000])], ids=str)
def test_many_more_queries_than_keys(lens, keys, window, D):
    """Whole row tiles that see no key are taken like the others."""
    _run(lens, 8, 2, D, window=window, keys=keys, seed=53)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("lens,keys", [([35], [26]), ([300, 40], [200, 25]), ([70, 5], [20, 2500])], ids=str)
def test_bad_values_do_not_reach_rows_that_see_no_key(lens, keys, bad, D):
    q, k, v = _inputs(lens, keys, 8, 2, D, 52)
    want, mag = _formula(q, k, v, lens, keys, 0)
    v[3] = bad                                         # key 3 of the first sequence
    k[7] = math.nan
    got = exactkv.prompt_attention(q, k, v, _cu(lens), cu_seqlens_k=_cu(keys))
    none = lens[0] - keys[0]
    assert (got[:none] == 0).all()
    _check(got[none:none + 3], want[none:none + 3], mag[none:none + 3])
    assert got[none + 7:lens[0]].isnan().all()
    _check(got[lens[0]:], want[lens[0]:], mag[lens[0]:])


def test_split_rows_without_a_finite_score():
    q, k, v = _inputs([5], [2000], 1, 1, 64, 44)
    q[:] = 1.0
    k[:] = -math.inf
    assert exactkv.prompt_attention(q, k, v, _cu([5]), cu_seqlens_k=_cu([2000])).isnan().all()
    k[1997] = 0.25                                     # the third query's own token
    got = exactkv.prompt_attention(q, k, v, _cu([5]), cu_seqlens_k=_cu([2000]))
    assert got[:2].isnan().all() and same_bits(got[2:], v[1997:1998].expand(3, 1, 64).contiguous())


def test_no_keys_at_all_and_the_widest_windows():
    q, k, v = _inputs([9], [9], 8, 2, 128, 45)
    got = exactkv.prompt_attention(q, k[:0], v[:0], _cu([4, 5]), cu_seqlens_k=_cu([0, 0]))
    assert (got == 0).all()
    whole = exactkv.prompt_attention(q, k, v, _cu([9]))
    for window in (9, 10, 1 << 30, 0x7FFFFFFF):
        assert same_bits(exactkv.prompt_attention(q, k, v, _cu([9]), window=window), whole)
    lens, keys = [12, 9], [5, 9]                        # queries before the first key, with a wide window
    q, k, v = _inputs(lens, keys, 8, 2, 128, 46)
    whole = exactkv.prompt_attention(q, k, v, _cu(lens), cu_seqlens_k=_cu(keys))
    got = exactkv.prompt_attention(q, k, v, _cu(lens), cu_seqlens_k=_cu(keys), window=0x7FFFFFFF)
    assert same_bits(got, whole)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_offsets_past_32_bits(D):
    """Rows so far apart that element offsets pass 2^31, for queries, keys and values."""
    n, pitch = 300, 1 << 23
    q, k, v = _inputs([n], [n], 2, 1, D, 47)
    want = exactkv.prompt_attention(q, k, v, _cu([n]))
    wide = torch.empty(n * pitch, dtype=torch.bfloat16, device=DEV)
    far = [wide.as_strided(t.shape, (pitch, D, 1), at) for t, at in ((q, 0), (k, 4096), (v, 8192))]
    for dst, src in zip(far, (q, k, v)):
        dst.copy_(src)
    assert same_bits(exactkv.prompt_attention(*far, _cu([n])), want)


def test_more_sequences_than_a_wavefront_scans():
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 9, (200,), generator=g).tolist()
    _run(lens, 8, 2, 64)


def test_no_sequence_and_no_row():
    q, k, v = _inputs([5], [5], 8, 2, 128, 1)
    assert (exactkv.prompt_attention(q, k, v, _cu([])) == 0).all()
    e = exactkv.prompt_attention(q[:0], k[:0], v[:0], _cu([0, 0]))
    assert e.shape == (0, 8, 128)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_strided_inputs(D):
    """Views of one fused projection, and of [1, H, N, D] tensors as an attention module has them."""
    lens, Hq, Hkv = [100, 37], 8, 2
    q, k, v = _inputs(lens, lens, Hq, Hkv, D, 7)
    want = exactkv.prompt_attention(q, k, v, _cu(lens))
    fused = torch.cat([q, k, v], dim=1)
    got = exactkv.prompt_attention(fused[:, :Hq], fused[:, Hq:Hq + Hkv], fused[:, Hq + Hkv:], _cu(lens))
    assert same_bits(got, want)
    hq, hk, hv = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    assert same_bits(exactkv.prompt_attention(hq, hk, hv, _cu(lens)), want)
    # keys and values of one head, broadcast over the KV heads
    got = exactkv.prompt_attention(q, k[:, :1].expand(-1, Hkv, -1), v[:, :1].expand(-1, Hkv, -1), _cu(lens))
    one = exactkv.prompt_attention(q, k[:, :1].contiguous(), v[:, :1].contiguous(), _cu(lens))
    assert same_bits(got, one)


def test_rows_behind_the_last_sequence():
    q, k, v = _inputs([50], [50], 8, 2, 128, 9)
    cu = _cu([20, 13])
    fresh = exactkv.prompt_attention(q, k, v, cu)
    assert (fresh[33:] == 0).all()
    out = torch.full_like(q, 7.0)
    assert exactkv.prompt_attention(q, k, v, cu, out=out) is out
    assert (out[33:] == 7).all() and same_bits(out[:33], fresh[:33])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_no_row_looks_at_do_not_reach_it(bad, D):
    """A key or value that is infinite or NaN reaches the rows that see it and no other: later
    tokens of the sequence under the causal mask, those past the window, other sequences."""
    lens, at = [90, 130, 20], 40
    q, k, v = _inputs(lens, lens, 4, 2, D, 11)
    for window in (0, 16):
        clean = exactkv.prompt_attention(q, k, v, _cu(lens), window=window)
        for name in ("v", "k"):
            kk, vv = k.clone(), v.clone()
            (vv if name == "v" else kk)[90 + at, 1] = bad
            got = exactkv.prompt_attention(q, kk, vv, _cu(lens), window=window)
            seen = torch.zeros(240, 4, dtype=torch.bool, device=DEV)
            seen[90 + at:90 + (at + window if window else 130), 2:] = True
            want, mag = _formula(q, k, v, lens, lens, window)
            assert torch.isfinite(got[~seen]).all()
            far = (got.double() - want).abs() - (2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -11) * mag)
            assert (far[~seen] <= 0).all()
            if name == "v":                            # every channel of a row that sees it is what p v gives
                rows = got[seen]
                assert (rows.isnan() if math.isnan(bad) else rows == bad).all()
            elif math.isnan(bad):
                assert got[seen].isnan().all()
        assert same_bits(exactkv.prompt_attention(q, k, v, _cu(lens), window=window), clean)


def test_scores_without_a_finite_value():
    """Rows whose every visible score is -inf have no softmax (NaN); with one finite score among
    them, that key's value."""
    q, k, v = _inputs([40], [40], 1, 1, 64, 13)
    q[:] = 1.0
    k[:] = -math.inf
    got = exactkv.prompt_attention(q, k, v, _cu([40]))
    assert got.isnan().all()
    k[3] = 0.5
    got = exactkv.prompt_attention(q, k, v, _cu([40]))
    assert got[:3].isnan().all() and same_bits(got[3:], v[3:4].expand(37, 1, 64).contiguous())


def test_large_and_far_scores():
    """Scores of thousands, of either sign, and a maximum that rises with every tile."""
    n, D = 300, 128
    q, k, v = _inputs([n], [n], 2, 1, D, 15)
    for factor in (60.0, -60.0):
        kk = (k.float() + factor * torch.arange(n, device=DEV).view(n, 1, 1) / n).bfloat16()
        qq = (q.float().abs() * 4).bfloat16()
        got = exactkv.prompt_attention(qq, kk, v, _cu([n]))
        want, mag = _formula(qq, kk, v, [n], [n], 0)
        # scores s up to 4 x 60 x 0.8 x sqrt(128) = 2^11: their fp32 error 128 x 2^-24 x s, and
        # 2^-23 of 1.44 s in the exponent, each at most 2^-6 of a weight
        assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -5) * mag).all()


def test_offsets_out_of_range_are_clamped_and_reported():
    q, k, v = _inputs([50], [50], 8, 2, 128, 17)
    for cu in ([0, 20, 90], [0, 30, 10, 50], [-4, 50], [3, 50]):
        exactkv.prompt_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device=DEV))
        assert kernels.error_bits() == 0x20, cu


@pytest.mark.parametrize("D", [64, 128, 256])
def test_split_offsets_out_of_range_are_clamped_and_reported(D):
    """A split call's too; sequences that are sound keep their rows."""
    q, k, v = _inputs([50], [3000], 8, 2, D, 48)
    want = exactkv.prompt_attention(q[:20], k[:1500], v[:1500], _cu([20]), cu_seqlens_k=_cu([1500])).double()
    for cu, cu_k in (([0, 20, 90], [0, 1500, 3000]), ([0, 20, 50], [0, 1500, 9000]), ([0, 20, 10, 50], [0, 1500, 1500, 3000]),
                     ([3, 50], [0, 3000]), ([5, 5], [0, 3000]), ([0, 50], [-7, 3000]), ([0, 20, 50], [0, 1500, -5])):
        print("[case]", D, cu, cu_k, flush=True)
        got = exactkv.prompt_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device=DEV),
                                       cu_seqlens_k=torch.tensor(cu_k, dtype=torch.int32, device=DEV))
        assert kernels.error_bits() == 0x20, (cu, cu_k)
        if cu[1] == 20 and cu[2] >= 50:
            assert (got[:20].double() - want).norm() <= 2.0 ** -7 * want.norm()


def test_captured_and_replayed():
    """A graph with static buffers: new values and new offsets between replays, beside eager work."""
    N, Hq, Hkv, D = 200, 8, 2, 128
    q, k, v = _inputs([N], [N], Hq, Hkv, D, 19)
    cu = _cu([N, 0, 0])
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        exactkv.prompt_attention(q, k, v, cu)
    stream.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        out = exactkv.prompt_attention(q, k, v, cu)
    for i, lens in enumerate(([100, 90, 10], [1, 0, 150], [66, 67, 67], [200, 0, 0])):
        for t, x in zip((q, k, v), _inputs([N], [N], Hq, Hkv, D, 20 + i)):
            t.copy_(x)
        cu.copy_(_cu(lens))
        eager = exactkv.prompt_attention(q, k, v, cu)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert same_bits(out, eager)


def test_split_keys_captured():
    """Two captured calls with split keys (a workspace each), replayed in either order."""
    graphs, stream = [], torch.cuda.Stream()
    for seed, lens, keys in ((3, [20], [3000]), (4, [7, 9], [2000, 1500])):
        q, k, v = _inputs(lens, keys, 8, 2, 128, seed)
        cu, ck = _cu(lens), _cu(keys)
        want = exactkv.prompt_attention(q, k, v, cu, cu_seqlens_k=ck)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = exactkv.prompt_attention(q, k, v, cu, cu_seqlens_k=ck)
        graphs.append((g, out, want, (q, k, v, cu, ck)))
    for order in ((0, 1), (1, 0), (1, 1)):
        for i in order:
            graphs[i][1].zero_()
            graphs[i][0].replay()
        torch.cuda.synchronize()
        for i in order:
            assert same_bits(graphs[i][1], graphs[i][2])


def test_on_another_stream():
    lens = [300, 200]
    q, k, v = _inputs(lens, lens, 8, 2, 128, 23)
    cu = _cu(lens)
    want = exactkv.prompt_attention(q, k, v, cu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = exactkv.prompt_attention(q, k, v, cu)
    s.synchronize()
    assert same_bits(got, want)


def test_same_call_same_bits():
    lens = [700, 65, 300]
    q, k, v = _inputs(lens, lens, 28, 4, 128, 29)
    first = exactkv.prompt_attention(q, k, v, _cu(lens))
    for _ in range(3):
        assert same_bits(exactkv.prompt_attention(q, k, v, _cu(lens)), first)


def test_last_token_is_decode_attention():
    """A prompt's last row is what decode_attention gives over a cache of the same tokens, to both
    kernels' rounding (2^-8 of A each, and the stores')."""
    T, Hq, Hkv, D = 333, 32, 8, 128
    q, k, v = _inputs([T], [T], Hq, Hkv, D, 31)
    kc, vc = exactkv.BF16KV(1, 336, Hkv, D), exactkv.BF16KV(1, 336, Hkv, D)
    kc.prefill_slot(0, k[None])
    vc.prefill_slot(0, v[None])
    for window in (0, 100):
        one = exactkv.decode_attention(q[-1:].contiguous(), kc, vc, window=window)
        got = exactkv.prompt_attention(q, k, v, _cu([T]), window=window)[-1:]
        want, mag = _formula(q, k, v, [T], [T], window)
        far = (got.double() - one.double()).abs()
        assert (far <= 2 * (2.0 ** -8 * want[-1:].abs() + (2.0 ** -8 + 2.0 ** -11) * mag[-1:])).all()


@pytest.mark.parametrize("what", ["dtype", "heads", "dim", "rows", "alias", "align", "offsets", "device", "window", "out"])
def test_refusals(what):
    q, k, v = _inputs([64], [64], 8, 2, 128, 37)
    cu, kw = _cu([64]), {}
    if what == "dtype":
        q = q.float()
    elif what == "heads":
        q = q[:, :7]
    elif what == "dim":
        q, k, v = q[..., :96], k[..., :96], v[..., :96]
    elif what == "rows":
        k, v = k[:60], v[:60]
    elif what == "alias":
        kw["out"] = q
    elif what == "align":
        q = torch.empty(64 * 8 * 128 + 8, dtype=torch.bfloat16, device=DEV)[1:-7].view(64, 8, 128)
    elif what == "offsets":
        cu = cu.long()
    elif what == "device":
        cu = cu.cpu()
    elif what == "window":
        kw["window"] = -1
    else:
        kw["out"] = torch.empty(64, 8, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises((ValueError, RuntimeError)):
        exactkv.prompt_attention(q, k, v, cu, **kw)
