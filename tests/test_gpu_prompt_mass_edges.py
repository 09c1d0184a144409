"""prompt_mass where its inputs are odd: offsets that do not begin at 0 or ascend, and keys that are infinite.

Tolerances are those of tests/test_gpu_mass.py, per entry.

No counterpart in the reference, which keeps no weights."""
import math

import pytest
import torch

import exactkv_amd as exactkv
from exactkv_amd import kernels
from tests.test_gpu_mass import _gen, _near, _rows, _weights

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _cu(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _mass(q, k, cu, **kw):
    """prompt_mass into memory that held NaN before."""
    torch.cuda.synchronize()
    out = torch.full((k.shape[1], k.shape[0]), math.nan, device=DEV)
    del out
    return exactkv.prompt_mass(q, k, cu, **kw)


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (4, 4, 64), (6, 1, 256)])
@pytest.mark.parametrize("cu,n", [((5, 20, 64), 64), ((300, 301, 900), 1000), ((1, 2000), 2000), ((700, 700), 700), ((900, 2000), 1500), ((64,), 64)], ids=str)
def test_offsets_that_begin_behind_0(cu, n, Hq, Hkv, D):
    """Keys before the first sequence are keys that no sequence holds; the offsets are reported."""
    print("[case]", cu, n, Hq, Hkv, D, flush=True)
    g = _gen(n)
    q, k = torch.randn(n, Hq, D, generator=g, device=DEV).bfloat16(), _rows(g, n, Hkv, D)
    got = _mass(q, k, _cu(*cu))
    assert kernels.error_bits(clear=True) == (0x20 if len(cu) > 1 else 0)
    ends = [min(c, n) for c in cu]
    want, bound = (torch.zeros(Hkv, n, dtype=torch.float64, device=DEV) for _ in range(2))
    for a, e in zip(ends, ends[1:]):
        if e > a:
            w, err = _weights(q[a:e], k[a:e], torch.arange(e - a, device=DEV), 0)
            want[:, a:e], bound[:, a:e] = (x.view(Hkv, -1, e - a).sum(1) for x in (w, err))
    _near(got, want, bound)
    assert (got[:, : ends[0]] == 0).all()


@pytest.mark.parametrize("cu", [(0, 900, 0, 1000), (0, 1000, 500, 600), (900, 100), (0, 400, 300, 1000, 200)], ids=str)
def test_offsets_that_do_not_ascend(cu):
    """Reported, and no entry is left unwritten."""
    g = _gen(3)
    q, k = torch.randn(1000, 8, 128, generator=g, device=DEV).bfloat16(), _rows(g, 1000, 2, 128)
    got = _mass(q, k, _cu(*cu))
    assert kernels.error_bits(clear=True) == 0x20
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (4, 4, 64), (6, 1, 256)])
@pytest.mark.parametrize("lens,last", [((100,), 0), ((64,), 0), ((65, 31, 300), 0), ((700,), 33), ((2001, 5), 0), ((333, 200), 100)], ids=str)
def test_keys_whose_scores_are_all_minus_infinity(lens, last, Hq, Hkv, D):
    """An infinite key that every query scores with -infinity gets nothing and takes nothing from the others, wherever the queries' rows end."""
    print("[case]", lens, last, Hq, Hkv, D, flush=True)
    g = _gen(sum(lens))
    n = sum(lens)
    q, k = torch.randn(n, Hq, D, generator=g, device=DEV).bfloat16(), _rows(g, n, Hkv, D)
    q[..., 3] = q[..., 3].abs() + 0.5
    ends = [0]
    far = torch.zeros(n, dtype=torch.bool, device=DEV)
    for m in lens:
        ends.append(ends[-1] + m)
        far[[ends[-2] + i for i in (1, 2, m // 2, m - 2)]] = True              # (never a sequence's first key)
    k[far, :, 3] = -math.inf
    got = exactkv.prompt_mass(q, k, _cu(*ends), last=last)
    want, bound = (torch.zeros(Hkv, n, dtype=torch.float64, device=DEV) for _ in range(2))
    for a, e in zip(ends, ends[1:]):
        keep = (~far[a:e]).nonzero()[:, 0]
        rows = torch.arange(max(0, e - a - last) if last else 0, e - a, device=DEV)
        # (the others' weights are those of a row without these keys: each query stands behind the kept keys up to its own)
        pos = torch.searchsorted(keep, rows, right=True) - 1
        w, err = _weights(q[a:e][rows], k[a:e][keep], pos, 0)
        for x, y in ((want, w), (bound, err)):
            x[:, a + keep] = y.view(Hkv, -1, keep.numel()).sum(1)
    assert (got[:, far] == 0).all()
    _near(got, want, bound)
