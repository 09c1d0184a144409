"""add_norm against the formula in 64 bits: every width around the kernel's pieces, odd and
unaligned rows, each of post norm, gate, scale and residual, strides, graphs, refusals.

Tolerance, per value: the stores round by at most 2^-8 of it. fp32: a sum of C squares is off by at
most (C / 64 + 10) 2^-24 of it (C / 64 terms in a lane at most, then the tree), the reciprocal root
by half of that and 2^-22, products by 2^-24 each: below 2^-15 for C <= 16384, of |r| + |scale u|
for h, and of that times its rsqrt and weight for y.

No counterpart in the reference (the model's own modules do this, engine.py:75-91)."""
import pytest
import torch

import exactkv_amd as exactkv
from tests.conftest import same_bits

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _formula(x, r, w, eps, post, gate, scale):
    """(h, y, bound of h, bound of y) in 64 bits."""
    def unit(z):
        return 1.0 / (z.square().mean(-1, keepdim=True) + eps).sqrt()
    u = x.double()
    if post is not None:
        u = u * unit(u) * post.double()
    if gate is not None:
        u = u * gate.double()
    u = scale * u
    r = torch.zeros_like(u) if r is None else r.double()
    h, mag = r + u, r.abs() + u.abs()
    y = h * unit(h) * w.double()
    hb = 2.0 ** -8 * h.abs() + 2.0 ** -15 * mag + 1e-37
    yb = 2.0 ** -8 * y.abs() + 2.0 ** -15 * mag * unit(h) * w.double().abs() * 2 + 1e-37
    return h, y, hb, yb


def _inputs(N, C, seed, post=True, gate="full"):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rows(*shape):
        return torch.randn(*shape, generator=g, device=DEV)
    return dict(x=rows(N, C).bfloat16(), residual=(3 * rows(N, C)).bfloat16(), weight=(1 + 0.3 * rows(C)).bfloat16(),
                post_weight=(1 + 0.3 * rows(C)).bfloat16() if post else None,
                gate=None if gate == "none" else rows(N, C).sigmoid().bfloat16() if gate == "full" else rows(C).bfloat16())


def _check(d, eps=1e-6, scale=1.0):
    h, y = exactkv.add_norm(eps=eps, scale=scale, **d)
    wh, wy, hb, yb = _formula(d["x"], d["residual"], d["weight"], eps, d["post_weight"], d["gate"], scale)
    assert ((h.double() - wh).abs() <= hb).all()
    assert ((y.double() - wy).abs() <= yb).all()
    return h, y


WIDTHS = [1, 2, 7, 8, 63, 64, 65, 511, 512, 513, 1000, 1024, 1025, 2047, 2048, 2049, 3584, 4096, 4104, 5120, 8191, 8192,
          8200, 16384]


@pytest.mark.parametrize("C", WIDTHS)
def test_widths(C):
    print("[case]", C, flush=True)
    _check(_inputs(5, C, C), scale=0.22)
    _check(_inputs(3, C, C + 1, post=False, gate="none"))


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("scale", [1.0, -0.5])
@pytest.mark.parametrize("gate", ["none", "channel", "full"])
@pytest.mark.parametrize("post", [False, True])
def test_parts(post, gate, scale, residual):
    d = _inputs(33, 896, 3, post, gate)
    if not residual:
        d["residual"] = None
    h, _ = _check(d, eps=1e-5, scale=scale)
    if not residual and not post and gate == "none" and scale == 1.0:
        assert h is d["x"]


@pytest.mark.parametrize("N", [1, 2, 255, 1000])
def test_rows(N):
    _check(_inputs(N, 4096, N, post=False, gate="none"))


def test_no_rows():
    h, y = exactkv.add_norm(**_inputs(0, 64, 1))
    assert h.shape == y.shape == (0, 64)


def test_shapes_strides_and_alignment():
    d = _inputs(24, 512, 5)
    h, y = exactkv.add_norm(**d)
    cube = {k: v.view(2, 12, 512) if v.shape == (24, 512) else v for k, v in d.items()}
    h3, y3 = exactkv.add_norm(**cube)
    assert h3.shape == (2, 12, 512) and same_bits(h3.view(24, 512), h) and same_bits(y3.view(24, 512), y)
    one = {k: v[0] if v.shape == (24, 512) else v for k, v in d.items()}
    h1, y1 = exactkv.add_norm(**one)
    assert same_bits(h1, h[0]) and same_bits(y1, y[0])
    for pad in (1, 2, 8):                              # rows 2-byte, 4-byte and 16-byte aligned
        wide = {}
        for k, v in d.items():
            if v.shape == (24, 512):
                w = torch.zeros(24, 512 + pad, dtype=torch.bfloat16, device=DEV)
                w[:, pad:] = v
                wide[k] = w[:, pad:]
            else:
                wide[k] = v
        hw, yw = exactkv.add_norm(**wide)
        # unaligned rows take other lanes' order of the sums: fp32 rounding apart, so at most a step
        for a, b in ((hw, h), (yw, y)):
            assert ((a.double() - b.double()).abs() <= 2.0 ** -7 * b.double().abs() + 1e-30).all()
    got = exactkv.add_norm(d["x"][:, :512][::2], d["residual"][::2], d["weight"])
    want = exactkv.add_norm(d["x"][::2].contiguous(), d["residual"][::2].contiguous(), d["weight"])
    assert same_bits(got[0], want[0]) and same_bits(got[1], want[1])


def test_a_zero_row_and_bad_values_stay_in_their_row():
    d = _inputs(6, 1024, 7, post=False, gate="none")
    clean = exactkv.add_norm(**d)
    d["x"][1], d["residual"][1] = 0, 0
    d["x"][3, 5] = float("nan")
    d["x"][4, 6] = float("inf")
    h, y = exactkv.add_norm(**d)
    for a, b in zip((h, y), clean):
        assert same_bits(a[[0, 2, 5]], b[[0, 2, 5]])
        assert (a[1] == 0).all()
    assert y[3].isnan().all() and h[3].isnan().sum() == 1
    assert h[4, 6] == float("inf") and y[4, 6].isnan() and (y[4, :6] == 0).all()


def test_captured_and_replayed():
    d = _inputs(40, 2048, 9)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        exactkv.add_norm(**d)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        h, y = exactkv.add_norm(**d)
    for i in range(3):
        d["x"].copy_(_inputs(40, 2048, 10 + i)["x"])
        want = exactkv.add_norm(**d)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert same_bits(h, want[0]) and same_bits(y, want[1])


@pytest.mark.parametrize("what", ["type", "wide", "residual", "weight", "gate", "rows", "device"])
def test_refusals(what):
    d = _inputs(4, 64, 11)
    if what == "type":
        d["x"] = d["x"].float()
    elif what == "wide":
        d = _inputs(1, 16392, 11)
    elif what == "residual":
        d["residual"] = d["residual"][:3]
    elif what == "weight":
        d["weight"] = d["weight"][:63]
    elif what == "gate":
        d["gate"] = d["gate"][:, :1]
    elif what == "rows":
        d["x"] = d["x"].t().contiguous().t()
    else:
        d["weight"] = d["weight"].cpu()
    with pytest.raises(ValueError):
        exactkv.add_norm(**d)
