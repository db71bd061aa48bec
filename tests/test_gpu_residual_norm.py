"""The residual stream's update and the norms before and after a block against their definition in 64 bits."""
import math

import pytest
import torch

import int8_ref as ref
from lightbulb_amd import int8

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def values(gen, m, k, dtype, dev, spread=1.0):
    return (torch.randn(m, k, generator=gen) * spread).to(dtype).to(dev)


def make_norm(gen, k, kind, dev, bias=None, offset=0.0, eps=1e-5):
    """(Norm, its plain form), or (None, None)."""
    if not kind:
        return None, None
    w = 1 + 0.3 * torch.randn(k, generator=gen) - offset
    b = torch.randn(k, generator=gen) if (kind == "layer" if bias is None else bias) else None
    return (int8.Norm(w.to(dev), eps, bias=None if b is None else b.to(dev), kind=kind, offset=offset),
            {"kind": kind, "weight": w, "bias": b, "eps": torch.tensor(eps, dtype=torch.float32).item(), "offset": torch.tensor(offset, dtype=torch.float32).item()})


def spread_of(u, n):
    """sqrt(mean + eps) of a norm's rows, and the values over it."""
    d = u - u.mean(-1, keepdim=True) if n["kind"] == "layer" else u
    s = ((d * d).mean(-1, keepdim=True) + n["eps"]).sqrt()
    return s, d / s


def norm_bound(u, du, n):
    """How far a norm of rows within du of u may be in f32: 8 roundings of the scaled value (two of the distance from the mean,
    of 1 / spread, of weight + offset, two products, and two more for the spread's own), the bias's, and what du does by itself, through the mean and
    through the spread.  Subnormal: a half step of the first product, times the weight, and one of the second."""
    w = (n["weight"].double() + n["offset"]).abs()
    s, v = spread_of(u, n)
    y = ref.normed(u, n)
    most = du.amax(-1, keepdim=True) / s.clamp(min=1e-300)
    return 8 * ref.U * (v * w).abs() + ref.U * y.abs() + most * w * (2 + v.abs()) + ref.least(torch.float32) * (1 + w)


def check(x, residual, gate, scale, post, pre, quantize=False, **kw):
    """One call against its definition.  Codes: 64 bits, which leave about 1e-13 of the terms, then the roundings of what is stored.
    Values: f32 with the bounds above."""
    r, y = int8.residual_norm(x, residual, post=post[0], gate=gate, scale=scale, norm=pre[0], quantize=quantize)
    scale = torch.tensor(scale, dtype=torch.float32).double().item()
    rw, yw = ref.residual_norm(x, residual, post[1], gate, scale, pre[1])
    # f32: the first norm, the gate, the scale with the residual
    u = x.cpu().double()
    du = norm_bound(u, torch.zeros_like(u), post[1]) if post[1] else torch.zeros_like(u)
    g = gate.cpu().double().abs() if gate is not None else 1.0
    u = ref.normed(u, post[1]).abs() * g
    dr = abs(scale) * (du * g + (ref.U * u if gate is not None else 0.0)) + ref.U * rw.abs() + ref.least(torch.float32)
    if quantize:
        dr = ref.U * rw.abs() + 1e-13 * (rw.abs() + (0 if residual is None else residual.cpu().double().abs())) + ref.least(torch.float32)
    if residual is None and gate is None and post[0] is None and scale == 1.0:
        assert r is x
        dr = torch.zeros_like(dr)
    else:
        rt = x.dtype if residual is None else residual.dtype
        assert r.dtype == rt and r.shape == x.shape
        ref.close(r, rw, ref.stored(rw, dr, rt))
    if pre[0] is None:
        assert y is None
        return
    if quantize:
        c, s = ref.codes(yw.float())
        assert torch.equal(y.codes.cpu().double(), c) and torch.equal(torch.nan_to_num(y.scales.cpu(), nan=-1.0), torch.nan_to_num(s, nan=-1.0))
        assert not y._rows.cpu()[:, x.shape[-1]:].any()
    else:
        assert y.dtype == x.dtype and y.shape == x.shape
        ref.close(y, yw, ref.stored(yw, norm_bound(rw, dr, pre[1]), x.dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 8), (1, 100), (5, 512), (2, 513), (9, 1000), (1, 2048), (4, 2049), (1, 4096), (6, 5000), (2, 8192),
                                 (3, 8200), (1, 16384), (2, 16385), (1, 32768)])
def test_widths(dev, dtype, quantize, m, k):
    gen = torch.Generator().manual_seed(m + k)
    x, res = values(gen, m, k, dtype, dev), values(gen, m, k, torch.float32, dev, 2.0)
    check(x, res, None, 1.0, make_norm(gen, k, "rms", dev), make_norm(gen, k, "rms", dev), quantize)
    check(x, None, None, 1.0, (None, None), make_norm(gen, k, "layer", dev), quantize)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("k", [8200, 10001, 12289, 14336])
def test_many_wide_rows(dev, dtype, quantize, k):
    gen = torch.Generator().manual_seed(k)
    x, res = values(gen, 258, k, dtype, dev, 2.0), values(gen, 258, k, torch.float32, dev)
    check(x, res, None, 1.0, make_norm(gen, k, "rms", dev), make_norm(gen, k, "layer", dev), quantize)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stream", DTYPES)
@pytest.mark.parametrize("post", ["", "rms", "layer"])
@pytest.mark.parametrize("pre", ["", "rms", "layer"])
def test_forms(dev, dtype, stream, post, pre):
    gen = torch.Generator().manual_seed(len(post) + 3 * len(pre))
    m, k = 7, 700
    x, res = values(gen, m, k, dtype, dev), values(gen, m, k, stream, dev)
    gates = [None, values(gen, 1, k, dtype, dev)[0], values(gen, m, k, dtype, dev)]
    for gate in gates:
        for scale in (1.0, 0.22):
            for offset in (0.0, 1.0):
                ps, pr = make_norm(gen, k, post, dev, offset=offset), make_norm(gen, k, pre, dev, bias=offset == 0.0, offset=offset)
                for residual in (res, None):
                    check(x, residual, gate, scale, ps, pr)
                if pre:
                    check(x, res, gate, scale, ps, pr, quantize=True)


@pytest.mark.parametrize("quantize", [False, True])
def test_layer_norm_of_shifted_rows(dev, quantize):
    # a mean a million times the spread: the sums hold it, and what f32 rows lose is r's own rounding
    gen = torch.Generator().manual_seed(1)
    x = values(gen, 4, 1500, torch.float32, dev) + torch.tensor([1e6, -3e5, 0.0, 1e3], device=dev)[:, None]
    check(x, None, None, 1.0, (None, None), make_norm(gen, 1500, "layer", dev), quantize)
    check(x, values(gen, 4, 1500, torch.float32, dev), None, 0.5, (None, None), make_norm(gen, 1500, "layer", dev), quantize)


def test_rows_of_odd_values(dev):
    gen = torch.Generator().manual_seed(2)
    k = 600
    x = torch.randn(9, k, generator=gen)
    x[0] = 0.0
    x[1] *= 1e30   # squares beyond f32
    x[2] *= 1e-30  # under eps
    x[3, 5] = math.nan
    x[4, 599] = math.inf
    x[5] = 1.0
    x[6] = torch.randn(k, generator=gen) * 1e-42  # subnormal
    x = x.to(dev)
    rms, layer = make_norm(gen, k, "rms", dev), make_norm(gen, k, "layer", dev)
    for pre in (rms, layer):
        for quantize in (False, True):
            check(x, None, None, 1.0, (None, None), pre, quantize)
    r, y = int8.residual_norm(x, torch.ones_like(x), norm=rms[0])
    assert torch.isnan(y[3]).all() and torch.isfinite(y[[0, 1, 2, 5, 6, 7, 8]]).all() and torch.isnan(r[3, 5]) and torch.isfinite(r[3, 6])


def test_no_eps(dev):
    # a zero row over eps = 0 is 0 / 0, by the formula; others are as they are
    gen = torch.Generator().manual_seed(3)
    x = values(gen, 3, 130, torch.float32, dev)
    x[1] = 0.0
    for quantize in (False, True):
        check(x, None, None, 1.0, (None, None), make_norm(gen, 130, "rms", dev, eps=0.0), quantize)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_rows_at_the_ends_of_the_range(dev, kind):
    # no eps: 1 / spread of these is itself beyond f32 or subnormal; the norms' values are ordinary
    gen = torch.Generator().manual_seed(7)
    x = torch.randn(8, 700, generator=gen).clamp(-3, 3) * torch.tensor([1e-44, 1e-40, 1e-37, 1e-31, 1e29, 1e32, 1e36, 1e38])[:, None]
    x[7] = torch.where(x[7] < 0, -3.4e38, 3.4e38)
    x = x.to(dev)
    for eps in (0.0, 1e-30):
        n = make_norm(gen, 700, kind, dev, eps=eps)
        for quantize in (False, True):
            check(x, None, None, 1.0, (None, None), n, quantize)
        check(x, None, None, 1.0, n, make_norm(gen, 700, kind, dev))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_inputs(dev, dtype):
    gen = torch.Generator().manual_seed(4)
    base = values(gen, 24, 900, dtype, dev)
    rms = make_norm(gen, 301, "rms", dev)
    x, res, gate = base[:8, 1:302], base[8:24:2, 300:601], base[3:4, 7:308].expand(8, 301)
    check(x, res, gate, 0.5, make_norm(gen, 301, "layer", dev), rms)
    check(x, res, None, 1.0, (None, None), rms, quantize=True)
    x3 = base.view(4, 6, 900)[:, :1, 2:303]
    r, y = int8.residual_norm(x3, x3, norm=rms[0])
    assert r.shape == y.shape == (4, 1, 301)
    rw, yw = ref.residual_norm(x3, x3, None, None, 1.0, rms[1])
    ref.close(y, yw, ref.stored(yw, norm_bound(rw, ref.U * rw.abs(), rms[1]), dtype))


def test_no_rows(dev):
    n = int8.Norm(torch.ones(64, device=dev), 1e-5)
    r, y = int8.residual_norm(torch.empty(0, 64, device=dev), torch.empty(0, 64, device=dev), norm=n)
    assert r.shape == y.shape == (0, 64)
    r, y = int8.residual_norm(torch.empty(2, 0, 64, device=dev), norm=n, quantize=True)
    assert y.shape == (2, 0, 64) and y.scales.shape == (2, 0)
