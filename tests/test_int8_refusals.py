"""What the integer linears and the norms between them refuse, without a device: the C entry points check before any HIP
call, and the Python ones before they reach the library."""
import ctypes
import math

import pytest
import torch

from lightbulb_amd import _lib, int8

D = 1 << 12  # addresses that are aligned and never read
FAR = 1 << 40
INVALID, TYPE, SHAPE, LIMIT = -1, -2, -3, -6


def at(struct):
    return None if struct is None else ctypes.addressof(struct)


def weight(**kw):
    f = dict(d_codes=D, d_scales=D, d_bias=None, n=64)
    f.update(kw)
    return _lib.I8WeightStruct(**f)


def quantize(lbq, ctx=D, type=0, x=D, stride=100, m=3, k=100, codes=FAR, scales=2 * FAR):
    return lbq.lbq_i8_quantize(ctx, type, x, stride, m, k, codes, scales, None)


def linear(lbq, ws=None, ctx=D, type=0, x=D, stride=100, codes=FAR, scales=2 * FAR, m=5, k=100, count=None, out=0, ys=None):
    ws = [weight()] if ws is None else ws
    array = (ctypes.c_void_p * 8)(*[at(w) for w in ws])
    ys = (ctypes.c_void_p * 8)(*(ys or [3 * FAR] * 8))
    return lbq.lbq_i8_linear(ctx, type, x, stride, codes, scales, m, k, array, len(ws) if count is None else count, out, ys, None)


def gate_up(lbq, gate=None, up=None, ctx=D, type=0, x=D, stride=100, codes=FAR, scales=2 * FAR, m=5, k=100, out=0, y=3 * FAR):
    gate, up = gate or weight(), up or weight()
    return lbq.lbq_i8_gate_up_silu(ctx, type, x, stride, codes, scales, m, k, at(gate), at(up), out, y, None)


def norm(**kw):
    f = dict(kind=0, eps=1e-5, offset=0.0, d_weight=D, d_bias=None)
    f.update(kw)
    return _lib.NormStruct(**f)


def residual_norm(lbq, ctx=D, type=0, x=D, stride=100, rt=0, res=FAR, res_stride=100, post=None, gate=None, gate_stride=0, pre=True, m=3, k=100,
                  r=2 * FAR, y=3 * FAR, codes=None, scales=None):
    pre = norm() if pre is True else pre
    return lbq.lbq_residual_norm(ctx, type, x, stride, rt, res, res_stride, at(post), gate, gate_stride, 1.0, at(pre), m, k, r, y,
                                 codes, scales, None)


SIZES = [(dict(ctx=None), INVALID), (dict(type=8), TYPE), (dict(m=-1), SHAPE), (dict(k=0), SHAPE), (dict(k=131072), LIMIT), (dict(m=1 << 25), LIMIT),
         (dict(stride=-1), SHAPE), (dict(x=D + 2), INVALID), (dict(type=1, x=D + 1), INVALID)]


@pytest.mark.parametrize("kw,status", SIZES + [
    (dict(x=None), INVALID), (dict(codes=None), INVALID), (dict(scales=None), INVALID), (dict(codes=FAR + 8), INVALID),
    (dict(scales=2 * FAR + 2), INVALID), (dict(codes=D + 16), INVALID), (dict(scales=D + 1196), INVALID)])
def test_quantize(lbq, kw, status):
    assert quantize(lbq, **kw) == status and lbq.lbq_last_error()


@pytest.mark.parametrize("kw,status", SIZES + [
    (dict(out=12), TYPE), (dict(codes=FAR + 4, x=None), INVALID), (dict(codes=None, x=None), INVALID), (dict(scales=None, x=None), INVALID),
    (dict(codes=D), INVALID), (dict(m=1 << 24, k=1, out=0), LIMIT)])
def test_products(lbq, kw, status):
    ws = [weight(n=1 << 14)]
    assert linear(lbq, ws, **kw) == status and lbq.lbq_last_error()
    assert gate_up(lbq, *ws, *ws, **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(d_codes=None), INVALID), (dict(d_scales=None), INVALID), (dict(d_codes=D + 8), INVALID), (dict(d_scales=D + 1), INVALID),
    (dict(d_bias=D + 2), INVALID), (dict(n=0), SHAPE), (dict(n=1 << 25), LIMIT)])
def test_weights(lbq, kw, status):
    assert linear(lbq, [weight(**kw)]) == status
    assert linear(lbq, [weight(), weight(**kw)]) == status
    assert gate_up(lbq, weight(**kw)) == status and gate_up(lbq, None, weight(**kw)) == status


def test_outputs(lbq):
    assert linear(lbq, count=0) == SHAPE and linear(lbq, [weight()] * 5) == SHAPE
    assert linear(lbq, [weight(), None], ) == INVALID
    assert linear(lbq, ys=[None]) == INVALID and linear(lbq, ys=[3 * FAR + 2]) == INVALID
    assert linear(lbq, [weight(), weight()], ys=[3 * FAR, None]) == INVALID
    assert linear(lbq, ys=[D + 1996]) == INVALID  # the last of x's rows
    assert linear(lbq, x=None, ys=[FAR + 128]) == INVALID and linear(lbq, x=None, ys=[2 * FAR + 8]) == INVALID
    assert gate_up(lbq, y=None) == INVALID and gate_up(lbq, y=D) == INVALID
    assert gate_up(lbq, weight(n=32)) == SHAPE
    assert lbq.lbq_i8_linear(D, 0, D, 1, FAR, FAR, 1, 1, None, 1, 0, (ctypes.c_void_p * 1)(FAR), None) == INVALID
    assert lbq.lbq_i8_linear(D, 0, D, 1, FAR, FAR, 1, 1, (ctypes.c_void_p * 1)(D), 1, 0, None, None) == INVALID
    # no tokens: checked, and nothing to do
    assert linear(lbq, m=0, x=None, codes=None, scales=None, ys=[None]) == 0 and quantize(lbq, m=0, x=None) == 0
    assert linear(lbq, [weight(n=0)], m=0) == SHAPE


@pytest.mark.parametrize("kw,status", [
    (dict(ctx=None), INVALID), (dict(type=8), TYPE), (dict(rt=8), TYPE), (dict(m=-1), SHAPE), (dict(k=0), SHAPE), (dict(k=32769), LIMIT),
    (dict(x=None), INVALID), (dict(x=D + 2), INVALID), (dict(stride=-4), SHAPE), (dict(res=FAR + 1), INVALID), (dict(res_stride=-1), SHAPE),
    (dict(gate=D + 1), INVALID), (dict(gate=D, gate_stride=-1), SHAPE), (dict(r=None, y=None, pre=None), INVALID), (dict(y=None), INVALID),
    (dict(pre=None), INVALID), (dict(codes=4 * FAR, scales=5 * FAR), INVALID), (dict(y=None, codes=4 * FAR), INVALID),
    (dict(y=None, codes=4 * FAR + 8, scales=5 * FAR), INVALID), (dict(pre=None, y=None, codes=4 * FAR, scales=5 * FAR), INVALID),
    (dict(r=2 * FAR + 2), INVALID), (dict(type=1, y=3 * FAR + 1), INVALID), (dict(r=D + 400), INVALID), (dict(y=FAR + 400), INVALID),
    (dict(r=FAR, res_stride=128), INVALID), (dict(r=FAR + 4), INVALID), (dict(y=2 * FAR + 4), INVALID), (dict(gate=3 * FAR), INVALID),
    (dict(y=None, codes=2 * FAR + 16, scales=5 * FAR), INVALID)])
def test_residual_norm(lbq, kw, status):
    assert residual_norm(lbq, **kw) == status and lbq.lbq_last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(kind=2), TYPE), (dict(kind=-1), TYPE), (dict(d_weight=None), INVALID), (dict(d_weight=D + 2), INVALID), (dict(d_bias=D + 1), INVALID),
    (dict(eps=-1.0), SHAPE), (dict(eps=math.nan), SHAPE)])
def test_norms(lbq, kw, status):
    assert residual_norm(lbq, pre=norm(**kw)) == status and residual_norm(lbq, post=norm(**kw)) == status


def test_results_in_one_place(lbq):
    # outputs of one call, and tokens' codes and scales, must lie apart
    ws = [weight(n=40), weight(n=40)]
    assert linear(lbq, ws, ys=[3 * FAR, 3 * FAR]) == INVALID
    assert linear(lbq, ws, ys=[3 * FAR, 3 * FAR + 5 * 40 * 4 - 4]) == INVALID
    assert linear(lbq, ws, ys=[3 * FAR + 5 * 40 * 4 - 4, 3 * FAR]) == INVALID
    assert linear(lbq, [weight()], scales=FAR + 4 * 128) == INVALID and linear(lbq, [weight()], x=None, scales=FAR) == INVALID
    assert quantize(lbq, scales=FAR + 2 * 128) == INVALID and gate_up(lbq, scales=FAR + 4 * 128) == INVALID
    assert residual_norm(lbq, y=None, codes=4 * FAR, scales=4 * FAR + 128) == INVALID
    assert quantize(lbq, stride=(1 << 38) + 1) == SHAPE


# ---------------------------------------------------------------------------
# Python
# ---------------------------------------------------------------------------
def refuses(match, f, *a, **kw):
    with pytest.raises(ValueError, match=match):
        f(*a, **kw)


def fake_linear(n, k, device="cpu"):
    """A linear without a device's context."""
    lin = int8.Int8Linear.__new__(int8.Int8Linear)
    w = int8.Int8Weight(torch.zeros(n, k, dtype=torch.int8), torch.ones(n))
    vars(lin).update(weight=w, bias=None, device=torch.device(device), _n=n, _k=k, _at=D, _ctx=D)
    return lin


def test_python_values():
    q = int8.quantize_tokens
    refuses("must be f32", q, torch.zeros(2, 3, dtype=torch.float64))
    refuses("one dimension", q, torch.zeros(3))
    refuses("contiguous", q, torch.zeros(4, 6).t())
    refuses("evenly apart", q, torch.zeros(4, 6, 8)[:, :5])
    refuses("runs on the GPU", q, torch.zeros(2, 3))


def test_python_weights():
    w = int8.Int8Weight
    refuses("int8 tensor", w, torch.zeros(2, 3), torch.ones(2))
    refuses("int8 tensor", w, torch.zeros(3, dtype=torch.int8), torch.ones(3))
    refuses("int8 tensor", w, torch.zeros(0, 3, dtype=torch.int8), torch.ones(0))
    refuses("exceeds", w, torch.zeros(1, 131072, dtype=torch.int8), torch.ones(1))
    refuses("scales", w, torch.zeros(2, 3, dtype=torch.int8), torch.ones(3))
    refuses("scales", w, torch.zeros(2, 3, dtype=torch.int8), torch.ones(2).half())
    refuses("2-D", w.quantize, torch.zeros(3))
    one = w(torch.ones(2, 3, dtype=torch.int8), torch.ones(2))
    assert one.shape() == (2, 3) and one._rows.shape == (2, 128) and torch.equal(one.dequantize(), torch.ones(2, 3))
    refuses("bias", int8.Int8Linear, one, torch.ones(3))
    with pytest.raises(AttributeError, match="fixed"):
        one.scales = torch.ones(2)


def test_python_products():
    a, b = fake_linear(4, 16), fake_linear(4, 32)
    refuses("between 1 and 4", int8.int8_linear_group, [], torch.zeros(1, 16))
    refuses("between 1 and 4", int8.int8_linear_group, [a] * 5, torch.zeros(1, 16))
    refuses("share k", int8.int8_linear_group, [a, b], torch.zeros(1, 16))
    refuses("incompatible", a, torch.zeros(1, 17))
    refuses("incompatible", a, torch.tensor(1.0))
    refuses("outputs must be", a, torch.zeros(1, 16), dtype=torch.float64)
    refuses("must be f32", a, torch.zeros(1, 16, dtype=torch.int32), dtype=torch.float32)
    refuses("weights on meta", fake_linear(4, 16, "meta"), torch.zeros(1, 16))
    refuses("must share shape", int8.int8_gate_up_silu, a, b, torch.zeros(1, 16))
    refuses("must share shape", int8.int8_gate_up_silu, a, fake_linear(5, 16), torch.zeros(1, 16))


def test_python_norms():
    n, x = int8.Norm(torch.ones(8), 1e-5), torch.zeros(2, 8)
    refuses("kind", int8.Norm, torch.ones(8), 1e-5, kind="group")
    refuses("norm over", int8.Norm, torch.ones(40000), 1e-5)
    refuses("norm over", int8.Norm, torch.ones(0), 1e-5)
    refuses("weight", int8.Norm, torch.ones(8).half(), 1e-5)
    refuses("bias", int8.Norm, torch.ones(8), 1e-5, bias=torch.ones(7))
    refuses("eps", int8.Norm, torch.ones(8), -1.0)
    refuses("eps", int8.Norm, torch.ones(8), math.nan)
    with pytest.raises(AttributeError, match="fixed"):
        n.eps = 1.0
    r = int8.residual_norm
    refuses("norm over 8", r, torch.zeros(2, 9), norm=n)
    refuses("norm over 8", r, torch.zeros(2, 9), post=n)
    refuses("quantize needs a norm", r, x, quantize=True)
    refuses("residual", r, x, torch.zeros(1, 8), norm=n)
    refuses("residual must be", r, x, x.double(), norm=n)
    refuses("gate of", r, x, gate=torch.ones(8).half())
    refuses("gate", r, x, gate=torch.ones(1, 8))
    refuses("gate", r, x, gate=torch.ones(16)[::2])
    assert r(x)[0] is x and r(x)[1] is None
