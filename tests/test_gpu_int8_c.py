"""The integer linears and norms through the C entry points, as a caller of those may place buffers."""
import ctypes
import math

import pytest
import torch

import int8_ref as ref
from lightbulb_amd import _lib, int8
from lightbulb_amd.quantized import _stream, context

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
GUARD = 77


def linear(gen, n, k, dev, bias=True):
    w = torch.randint(-127, 128, (n, k), generator=gen, dtype=torch.int8).to(dev)
    t = ((0.5 + torch.rand(n, generator=gen)) * 2.0 ** -6 / math.sqrt(k)).to(dev)
    return int8.Int8Linear(int8.Int8Weight(w, t), torch.randn(n, generator=gen).to(dev) if bias else None)


def guarded(shape, dtype, dev, odd):
    """(whole, inside): `inside` of the shape with GUARD values or more on both sides, `odd` elements from alignment."""
    n = math.prod(shape)
    whole = torch.full((n + 2 * 128 + odd,), GUARD, dtype=dtype, device=dev)
    return whole, whole[128 + odd:128 + odd + n].view(shape)


def around(whole, inside):
    at, n = inside.storage_offset(), inside.numel()
    return bool((whole[:at] == GUARD).all()) and bool((whole[at + n:] == GUARD).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 3, 16, 30, 40, 70, 130, 300, 700])
@pytest.mark.parametrize("n", [96, 257])
@pytest.mark.parametrize("odd", [0, 1])
def test_outputs_at_any_address(dev, dtype, m, n, odd):
    # the same weight twice, another beside it, and a pair; nothing but the outputs is written
    gen = torch.Generator().manual_seed(m * n)
    k = 320
    x = torch.randn(m, k, generator=gen).to(dtype).to(dev)
    a, b = linear(gen, n, k, dev), linear(gen, n, k, dev, False)
    t = int8._DTYPES[dtype]
    codes, scales = torch.empty(m * 384, dtype=torch.int8, device=dev), torch.empty(m, device=dev)
    at = [a._at, b._at, a._at]
    outs = [guarded((m, n), dtype, dev, odd) for _ in at]
    lib, ctx = _lib.lib(), context(dev)
    _lib.check(lib.lbq_i8_linear(ctx, t, x.data_ptr(), k, codes.data_ptr(), scales.data_ptr(), m, k, (ctypes.c_void_p * 3)(*at), 3, t,
                                 (ctypes.c_void_p * 3)(*[y.data_ptr() for _, y in outs]), _stream(dev)))
    for lin, (whole, y) in zip((a, b, a), outs):
        assert around(whole, y) and torch.equal(y, lin(x))
    whole, y = guarded((m, n), dtype, dev, odd)
    _lib.check(lib.lbq_i8_gate_up_silu(ctx, t, x.data_ptr(), k, codes.data_ptr(), scales.data_ptr(), m, k, a._at, b._at, t, y.data_ptr(), _stream(dev)))
    assert around(whole, y) and torch.equal(y, int8.int8_gate_up_silu(a, b, x))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 5), (3, 130), (5, 512), (4, 2050), (3, 4100), (2, 9000), (1, 20000), (260, 9001)])
def test_rows_at_any_address(dev, dtype, m, k):
    # codes of rows of any alignment between guards, and norms whose r takes the residual's place
    gen = torch.Generator().manual_seed(m + k)
    _, x = guarded((m, k), dtype, dev, 1)
    x.copy_(torch.randn(m, k, generator=gen))
    t, row = int8._DTYPES[dtype], (k + 127) // 128 * 128
    lib, ctx = _lib.lib(), context(dev)
    codes, inside = guarded((m, row), torch.int8, dev, 0)
    scales, s = guarded((m,), torch.float32, dev, 1)
    _lib.check(lib.lbq_i8_quantize(ctx, t, x.data_ptr(), k, m, k, inside.data_ptr(), s.data_ptr(), _stream(dev)))
    c, sw = ref.codes(x)
    assert around(codes, inside) and around(scales, s) and torch.equal(s.cpu(), sw) and torch.equal(inside[:, :k].cpu().double(), c)
    assert not inside[:, k:].any()
    whole, r = guarded((m, k), dtype, dev, 1)
    r.copy_(torch.randn(m, k, generator=gen))
    gate = torch.randn(m, k + 3, generator=gen).to(dtype).to(dev)
    for kind in ("rms", "layer"):
        n = int8.Norm(torch.randn(k, generator=gen).to(dev), 1e-5, bias=torch.randn(k, generator=gen).to(dev), kind=kind)
        want = int8.residual_norm(x, r.clone(), post=n, gate=gate[:, :k], scale=0.5, norm=n)
        wq = int8.residual_norm(x, r.clone(), post=n, gate=gate[:, :k], scale=0.5, norm=n, quantize=True)
        old = r.clone()
        yw, y = guarded((m, k), dtype, dev, 1)
        _lib.check(lib.lbq_residual_norm(ctx, t, x.data_ptr(), k, t, r.data_ptr(), k, n._at, gate.data_ptr(), k + 3, 0.5, n._at, m, k, r.data_ptr(),
                                         y.data_ptr(), None, None, _stream(dev)))
        assert around(whole, r) and around(yw, y) and torch.equal(r, want[0]) and torch.equal(y, want[1])
        r.copy_(old)
        codes, inside = guarded((m, row), torch.int8, dev, 0)
        _lib.check(lib.lbq_residual_norm(ctx, t, x.data_ptr(), k, t, r.data_ptr(), k, n._at, gate.data_ptr(), k + 3, 0.5, n._at, m, k, r.data_ptr(),
                                         None, inside.data_ptr(), s.data_ptr(), _stream(dev)))
        assert around(whole, r) and around(codes, inside) and torch.equal(r, wq[0]) and torch.equal(inside[:, :k], wq[1].codes) and torch.equal(s, wq[1].scales)


def test_single_tokens_without_memory_for_codes(dev):
    gen = torch.Generator().manual_seed(5)
    lin = linear(gen, 100, 4096, dev)
    for m in (1, 2, 3, 4):
        x = torch.randn(m, 4096, generator=gen).to(dev)
        y = torch.empty(m, 100, device=dev)
        _lib.check(_lib.lib().lbq_i8_linear(context(dev), 0, x.data_ptr(), 4096, None, None, m, 4096, (ctypes.c_void_p * 1)(lin._at), 1, 0,
                                            (ctypes.c_void_p * 1)(y.data_ptr()), _stream(dev)))
        assert torch.equal(y, lin(x))
