"""Codes by token and products of 8-bit integers against their definitions in 64 bits."""
import math

import pytest
import torch

import int8_ref as ref
from lightbulb_amd import int8

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def values(gen, m, k, dtype, spread=1.0):
    x = torch.randn(m, k, generator=gen) * torch.where(torch.rand(k, generator=gen) < 0.05, 8.0, 1.0) * spread
    return x.to(dtype)


def weight(gen, n, k, dev, bias=False):
    w = torch.randint(-127, 128, (n, k), generator=gen, dtype=torch.int8)
    t = (0.5 + torch.rand(n, generator=gen)) * 2.0 ** -7 / math.sqrt(k)
    return int8.Int8Linear(int8.Int8Weight(w.to(dev), t.to(dev)), torch.randn(n, generator=gen).to(dev) if bias else None)


def check_linear(lin, xs, got, dtype):
    c, s = ref.codes(xs)
    y, bound = ref.product(c, s, lin.weight.codes, lin.weight.scales, lin.bias)
    ref.close(got, y, ref.stored(y, bound, dtype))


def check_tokens(got, xs):
    c, s = ref.codes(xs)
    assert torch.equal(got.codes.cpu().double(), c.to(torch.float64))
    assert torch.equal(torch.nan_to_num(got.scales.cpu(), nan=-1.0), torch.nan_to_num(s, nan=-1.0))
    rows = got._rows.cpu()
    assert not rows[:, xs.shape[-1]:].any()  # the rows' ends


# ---------------------------------------------------------------------------
# codes
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (5, 64), (2, 129), (9, 500), (4, 513), (7, 2047), (3, 2049), (2, 4096), (3, 5000), (2, 8193),
                                 (1, 16384), (2, 16385), (1, 40001), (2, 65537), (1, 131071)])
def test_codes(dev, dtype, m, k):
    gen = torch.Generator().manual_seed(m + k)
    x = values(gen, m, k, dtype).to(dev)
    check_tokens(int8.quantize_tokens(x), x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_codes_of_ties_and_ends(dev, dtype):
    # scales that are powers of two times odd numbers: quotients that fall on halves, and next to them
    rows = []
    for unit in (1.0, 3.0, 2.0 ** -9, 5.0 * 2.0 ** -14, 2.0 ** 8):
        row = torch.arange(-127, 127.5, 0.5) * unit
        rows.append(torch.cat([row, torch.zeros(521 - row.numel())]))
    near = torch.cat([torch.arange(-127, 127.5, 0.5) + d for d in (2.0 ** -12, -(2.0 ** -12))]).clamp(-127, 127)[:521]
    rows.append(torch.cat([near, torch.zeros(521 - near.numel())]))
    x = torch.stack(rows).to(dtype).to(dev)
    check_tokens(int8.quantize_tokens(x), x)


def test_codes_of_odd_values(dev):
    k = 300
    tiny, big = torch.finfo(torch.float32).smallest_normal, torch.finfo(torch.float32).max
    x = torch.zeros(12, k)
    x[0] = 0.0
    x[1, 3] = math.inf
    x[2, 299] = math.nan
    x[3] = -0.0
    x[4] = torch.linspace(-1, 1, k) * tiny  # subnormals under the least scale
    x[5, 7] = torch.finfo(torch.float32).smallest_normal * 2.0 ** -23
    x[6] = torch.linspace(-1, 1, k) * big
    x[7] = torch.linspace(-1, 1, k) * tiny * 127
    x[8] = -math.inf
    x[9, 0], x[9, 1] = math.inf, math.nan
    x[10] = 1.0
    x[11] = torch.linspace(0, 1, k)
    x = x.to(dev)
    check_tokens(int8.quantize_tokens(x), x)
    for dtype, top in ((torch.float16, 65504.0), (torch.bfloat16, 3e38)):
        y = torch.stack([torch.linspace(-1, 1, k) * top, torch.linspace(-1, 1, k) * 6e-8, torch.full((k,), math.inf)]).to(dtype).to(dev)
        check_tokens(int8.quantize_tokens(y), y)


@pytest.mark.parametrize("dtype", DTYPES)
def test_codes_of_strided_rows(dev, dtype):
    gen = torch.Generator().manual_seed(4)
    base = values(gen, 12, 700, dtype).to(dev)
    for x in (base[:, 1:], base[:, 3:516], base[::2, :77], base[1:2].expand(5, 700), base.view(3, 4, 700), base.view(3, 4, 700)[:, ::2],
              base.view(3, 4, 700)[:, :1, 5:600], base[:, 5:6], base[3:3]):
        got = int8.quantize_tokens(x)
        assert got.shape == x.shape and got.codes.shape == x.shape and got.scales.shape == x.shape[:-1]
        if x.numel():
            c, s = ref.codes(x)
            assert torch.equal(got.codes.cpu().double(), c) and torch.equal(got.scales.cpu(), s)


def test_weights_from_values(dev):
    gen = torch.Generator().manual_seed(5)
    for dtype in DTYPES:
        w = values(gen, 33, 260, dtype, 0.02).to(dev)
        q = int8.Int8Weight.quantize(w)
        c, s = ref.codes(w)
        assert torch.equal(q.codes.cpu().double(), c) and torch.equal(q.scales.cpu(), s) and q.shape() == (33, 260)
        assert ((q.dequantize().cpu() - w.float().cpu()).abs() <= 0.5001 * s[:, None]).all()


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 33, 64), (2, 100, 129), (3, 257, 1000), (4, 16, 4096), (5, 130, 333), (8, 1000, 127), (15, 47, 640),
                                   (16, 64, 2048), (17, 63, 128), (31, 129, 511), (33, 300, 1024), (64, 31, 4096), (65, 200, 100), (100, 500, 77),
                                   (128, 128, 128), (129, 1, 2000), (200, 385, 1500), (257, 513, 384), (513, 260, 640), (1000, 66, 256)])
def test_linear(dev, dtype, m, n, k):
    gen = torch.Generator().manual_seed(m * n + k)
    x = values(gen, m, k, dtype).to(dev)
    lin = weight(gen, n, k, dev, bias=n % 2 == 1)
    check_linear(lin, x, lin(x), dtype)


@pytest.mark.parametrize("m", [1, 4, 16, 40, 130])
@pytest.mark.parametrize("out", DTYPES)
def test_output_types(dev, m, out):
    gen = torch.Generator().manual_seed(m)
    for dtype in DTYPES:
        x = values(gen, m, 320, dtype).to(dev)
        lin = weight(gen, 90, 320, dev)
        y = lin(x, dtype=out)
        assert y.dtype == out
        check_linear(lin, x, y, out)
        assert torch.equal(lin(int8.quantize_tokens(x), dtype=out), y)  # codes made before: the same bits
        assert lin(int8.quantize_tokens(x)).dtype == dtype


@pytest.mark.parametrize("k", [64, 1000, 4096])
def test_rows_do_not_go_by_their_batch(dev, k):
    gen = torch.Generator().manual_seed(k)
    x = values(gen, 700, k, torch.float32).to(dev)
    lin, up = weight(gen, 192, k, dev, bias=True), weight(gen, 192, k, dev)
    y, h = lin(x), int8.int8_gate_up_silu(lin, up, x)
    for m in (1, 2, 3, 4, 5, 16, 17, 33, 64, 65, 128, 129, 300):
        assert torch.equal(lin(x[7:7 + m]), y[7:7 + m]), m
        assert torch.equal(int8.int8_gate_up_silu(lin, up, x[7:7 + m]), h[7:7 + m]), m


@pytest.mark.parametrize("m", [1, 3, 16, 50, 140, 300])
@pytest.mark.parametrize("ns", [(64,), (128, 32, 32), (33, 1, 100, 17), (200, 300)])
def test_group(dev, m, ns):
    gen = torch.Generator().manual_seed(m)
    x = values(gen, m, 384, torch.bfloat16).to(dev)
    lins = [weight(gen, n, 384, dev, bias=i % 2 == 0) for i, n in enumerate(ns)]
    for lin, y in zip(lins, int8.int8_linear_group(lins, x)):
        check_linear(lin, x, y, torch.bfloat16)
        assert torch.equal(y, lin(x))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k,bias", [(1, 1, 1, False), (1, 129, 512, True), (2, 64, 1000, False), (4, 200, 4096, False), (7, 33, 130, True),
                                        (16, 320, 768, False), (40, 100, 257, False), (65, 47, 384, True), (130, 300, 640, False),
                                        (300, 65, 200, False), (600, 260, 128, True)])
def test_gate_up(dev, dtype, m, n, k, bias):
    gen = torch.Generator().manual_seed(m + n + k)
    x = values(gen, m, k, dtype).to(dev)
    gate, up = weight(gen, n, k, dev, bias), weight(gen, n, k, dev, bias)
    got = int8.int8_gate_up_silu(gate, up, x)
    c, s = ref.codes(x)
    y, bound = ref.silu_mul(*ref.product(c, s, gate.weight.codes, gate.weight.scales, gate.bias),
                            *ref.product(c, s, up.weight.codes, up.weight.scales, up.bias))
    ref.close(got, y, ref.stored(y, bound, dtype))


def test_silu_far_from_zero(dev):
    # a gate of -200 to 200: the exponential's own range and beyond it
    g = torch.linspace(-200, 200, 801)
    x = torch.ones(2, 1, device=dev)
    one, bias = torch.zeros(801, 1, dtype=torch.int8, device=dev), torch.ones(801, device=dev)
    gate = int8.Int8Linear(int8.Int8Weight(one, bias), g.to(dev))
    up = int8.Int8Linear(int8.Int8Weight(one, bias), bias)
    got = int8.int8_gate_up_silu(gate, up, x)
    y = g.double() * torch.sigmoid(g.double())
    # below -87.3 the result is under 2^-119 and zero stands for it
    ref.close(got, y.expand(2, -1), (8 * ref.U * y.abs() + torch.where(g < -87.3, y.abs(), 0.0)).expand(2, -1) + 1e-45)


@pytest.mark.parametrize("m", [1, 16, 64, 200])
def test_rows_without_values(dev, m):
    # zero rows give the bias, rows that are not finite NaN, and neither touches its neighbours
    gen = torch.Generator().manual_seed(m)
    x = values(gen, m, 512, torch.float32)
    x[0] = 0.0
    if m > 1:
        x[m // 2, 17], x[m - 1, 511] = math.nan, -math.inf
    x = x.to(dev)
    lin, up = weight(gen, 70, 512, dev, bias=True), weight(gen, 70, 512, dev)
    y = lin(x)
    check_linear(lin, x, y, torch.float32)
    assert torch.equal(y[0], lin.bias)
    h = int8.int8_gate_up_silu(lin, up, x)
    assert torch.equal(torch.isnan(h).all(1), torch.isnan(y).all(1)) and not h[0].any()
    bad = lin(torch.full((m, 512), math.nan, device=dev))
    assert torch.isnan(bad).all()


@pytest.mark.parametrize("m", [1, 5, 33, 130])
def test_scales_of_any_size(dev, m):
    # beside the usual range: products of scales that would overflow or lose their bits in f32
    gen = torch.Generator().manual_seed(m)
    k = 200
    x = values(gen, m, k, torch.float32) * torch.exp2(torch.randint(-120, 100, (m, 1), generator=gen).float())
    w = torch.randint(-127, 128, (150, k), generator=gen, dtype=torch.int8)
    t = torch.exp2(torch.randint(-126, 100, (150,), generator=gen).float()) * (1 + torch.rand(150, generator=gen))
    t[5], t[6] = 0.0, 2.0 ** -140
    x = x.to(dev)
    lin = int8.Int8Linear(int8.Int8Weight(w.to(dev), t.to(dev)))
    c, s = ref.codes(x)
    y, bound = ref.product(c, s, w, t, None)
    over = y.abs() > torch.finfo(torch.float32).max * (1 + 2.0 ** -24)
    got = lin(x).cpu()
    assert torch.equal(torch.isinf(got), over) and not torch.isnan(got).any()
    ref.close(torch.where(over, 0.0, got.double()), torch.where(over, 0.0, y), bound)


def test_longest_sums(dev):
    # k = 131071 of codes -128 (from a checkpoint) and -127: sums next to 2^31
    k = int8.MAX_K
    x = torch.full((3, k), -1.0, device=dev)
    x[1], x[2, ::2] = 1.0, 0.0
    for code in (-128, 127):
        w = torch.full((5, k), code, dtype=torch.int8, device=dev)
        lin = int8.Int8Linear(int8.Int8Weight(w, torch.full((5,), 2.0 ** -20, device=dev)))
        check_linear(lin, x, lin(x), torch.float32)
        t = int8.quantize_tokens(x)
        t._rows[:, :k] = -128  # codes that a caller made
        y, bound = ref.product(t.codes.cpu(), t.scales, w, lin.weight.scales, None)
        ref.close(lin(t), y, bound)


@pytest.mark.parametrize("m", [2, 20, 70])
def test_inputs_as_they_lie(dev, m):
    gen = torch.Generator().manual_seed(m)
    lin = weight(gen, 48, 250, dev, bias=True)
    base = values(gen, 2 * m, 600, torch.float16).to(dev)
    for x in (base[:m, 1:251], base[::2, 300:550], base[:1, 7:257].expand(m, 250), base[:, :250].unflatten(0, (2, m)),
              base[:, 2:252].unflatten(0, (2, m))[:, :1]):
        y = lin(x)
        assert y.shape == (*x.shape[:-1], 48)
        check_linear(lin, x.reshape(-1, 250), y.reshape(-1, 48), torch.float16)
    # a weight's codes that are rows of a wider matrix, or begin at an odd byte
    wide = torch.randint(-127, 128, (48, 777), generator=gen, dtype=torch.int8).to(dev)
    for w in (wide[:, 5:255], wide[:, :256], wide.flatten()[3:3 + 48 * 256].view(48, 256)):
        l2 = int8.Int8Linear(int8.Int8Weight(w, lin.weight.scales))
        x = base[:m, :w.shape[1]]
        check_linear(l2, x, l2(x), torch.float16)


def test_no_rows(dev):
    gen = torch.Generator().manual_seed(0)
    lin = weight(gen, 40, 64, dev)
    assert lin(torch.empty(0, 64, device=dev)).shape == (0, 40)
    assert lin(torch.empty(3, 0, 64, device=dev, dtype=torch.bfloat16)).shape == (3, 0, 40)
    assert int8.int8_gate_up_silu(lin, lin, torch.empty(0, 64, device=dev)).shape == (0, 40)
    assert lin(int8.quantize_tokens(torch.empty(0, 64, device=dev))).shape == (0, 40)
