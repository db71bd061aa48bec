"""Integer products of the shapes that real layers have: every tile, its ragged edges and stages, and the streams of two
tiles a wave, whole outputs against exact sums.

Which kernel a shape takes goes by rows and channels; the ones named here are those of a card of 256 CUs."""
import math

import pytest
import torch

import int8_ref as ref
from lightbulb_amd import int8

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def linear(gen, n, k, dev, bias):
    w = torch.randint(-128, 128, (n, k), generator=gen, device=dev, dtype=torch.int8)
    t = (0.5 + torch.rand(n, generator=gen, device=dev)) * 2.0 ** -7 / math.sqrt(k)
    t[7 % n] = 2.0 ** -70  # (outside what f32 products of scales are used for: these waves go by 64 bits)
    return int8.Int8Linear(int8.Int8Weight(w, t), torch.randn(n, generator=gen, device=dev) if bias else None)


def rows(gen, m, k, dtype, dev):
    x = torch.randn(m, k, generator=gen, device=dev)
    if m > 4:
        x[3], x[m // 2, k - 1] = 0.0, math.nan
    if m > 4 and dtype != torch.float16:
        x[m - 1], x[m // 3] = x[m - 1] * 2.0 ** 60, x[m // 3] * 2.0 ** -80
    return x.to(dtype)


def product(x, lin):
    """ref.product of values, on the device."""
    c, s = (v.to(x.device) for v in ref.codes(x))
    y = c @ lin.weight.codes.to(ref.F64).t().contiguous() * s.to(ref.F64)[:, None] * lin.weight.scales.to(ref.F64)
    bound = 2.001 * ref.U * y.abs()
    if lin.bias is not None:
        y = y + lin.bias.to(ref.F64)
    return y, bound + ref.U * y.abs() + ref.least(torch.float32)


def close(got, y, bound, dtype):
    assert got.dtype == dtype and got.shape == y.shape
    got, bound = got.to(ref.F64), ref.stored(y, bound, dtype)
    assert torch.equal(torch.isnan(got), torch.isnan(y))
    off = ((got - y).abs() - bound)[~torch.isnan(y)]
    assert not off.numel() or off.max().item() <= 0, f"{off.max().item():.3g} beyond the bound"


def check_linears(lins, x, dtype):
    tokens = int8.quantize_tokens(x)
    ys = int8.int8_linear_group(lins, x)
    for lin, y, z in zip(lins, ys, int8.int8_linear_group(lins, tokens)):
        close(y, *product(x, lin), dtype)
        assert torch.equal(torch.nan_to_num(z.float()), torch.nan_to_num(y.float()))
    few = slice(x.shape[0] // 2 + 1, x.shape[0] // 2 + 17)  # (streamed in any case)
    for y, z in zip(ys, int8.int8_linear_group(lins, x[few])):
        assert torch.equal(y[few], z)


def check_pair(gate, up, x, dtype):
    got = int8.int8_gate_up_silu(gate, up, x)
    (g, dg), (u, du) = product(x, gate), product(x, up)
    y, bound = ref.silu_mul(g, dg, u, du)
    # (silu(g) is an f32 value: where it is subnormal, as in the channel of small scales, its own rounding is half of the least step
    # however small it is, which relative bounds do not hold, and u multiplies that)
    bound = bound + ref.least(torch.float32) * (u.abs() + du)
    if dtype != torch.float32:
        bound = bound + 2 * ref.U * g.abs() * y.abs()  # (the exponent's own rounding)
    close(got, y, bound, dtype)
    few = slice(x.shape[0] // 2 + 1, x.shape[0] // 2 + 17)
    assert torch.equal(got[few], int8.int8_gate_up_silu(gate, up, x[few]))


# k of 1, 2, 3 and 5 stages of 128
KS = [100, 256, 300, 640]
# 32 x 64, 64 x 64, 128 x 64, 128 x 128 of one weight and of three, 128 x 256, 256 x 256, and 256 x 256 with a last round of 128 x 256
SINGLE = [(70, (1003,)), (397, (2045,)), (397, (4093,)), (1021, (4093,)), (397, (4093, 1021, 1024)), (1933, (4093,)), (3891, (4091,)), (3891, (6101,))]
# 64 x 128, 128 x 128, 128 x 256, 256 x 256, and that with 128 x 256
PAIR = [(397, 1021), (397, 4093), (909, 4093), (909, 8191), (1933, 14333)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", KS)
@pytest.mark.parametrize("m,ns", SINGLE)
def test_tiles(dev, dtype, k, m, ns):
    gen = torch.Generator(dev).manual_seed(m + k)
    lins = [linear(gen, n, k, dev, (i + k // 4) % 2 == 1) for i, n in enumerate(ns)]
    check_linears(lins, rows(gen, m, k, dtype, dev), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", KS)
@pytest.mark.parametrize("m,n", PAIR)
def test_pair_tiles(dev, dtype, k, m, n):
    gen = torch.Generator(dev).manual_seed(m + k)
    check_pair(linear(gen, n, k, dev, k == 300), linear(gen, n, k, dev, k != 256), rows(gen, m, k, dtype, dev), dtype)


@pytest.mark.parametrize("m,ns", [(397, (4093, 1021, 1024)), (1933, (4093,)), (3891, (6101,))])
def test_tiles_over_long_rows(dev, m, ns):
    # 33 stages: every slot of LDS many times over
    gen = torch.Generator(dev).manual_seed(m)
    lins = [linear(gen, n, 4200, dev, i == 0) for i, n in enumerate(ns)]
    check_linears(lins, rows(gen, m, 4200, torch.bfloat16, dev), torch.bfloat16)


# k of 1, 2, 5, 8, 9 and 32 blocks of 128: one share of it, two, four and eight
STREAM_KS = [100, 256, 600, 1000, 1100, 4096]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", STREAM_KS)
@pytest.mark.parametrize("m", [1, 2, 3, 4, 9, 16, 23])
@pytest.mark.parametrize("ns", [(4096, 1024, 1000), (5003,)])
def test_streams(dev, dtype, k, m, ns):
    # two tiles a wave, quantising its values up to four tokens
    gen = torch.Generator(dev).manual_seed(m + k)
    lins = [linear(gen, n, k, dev, (i + m) % 2 == 1) for i, n in enumerate(ns)]
    check_linears(lins, rows(gen, m, k, dtype, dev), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", STREAM_KS)
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 16, 23])
@pytest.mark.parametrize("n", [1000, 4100, 8190, 14333])
def test_pair_streams(dev, dtype, k, m, n):
    # the same of a pair: one tile a wave or two, and, of two over wide pairs, k in four shares for eight
    gen = torch.Generator(dev).manual_seed(m + k + n)
    gate, up, x = linear(gen, n, k, dev, m % 2 == 0), linear(gen, n, k, dev, m % 3 == 0), rows(gen, m, k, dtype, dev)
    check_pair(gate, up, x, dtype)
    y, z = int8.int8_gate_up_silu(gate, up, x), int8.int8_gate_up_silu(gate, up, int8.quantize_tokens(x))
    assert torch.equal(torch.nan_to_num(y.float()), torch.nan_to_num(z.float()))
