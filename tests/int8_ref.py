"""The integer linears and the norms between them from their definitions, in 64 bits on the CPU, and the bounds
that their arithmetic keeps."""
import math

import torch

F64 = torch.float64
U = 2.0 ** -24  # half a step of f32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the smallest step of a type: what a rounding of a subnormal result is off by."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def codes(x):
    """(codes, scales) of f32 rows; whole numbers in 64 bits, NaN scales as they are."""
    x = x.float().cpu()
    fine = torch.isfinite(x).all(-1)
    amax = torch.where(fine[..., None], x, 0.0).abs().amax(-1)
    s = (amax.to(F64) / 127).float().clamp(min=2.0 ** -126)  # (the f32 quotient: 53 bits round to 24 as if exact)
    s = torch.where(amax > 0, s, 0.0)
    # 53 bits hold x - h s of an f32 x, an f32 s and a half h: no quotient beside a tie rounds onto it
    q = torch.where((s > 0)[..., None], torch.where(fine[..., None], x, 0.0).to(F64) / torch.where(s > 0, s, 1.0).to(F64)[..., None], 0.0)
    return q.round(), torch.where(fine, s, math.nan)


def product(c, s, w, t, bias):
    """(y, bound of an f32 result's error): the codes' sums are exact in 64 bits."""
    acc = c.to(F64) @ w.cpu().to(F64).t()
    y = acc * s.cpu().to(F64)[..., None] * t.cpu().to(F64)
    # the sum to f32, the scales' product, the last rounding
    bound = 2.001 * U * y.abs()
    if bias is not None:
        y = y + bias.cpu().to(F64)
    return y, bound + U * y.abs() + least(torch.float32)


def stored(y, bound, dtype):
    """The bound after one more rounding to dtype."""
    return bound if dtype == torch.float32 else bound + half_step(dtype) * (y.abs() + bound) + least(dtype)


def silu_mul(g, dg, u, du):
    """(silu(g) u, bound) of factors within dg and du of g and u.  The exponential and the reciprocal are off by a step
    of f32 (2 U each), their sum and the products by half of one."""
    sig = torch.sigmoid(g)
    silu = g * sig
    slope = (sig * (1 + g * (1 - sig))).abs() + dg  # (silu's slope, whose own is below 1/2, over dg)
    y = silu * u
    return y, slope * dg * (u.abs() + du) + silu.abs() * du + 8 * U * (y.abs() + silu.abs() * du) + least(torch.float32)


def normed(u, norm):
    """A norm dict(kind, weight, bias, eps, offset) of rows in 64 bits."""
    if norm is None:
        return u
    if norm["kind"] == "layer":
        u = u - u.mean(-1, keepdim=True)
    y = u / ((u * u).mean(-1, keepdim=True) + norm["eps"]).sqrt() * (norm["weight"].to(F64) + norm["offset"])
    return y if norm["bias"] is None else y + norm["bias"].to(F64)


def residual_norm(x, residual, post, gate, scale, norm):
    """(r, y) in 64 bits; y None without a norm."""
    u = normed(x.cpu().to(F64), post)
    if gate is not None:
        u = u * gate.cpu().to(F64)
    r = u * scale
    if residual is not None:
        r = r + residual.cpu().to(F64)
    return r, None if norm is None else normed(r, norm)


def close(got, want, bound):
    """Within the bound, NaN where the definition is."""
    got = got.detach().cpu().to(F64)
    assert got.shape == want.shape, (got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    off = (got - want).abs()[fine] - bound.expand(want.shape)[fine]
    assert not off.numel() or off.max().item() <= 0, f"{off.max().item():.3g} beyond the bound"
