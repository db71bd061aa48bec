"""Where the integer linears' epilogue and the norms' sums could leave their definition: gates far from zero, lanes of one row."""
import pytest
import torch

import int8_ref as ref
from lightbulb_amd import int8

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [2, 16, 40, 300])
def test_silu_of_far_gates_over_large_values(dev, dtype, m):
    # gates whose exponential, or its reciprocal, is beyond f32 or next to its ends: silu(gate) is an f32 value all the same, and what
    # it is multiplied by may be large.  Eight roundings (the exponential, the sum, the reciprocal, the products), for 16-bit
    # outputs also the exponent's own, |g| 2^-23, and half of f32's least value of silu times u
    g = torch.linspace(-140, -75, 1301)
    one = torch.zeros(1301, 1, dtype=torch.int8, device=dev)
    t = torch.ones(1301, device=dev)
    gate = int8.Int8Linear(int8.Int8Weight(one, t), g.to(dev))
    x = torch.ones(m, 1, dtype=dtype, device=dev)
    for u in (1.0, -1e10, 1e20, -1e30):
        up = int8.Int8Linear(int8.Int8Weight(one, t), torch.full((1301,), u, device=dev))
        u = up.bias[0].double().item()
        y = g.double() * torch.sigmoid(g.double()) * u
        bound = (8 * ref.U + (0 if dtype == torch.float32 else 2 * ref.U * g.abs())) * y.abs() + ref.least(torch.float32) * (1 + abs(u))
        ref.close(int8.int8_gate_up_silu(gate, up, x), y.expand(m, -1), ref.stored(y, bound, dtype).expand(m, -1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [128, 512, 513])
@pytest.mark.parametrize("where", [(8, 104), (40, 8), (64, 16)])
def test_equal_values_of_a_row_stay_equal(dev, dtype, k, where):
    # 2^100 and -2^100 in different quads of a row's lanes, ones elsewhere: what the mean comes to goes by the order of the sum, but
    # one row has one mean, so that its equal values have one result (up to (1 - 0) 2^-96 here, far above f32's least)
    x = torch.ones(3, k)
    x[:, 0], x[:, where[0]], x[:, where[1]] = 0.0, 2.0 ** 100, -(2.0 ** 100)
    x = x.to(dtype).to(dev)
    ones = (x[0] == 1).nonzero()[:, 0]
    n = int8.Norm(torch.ones(k, device=dev), 0.0, kind="layer")
    for y in (int8.residual_norm(x, norm=n)[1], int8.residual_norm(x, post=n)[0]):
        assert torch.isfinite(y).all() and torch.equal(y[:, ones], y[:, ones[:1]].expand(3, ones.numel()))
