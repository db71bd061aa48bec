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
