"""Where the integer linears' epilogue and the norms' sums could leave their definition: gates far from zero, lanes of one row; and blocks whose
parts change, or that a graph holds."""
import pytest
import torch

import int8_ref as ref
from lightbulb_amd import attention as at
from lightbulb_amd import int8
from lightbulb_amd.quantized import Mlp
from test_gpu_int8_block import blocks, by_hand, i32, proj, qproj

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


def test_blocks_whose_projections_change(dev):
    # a projection of another kind, or another pair, after the block was made: it takes values in the place of codes, or codes again
    gen = torch.Generator().manual_seed(5)
    hidden, heads, kv, dim = 256, 4, 2, 64
    first, b = blocks(gen, dev, torch.float32, hidden, heads, kv, dim, False)
    table = at.PageTable(16, 16, 2, 8, dev)
    step = table.step(i32([0, 0], dev), i32([9, 2], dev), 11)
    x = torch.randn(11, hidden, generator=gen).to(dev)
    caches = iter([at.KvCache(16, 16, kv, dim, device=dev) for _ in range(12)])
    q, mlp = b.attention.q_proj, b.mlp
    b.attention.q_proj = qproj(gen, heads * dim, hidden, dev)
    b.mlp = Mlp(qproj(gen, 3 * hidden, hidden, dev), qproj(gen, 3 * hidden, hidden, dev), proj(gen, hidden, 3 * hidden, dev))
    h, normed = first(x, next(caches), step, next=b)
    assert isinstance(normed, torch.Tensor)
    y = b(h, next(caches), step, normed)[0]
    a = b.attention(int8.residual_norm(h, norm=b.input_norm)[1], next(caches), step)
    r, v = int8.residual_norm(a, h, norm=b.mlp_norm)
    # (the norm was formed with the update, of an h that is f32 as stored: the same values)
    assert torch.equal(y, int8.residual_norm(b.mlp(v), r)[0])
    b.attention.q_proj, b.mlp = q, mlp
    assert torch.equal(b(x, next(caches), step)[0], by_hand(b, x, next(caches), step))


@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_in_a_graph(dev, dtype):
    # a decode step of two blocks, captured once and replayed over new inputs, against the same steps by eager calls
    gen = torch.Generator().manual_seed(6)
    hidden, heads, kv, dim, n = 256, 4, 2, 64, 3
    layers = blocks(gen, dev, dtype, hidden, heads, kv, dim, True)

    def step_of(x, lens, table, caches):
        s = table.step(lens, torch.ones_like(lens), n)
        r, normed = x, None
        for i, b in enumerate(layers):
            r, normed = b(r, caches[i], s, normed=normed, next=layers[i + 1] if i + 1 < len(layers) else None)
        return r

    runs = []
    for _ in range(2):
        runs.append((at.PageTable(40, 16, n, 12, dev), [at.KvCache(40, 16, kv, dim, device=dev) for _ in layers]))
    x, lens = torch.randn(n, hidden, generator=gen).to(dtype).to(dev), i32([0] * n, dev)
    step_of(x, lens, *runs[0])
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step_of(x, lens, *runs[1])
        step_of(x, lens, *runs[1])
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step_of(x, lens, *runs[1])
    for at_token in range(1, 20):
        x.copy_(torch.randn(n, hidden, generator=gen))
        lens.fill_(at_token)
        graph.replay()
        if at_token % 3 == 0:
            torch.cuda.synchronize()
        want = step_of(x, lens, *runs[0])
        assert torch.isfinite(out).all() and torch.equal(out, want), at_token
