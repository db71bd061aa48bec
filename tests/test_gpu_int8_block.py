"""The integer linears and norms as they are used: in Mlp, Attention and Block, on streams, in graphs, at large offsets."""
import math

import pytest
import torch

import int8_ref as ref
from lightbulb_amd import attention as at
from lightbulb_amd import int8
from lightbulb_amd.block import Block
from lightbulb_amd.quantized import GgmlDType, Mlp, QMatMul, QTensor, QuantizableLinear

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def linear(gen, n, k, dev, bias=False):
    w = torch.randint(-127, 128, (n, k), generator=gen, dtype=torch.int8).to(dev)
    t = ((0.5 + torch.rand(n, generator=gen)) * 2.0 ** -6 / math.sqrt(k)).to(dev)
    return int8.Int8Linear(int8.Int8Weight(w, t), torch.randn(n, generator=gen).to(dev) * 0.1 if bias else None)


def proj(gen, n, k, dev, bias=False):
    return QuantizableLinear.from_int8(linear(gen, n, k, dev, bias))


def qproj(gen, n, k, dev, dtype=GgmlDType.Q8_0):
    return QuantizableLinear.from_qmatmul(QMatMul.from_qtensor(QTensor.quantize((torch.randn(n, k, generator=gen) / math.sqrt(k)).to(dev), dtype)))


def norm(gen, k, dev, kind="rms"):
    return int8.Norm((1 + 0.2 * torch.randn(k, generator=gen)).to(dev), 1e-5, kind=kind, bias=(0.1 * torch.randn(k, generator=gen)).to(dev) if kind == "layer" else None)


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 7, 200])
def test_mlp(dev, dtype, m):
    gen = torch.Generator().manual_seed(m)
    g, u, d = proj(gen, 300, 128, dev), proj(gen, 300, 128, dev), proj(gen, 128, 300, dev, True)
    x = torch.randn(2, m, 128, generator=gen).to(dtype).to(dev)
    mlp = Mlp(g, u, d)
    y = mlp(x)
    h = int8.int8_gate_up_silu(g.inner, u.inner, x)
    assert y.dtype == dtype and y.shape == x.shape and torch.equal(y, d.inner(h))
    assert torch.equal(mlp(int8.quantize_tokens(x)), y)
    # one of the pair of another kind: products by themselves
    other = Mlp(g, qproj(gen, 300, 128, dev), d)
    assert other(x.float()).shape == x.shape
    with pytest.raises(ValueError, match="go to 8-bit integer linears only"):
        other(int8.quantize_tokens(x))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kinds", ["iii", "qii", "qqi", "iqi"])
def test_attention_projections(dev, dtype, kinds):
    gen = torch.Generator().manual_seed(3)
    if "q" in kinds:
        dtype = torch.float32
    heads, kv, dim, hidden = 4, 2, 64, 256
    make = {"i": proj, "q": qproj}
    q, k, v = (make[c](gen, n * dim, hidden, dev) for c, n in zip(kinds, (heads, kv, kv)))
    o = proj(gen, hidden, heads * dim, dev)
    table, cache = at.PageTable(16, 16, 2, 8, dev), at.KvCache(16, 16, kv, dim, device=dev)
    layer = at.Attention(q, k, v, o, heads, kv, dim)
    step = table.step(i32([0, 0], dev), i32([20, 3], dev), 23)
    x = torch.randn(23, hidden, generator=gen).to(dtype).to(dev)
    y = layer(x, cache, step)
    other = at.KvCache(16, 16, kv, dim, device=dev)
    qs, ks, vs = (p.forward(x).view(23, -1, dim) for p in (q, k, v))
    other.append(ks, vs, step)
    want = o.forward(at.paged_attention(qs, other, step).view(23, heads * dim))
    assert y.dtype == dtype and torch.equal(y, want)
    if kinds == "iii":
        assert torch.equal(layer(int8.quantize_tokens(x), at.KvCache(16, 16, kv, dim, device=dev), step), y)
    else:
        with pytest.raises(ValueError, match="go to 8-bit integer linears only"):
            layer(int8.quantize_tokens(x), cache, step)


def blocks(gen, dev, dtype, hidden, heads, kv, dim, extras):
    out = []
    for i in range(2):
        attention = at.Attention(proj(gen, heads * dim, hidden, dev, i == 1), proj(gen, kv * dim, hidden, dev), proj(gen, kv * dim, hidden, dev),
                                 proj(gen, hidden, heads * dim, dev), heads, kv, dim, rotary=at.Rotary.from_theta(dim, 256, 10000.0, False, dev))
        mlp = Mlp(proj(gen, 3 * hidden, hidden, dev), proj(gen, 3 * hidden, hidden, dev), proj(gen, hidden, 3 * hidden, dev))
        kw = {}
        if extras:
            kw = dict(attn_post=norm(gen, hidden, dev, "layer"), mlp_post=norm(gen, hidden, dev), scale=0.5,
                      attn_gate=torch.randn(hidden, generator=gen).to(dtype).to(dev), mlp_gate=torch.randn(hidden, generator=gen).to(dtype).to(dev))
        out.append(Block(attention, mlp, norm(gen, hidden, dev), norm(gen, hidden, dev, "layer"), **kw))
    return out


def by_hand(b, x, cache, step):
    """A block as single calls, its input norm by itself."""
    t = int8.residual_norm(x, norm=b.input_norm, quantize=True)[1]
    n, a = step.num_tokens, b.attention
    q, k, v = (p.inner(t).view(n, -1, a.head_dim) for p in (a.q_proj, a.k_proj, a.v_proj))
    q = cache.append(k, v, step, rotary=a.rotary, q=q)
    o = a.o_proj.inner(at.paged_attention(q, cache, step).reshape(n, -1))
    h, t = int8.residual_norm(o, x, post=b.attn_post, gate=b.attn_gate, scale=b.scale, norm=b.mlp_norm, quantize=True)
    y = b.mlp.down_proj.inner(int8.int8_gate_up_silu(b.mlp.gate_proj.inner, b.mlp.up_proj.inner, t))
    return int8.residual_norm(y, h, post=b.mlp_post, gate=b.mlp_gate, scale=b.scale)[0]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extras", [False, True])
def test_blocks_over_prompts_and_tokens(dev, dtype, extras):
    gen = torch.Generator().manual_seed(11)
    hidden, heads, kv, dim = 256, 4, 2, 64
    layers = blocks(gen, dev, dtype, hidden, heads, kv, dim, extras)
    table = at.PageTable(40, 16, 3, 12, dev)
    caches, others = ([at.KvCache(40, 16, kv, dim, device=dev) for _ in layers] for _ in range(2))
    lens = [0, 0, 0]
    for new in ([50, 0, 7], [1, 20, 1], [1, 1, 1], [1, 1, 1]):
        t = sum(new)
        step = table.step(i32(lens, dev), i32(new, dev), t)
        x = torch.randn(t, hidden, generator=gen).to(dtype).to(dev)
        r, normed = x, None
        for i, b in enumerate(layers):
            r, normed = b(r, caches[i], step, normed=normed, next=layers[i + 1] if i + 1 < len(layers) else None)
        assert normed is None and r.dtype == dtype and torch.isfinite(r).all()
        want = x
        for b, c in zip(layers, others):
            want = by_hand(b, want, c, step)
        # (the second block's norm is of the stream before its rounding, so that codes next to a border may turn.  Were all of them
        # rounded anew, by 0.3 of a step of 1/127 of a row's largest value, some four times its spread, each of the second block's
        # four products would be off by 1 %: 2 % in all.  A wrong row is off by all of it)
        off = (r.float() - want.float()).norm(dim=-1) / want.float().norm(dim=-1)
        assert off.max() < 0.05, off.max()
        lens = [a + b for a, b in zip(lens, new)]


def test_one_block_in_16_bits(dev):
    # a block by itself: the same calls, the same bits
    gen = torch.Generator().manual_seed(12)
    for dtype in DTYPES:
        b = blocks(gen, dev, dtype, 128, 2, 1, 64, True)[0]
        table, caches = at.PageTable(16, 16, 2, 8, dev), [at.KvCache(16, 16, 1, 64, device=dev) for _ in range(2)]
        step = table.step(i32([0, 0], dev), i32([30, 2], dev), 32)
        x = torch.randn(32, 128, generator=gen).to(dtype).to(dev)
        assert torch.equal(b(x, caches[0], step)[0], by_hand(b, x, caches[1], step))


# ---------------------------------------------------------------------------
# streams and graphs
# ---------------------------------------------------------------------------
def calls(gen, dev, m, dtype):
    """One of each call at m rows: a list of functions of x, residual."""
    k = 256
    lins = [linear(gen, n, k, dev, True) for n in (192, 64, 64)]
    pair = [linear(gen, 320, k, dev) for _ in range(2)]
    n = norm(gen, k, dev)
    return [lambda x, r: int8.int8_linear_group(lins, x), lambda x, r: [lins[0](x)], lambda x, r: [int8.int8_gate_up_silu(*pair, x)],
            lambda x, r: list(int8.residual_norm(x, r, post=n, norm=n)),
            lambda x, r: [pair[0](int8.residual_norm(x, r, norm=n, quantize=True)[1])], lambda x, r: [int8.quantize_tokens(x).dequantize()]]


@pytest.mark.parametrize("m", [1, 3, 16, 30, 70, 300])
def test_graphs(dev, m):
    # two graphs of the same linears, replayed in turn with eager calls between, on inputs that change
    gen = torch.Generator().manual_seed(m)
    fs = calls(gen, dev, m, torch.bfloat16)
    graphs = []
    for _ in range(2):
        x, r = (torch.randn(m, 256, generator=gen).bfloat16().to(dev) for _ in range(2))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for f in fs:
                f(x, r)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = [f(x, r) for f in fs]
        graphs.append((g, x, r, outs))
    for _ in range(3):
        for g, x, r, _ in graphs:
            x.copy_(torch.randn(m, 256, generator=gen))
            r.copy_(torch.randn(m, 256, generator=gen))
            g.replay()
        for f in fs:
            f(graphs[0][1], graphs[0][2])
        torch.cuda.synchronize()
        for g, x, r, outs in graphs:
            for f, out in zip(fs, outs):
                for a, b in zip(out, f(x, r)):
                    assert torch.equal(a, b)


@pytest.mark.parametrize("m", [2, 40, 260])
def test_streams(dev, m):
    # calls on two streams at once, on inputs that the streams themselves make
    gen = torch.Generator().manual_seed(m)
    fs = calls(gen, dev, m, torch.float16)
    streams = [torch.cuda.Stream() for _ in range(2)]
    base = [torch.randn(m, 256, generator=gen).half().to(dev) for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for rep in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x = base[i] * (rep + 1)
                got[i].append((x, [f(x, base[i]) for f in fs]))
    torch.cuda.synchronize()
    for i in range(2):
        for x, outs in got[i]:
            for f, out in zip(fs, outs):
                for a, b in zip(out, f(x, base[i])):
                    assert torch.equal(a, b)


def test_leaves_the_current_device(dev):
    before = torch.cuda.current_device()
    gen = torch.Generator().manual_seed(0)
    linear(gen, 16, 16, dev)(torch.ones(2, 16, device=dev))
    assert torch.cuda.current_device() == before


# ---------------------------------------------------------------------------
# large offsets
# ---------------------------------------------------------------------------
def last_rows(lin, x, y, rows):
    c, s = ref.codes(x[-rows:])
    want, bound = ref.product(c, s, lin.weight.codes, lin.weight.scales, lin.bias)
    ref.close(y[-rows:], want, ref.stored(want, bound, y.dtype))


def test_outputs_beyond_32_bits(dev):
    gen = torch.Generator().manual_seed(1)
    m, n, k = 70000, 32768, 64
    lin = linear(gen, n, k, dev)
    x = torch.randn(m, k, generator=gen).half().to(dev)
    y = lin(x)
    last_rows(lin, x, y, 3)
    assert torch.equal(y[40000:40002], lin(x[40000:40002]))
    up = linear(gen, n, k, dev)
    h = int8.int8_gate_up_silu(lin, up, x)
    assert torch.equal(h[-2:].isfinite(), torch.ones_like(h[-2:], dtype=torch.bool)) and torch.equal(h[69990:69993], int8.int8_gate_up_silu(lin, up, x[69990:69993]).to(h.dtype))


def test_codes_beyond_32_bits(dev):
    gen = torch.Generator().manual_seed(2)
    k = 16384
    w = torch.randint(-127, 128, (140000, k), dtype=torch.int8, device=dev)
    lin = int8.Int8Linear(int8.Int8Weight(w, torch.full((140000,), 2.0 ** -12, device=dev)))
    few = int8.Int8Linear(int8.Int8Weight(w[-40:], torch.full((40,), 2.0 ** -12, device=dev)))
    for m in (1, 5, 40, 300):  # weights beyond 2^31 bytes
        x = torch.randn(m, k, generator=gen).to(dev)
        assert torch.equal(lin(x)[:, -40:], few(x))
    x = torch.randn(140000, k, dtype=torch.float16, device=dev)  # tokens likewise
    t = int8.quantize_tokens(x)
    c, s = ref.codes(x[-2:])
    assert torch.equal(t.codes[-2:].cpu().double(), c) and torch.equal(t.scales[-2:].cpu(), s)
    y = few(t)
    assert torch.equal(y[-5:], few(x[-5:]))
    n = norm(gen, k, dev)
    r, v = int8.residual_norm(x, x, norm=n)
    r2, v2 = int8.residual_norm(x[-3:], x[-3:], norm=n)
    assert torch.equal(r[-3:], r2) and torch.equal(v[-3:], v2)
