"""Attention over the 8-bit cache against the definition in 64 bits, with bounds from the arithmetic
(kv_ref.attention_bound), and the operators together as a layer runs them."""
import ctypes
import math
import random

import pytest
import torch

import kv_ref
from lightbulb_amd import attention as at
from lightbulb_amd import quantized as qz

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def random_codes(gen, shape, kind, dev):
    """Every code that an append writes: int8 -127 .. 127, finite e4m3."""
    if kind == "int8":
        return torch.randint(-127, 128, shape, generator=gen, dtype=torch.int8, device=dev)
    c = torch.randint(0, 254, shape, generator=gen, dtype=torch.uint8, device=dev)
    return torch.where(c >= 127, c + 1, c).view(torch.float8_e4m3fn)  # past 0x7f; 0xff is not reached


def setup(dev, kind, dtype, page, dim, kv, group, ctx, new, pad=3, seed=1, unused=None, slack=2, spread=4.0):
    """A filled cache in random pages and queries: (cache, step, q).  Pages that no sequence holds, and
    places behind a sequence's end, hold codes and scales that must not be read into a result."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    lens = [c + n for c, n in zip(ctx, new)]
    held = [-(-n // page) for n in lens]
    blocks = max(1, max(held)) + slack
    pages = sum(held) + 3
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    tables = torch.full((len(ctx), blocks), -1, dtype=torch.int32, device=dev)
    used = 0
    for b, n in enumerate(held):
        tables[b, :n] = order[used: used + n]
        used += n
    tables[tables < 0] = order[used]  # a real page, which is not the sequence's
    k, v = random_codes(gen, (pages, kv, page, dim), kind, dev), random_codes(gen, (pages, kv, dim, page), kind, dev)
    big = 127 if kind == "int8" else 448
    ks = torch.exp2(torch.rand(pages, kv, generator=gen, device=dev) * 4) * (spread / (16 * big))
    vs = torch.exp2(torch.rand(pages, kv, generator=gen, device=dev) * 12 - 6) / big
    ks[order[used:].long()], vs[order[used:].long()] = math.nan, math.nan
    for b, n in enumerate(lens):
        if n % page:
            last = int(tables[b, n // page])
            junk = -128 if kind == "int8" else 0x7f  # e4m3: NaN
            k.view(torch.int8)[last, :, n % page:] = junk
            v.view(torch.int8)[last, :, :, n % page:] = junk
    t = sum(new)
    q = torch.randn(t + pad, kv * group, dim, generator=gen, device=dev).to(dtype)
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    step = at.Step(tables, i32(lens, dev), i32(cu, dev), None, None, page_size=page, num_tokens=t + pad)
    return at.KvCache.wrap(k, v, ks, vs), step, q


def reference(q, cache, step, scale, causal=True, window=0):
    return kv_ref.attention(q, cache.k.double(), cache.v.double(), cache.k_scales, cache.v_scales, step.tables, step.seq_lens.tolist(),
                            step.cu_new.tolist(), scale, causal, window)


def check(q, cache, step, scale=None, causal=True, window=0, got=None):
    used = cache.head_dim ** -0.5 if scale is None else scale
    if got is None:
        out = torch.full(q.shape, 7.0, dtype=q.dtype, device=q.device)
        got = at.paged_attention(q, cache, step, scale=scale, causal=causal, window=window, out=out)
    want, mag, most, reach = reference(q, cache, step, used, causal, window)
    bound = kv_ref.attention_bound(q.dtype, mag, most, want, reach, step.seq_lens.max().item())
    total = step.cu_new[-1].item()
    assert (got[total:] == 7.0).all(), "rows behind the last sequence"
    off = (got[:total].double() - want[:total]).abs()
    assert (off <= bound[:total]).all(), f"off by {(off / bound[:total]).max().item():.3g} of the bound"
    return got


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,dim,kv,group", [(16, 64, 2, 4), (32, 96, 3, 1), (64, 128, 8, 4), (128, 192, 1, 7), (16, 256, 2, 2), (64, 128, 1, 71)])
def test_single_tokens(dev, kind, dtype, page, dim, kv, group):
    ctx = [0, 1, 14, 15, 16, 62, 63, 64, 127, 300, 1000]
    cache, step, q = setup(dev, kind, dtype, page, dim, kv, group, ctx, [1] * len(ctx))
    check(q, cache, step)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,dim,kv,group", [(16, 64, 2, 4), (32, 96, 1, 3), (64, 128, 2, 4), (128, 192, 1, 1), (64, 256, 1, 8), (16, 128, 1, 16)])
def test_prompts(dev, kind, dtype, page, dim, kv, group):
    ctx, new = [0, 0, 100, 0, 17, 300, 0, 1], [1, 65, 130, 0, 2, 31, 200, 4]
    cache, step, q = setup(dev, kind, dtype, page, dim, kv, group, ctx, new)
    check(q, cache, step)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 5, 150])
@pytest.mark.parametrize("window", [1, 16, 50, 64, 129, 5000])
def test_windows(dev, kind, dtype, new, window):
    cache, step, q = setup(dev, kind, dtype, 32, 64, 2, 2, [0, 100, 515], [new, new + 1, new])
    check(q, cache, step, window=window)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("src", [[1, 0, 333], [64, 128, 1500], [15, 16, 17]])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 0, 90], [200, 33, 1]])
def test_across(dev, kind, dtype, src, new):
    # a decoder's rows over an encoder's states: lengths apart; an encoder of no length gives zeros
    cache, source, _ = setup(dev, kind, dtype, 16, 64, 3, 2, src, [0, 0, 0])
    cu = [0, new[0], new[0] + new[1], sum(new)]
    mine = at.Step(torch.zeros(3, 1, dtype=torch.int32, device=dev), i32(new, dev), i32(cu, dev), None, None, page_size=64, num_tokens=cu[-1] + 2)
    q = torch.randn(cu[-1] + 2, 6, 64, device=dev).to(dtype)
    check(q, cache, mine.across(source), causal=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 4.0])
def test_scales(dev, dtype, scale):
    # flat, sharp and reversed weights
    cache, step, q = setup(dev, "int8", dtype, 64, 128, 2, 4, [200, 0, 77], [1, 90, 20])
    check(q, cache, step, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1, 1], [70, 33]])
def test_magnitudes(dev, dtype, new):
    # queries, keys and values at the ends of their types, and queries of zero
    cache, step, q = setup(dev, "int8", dtype, 16, 64, 1, 4, [200, 40], new)
    for scale_q, scale_v in ((1e-30 if dtype != torch.float16 else 1e-6, 1e-30), (1e25 if dtype != torch.float16 else 3e3, 1e3), (0.0, 1.0)):
        big = (q.float() * scale_q).to(dtype)
        c = at.KvCache.wrap(cache.k, cache.v, cache.k_scales, cache.v_scales * scale_v)
        check(big, c, step, scale=1.0 / scale_q if scale_q > 1 else None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("new", [1, 100])
def test_value_scales_far_apart(dev, dtype, kind, new):
    # pages whose values differ by twenty powers of ten, pages of zeros, in both orders
    for flip in (False, True):
        cache, step, q = setup(dev, kind, dtype, 16, 64, 1, 2, [600], [new], spread=0.5)
        pages = step.tables[0, : -(-(600 + new) // 16)].long()
        ramp = torch.logspace(-12, 3 if dtype == torch.float16 else 8, len(pages), device=dev)
        cache.v_scales[pages, 0] = (ramp.flip(0) if flip else ramp) / 448
        cache.v_scales[pages[::5], 0] = 0.0
        check(q, cache, step)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 70, 3]])
def test_rows_that_see_nothing(dev, dtype, new):
    # a sequence that was not granted (length 0), and one that is shorter than its rows
    cache, step, q = setup(dev, "e4m3", dtype, 16, 128, 2, 2, [50, 60, 1], new)
    step.seq_lens[0] = 0
    step.seq_lens[2] = max(0, new[2] - 2)
    got = check(q, cache, step)
    assert (got[: new[0]] == 0).all()


@pytest.mark.parametrize("new", [[1, 1], [130, 65]])
def test_entries_that_are_no_pages(dev, new):
    # -1 and numbers behind the last page: those keys are not there
    cache, step, q = setup(dev, "int8", torch.float32, 32, 64, 2, 4, [300, 200], new)
    for b, j, page in ((0, 0, -1), (0, 3, 1 << 30), (1, 2, cache.k.shape[0]), (1, 3, -(1 << 31))):
        step.tables[b, j] = page
    check(q, cache, step)
    step.tables[0] = -1  # none at all
    got = check(q, cache, step)
    assert (got[: new[0]] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 80])
def test_poisoned_pages(dev, dtype, new):
    # a page that reads as NaN: rows that see it are NaN, rows that do not are not
    cache, step, q = setup(dev, "int8", dtype, 16, 64, 2, 2, [100, 100], [new, new], pad=0)
    page = int(step.tables[0, 6 if new == 80 else 2])  # tokens 96 .. 111 or 32 .. 47
    for scales in (cache.k_scales, cache.v_scales):
        kept = scales[page, 1].item()
        scales[page, 1] = math.nan
        got = at.paged_attention(q, cache, step).float()
        bad = torch.isnan(got).view(2 * new, 2, 2, 64).all(3).all(2)  # [rows, kv heads]
        assert torch.isnan(got).any(2).view(2 * new, 2, 2).all(2).equal(bad)
        want = torch.zeros(2 * new, 2, dtype=torch.bool, device=dev)
        want[:new, 1] = True
        assert torch.equal(bad, want)
        scales[page, 1] = kept
    # one that only the later rows see: causal rows before it keep their values
    if new == 80:
        last = int(step.tables[0, 10])  # tokens 160 .. 175
        want, mag, most, reach = reference(q, cache, step, 64 ** -0.5)
        bound = kv_ref.attention_bound(dtype, mag, most, want, reach, 180)
        cache.k_scales[last, 0] = math.nan
        cache.v_scales[last, 1] = math.nan
        got = at.paged_attention(q, cache, step)
        assert torch.isnan(got[60:80].float()).all()
        for part in (slice(0, 60), slice(80, 160)):
            assert ((got[part].double() - want[part]).abs() <= bound[part]).all()


@pytest.mark.parametrize("new", [[1, 1], [66, 5]])
def test_queries_that_are_not_finite(dev, new):
    for bad in (math.nan, math.inf, -math.inf):
        cache, step, q = setup(dev, "int8", torch.float32, 64, 64, 1, 4, [100, 30], new, pad=0)
        clean = at.paged_attention(q, cache, step)
        q[0, 2, 9] = bad
        got = at.paged_attention(q, cache, step)
        assert torch.isnan(got[0, 2]).all()
        got[0, 2] = clean[0, 2]
        assert torch.equal(got, clean)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1, 1, 1], [70, 3, 128]])
def test_strided_queries(dev, dtype, new):
    cache, step, q = setup(dev, "int8", dtype, 64, 128, 2, 3, [64, 333, 0], new)
    want = check(q, cache, step)
    wide = torch.full((q.shape[0], 9, 131), math.nan, dtype=dtype, device=dev)
    wide[:, 1:7, 3:] = q
    assert torch.equal(at.paged_attention(wide[:, 1:7, 3:], cache, step)[: sum(new)], want[: sum(new)])
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(at.paged_attention(heads_first, cache, step)[: sum(new)], want[: sum(new)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("ctx,new", [([20000], [1]), ([9000, 50, 0], [1, 1, 1]), ([5000], [33]), ([3000, 10], [150, 1])])
def test_long_contexts(dev, dtype, kind, ctx, new):
    # work that is split over the keys, with and without the caller's bounds, and without a workspace
    cache, step, q = setup(dev, kind, dtype, 64, 128, 1, 4, ctx, new, slack=40)
    check(q, cache, step)
    lens = [c + n for c, n in zip(ctx, new)]
    hinted = at.Step(step.tables, step.seq_lens, step.cu_new, None, None, page_size=64, num_tokens=step.num_tokens, max_len=max(lens),
                     max_new=max(new))
    check(q, cache, hinted)
    check(q, cache, hinted, window=2500)


def test_without_workspace(dev, lbq):
    cache, step, q = setup(dev, "int8", torch.float32, 64, 128, 1, 4, [7000, 300], [1, 1], pad=0)
    out = torch.empty_like(q)
    for ws, n in ((None, 0), (torch.empty(4096, dtype=torch.uint8, device=dev), 4096)):
        assert lbq.lbq_kv_attention(cache._ctx, cache._struct, step._struct, 0, q.data_ptr(), q.stride(0), q.stride(1), 4, 128 ** -0.5, 1, 0,
                                    out.data_ptr(), ws.data_ptr() if n else None, n, torch.cuda.current_stream(dev).cuda_stream) == 0
        check(q, cache, step, got=out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [128, 192])
def test_long_contexts_beside_a_prompt(dev, dtype, dim):
    # single tokens' keys cut into parts whose rows are not the prompt's
    cache, step, q = setup(dev, "int8", dtype, 64, dim, 1, 4, [0, 30000, 9000, 50, 10], [700, 1, 2, 0, 4], slack=20)
    check(q, cache, step)
    hinted = at.Step(step.tables, step.seq_lens, step.cu_new, None, None, page_size=64, num_tokens=step.num_tokens, max_len=30001, max_new=700)
    check(q, cache, hinted)


def test_workspace_is_not_the_prompts(dev, lbq):
    # (parts of all 16000 tokens would be 4 GiB)
    cache, step, _ = setup(dev, "int8", torch.float32, 64, 128, 8, 4, [0, 100, 100], [16000 - 2, 1, 1], pad=0)
    wide = at.Step(step.tables, step.seq_lens, step.cu_new, None, None, page_size=64, num_tokens=16000)
    wide._struct.max_blocks = wide._struct.table_stride = 2048  # sequences of up to 131072 tokens; nothing is read
    n = ctypes.c_size_t()
    assert lbq.lbq_kv_attention_workspace(cache._ctx, cache._struct, wide._struct, 32, n) == 0
    assert 0 < n.value < 32 << 20


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,dim", [("int8", 64), ("e4m3", 128), ("int8", 256)])
def test_more_steps_than_are_looked_up_at_once(dev, lbq, dtype, kind, dim):
    # 33000 keys in one part, value scales that grow late, pages that are not there
    cache, step, q = setup(dev, kind, dtype, 64, dim, 1, 4, [33000 - 40], [40], pad=0)
    page = step.tables[0]
    cache.v_scales[page[300:520].long()] *= 1000
    page[270], page[400] = -1, cache.k.shape[0]
    out = torch.empty_like(q)
    assert lbq.lbq_kv_attention(cache._ctx, cache._struct, step._struct, at._DTYPES[dtype], q.data_ptr(), q.stride(0), q.stride(1), 4, dim ** -0.5,
                                1, 0, out.data_ptr(), None, 0, torch.cuda.current_stream(dev).cuda_stream) == 0
    check(q, cache, step, got=out)
    check(q, cache, step)


def test_same_bits_every_time(dev):
    cache, step, q = setup(dev, "int8", torch.float32, 64, 128, 2, 4, [9000, 4000, 70], [1, 40, 90])
    first = at.paged_attention(q, cache, step)[:131].clone()
    for _ in range(5):
        assert torch.equal(at.paged_attention(q, cache, step)[:131], first)


@pytest.mark.parametrize("batch", [1, 70, 4200])
def test_batches(dev, batch):
    rng = random.Random(batch)
    ctx = [rng.randint(0, 90) for _ in range(batch)]
    new = [rng.choice((0, 1, 1, 2, 30 if batch < 100 else 1)) for _ in range(batch)]
    cache, step, q = setup(dev, "int8", torch.float32, 16, 64, 1, 2, ctx, new)
    check(q, cache, step)


@pytest.mark.parametrize("batch", [2, 63, 64, 65, 256, 257])
@pytest.mark.parametrize("most", [1, 3, 150])
@pytest.mark.parametrize("hinted", [False, True])
def test_idle_sequences(dev, batch, most, hinted):
    # few of many sequences have new tokens, the first, the last and some between, of either form
    rng = random.Random(batch + most)
    new = [rng.choice((1, most, most)) if i in (0, batch - 1) or rng.random() < 0.15 else 0 for i in range(batch)]
    cache, step, q = setup(dev, "int8", torch.float32, 16, 64, 1, 4, [rng.randint(0, 60) for _ in new], new)
    if hinted:
        step = at.Step(step.tables, step.seq_lens, step.cu_new, None, None, page_size=16, num_tokens=step.num_tokens, max_len=step.seq_lens.max().item(),
                       max_new=max(new))
    check(q, cache, step)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("kv,group,ctx,new", [(1, 7, [5000], [5]), (2, 4, [300, 0, 2000], [16, 16, 3]), (1, 3, [700, 20], [21, 1]), (3, 8, [90] * 9, [5] * 9),
                                              (1, 17, [4000, 10], [1, 3]), (1, 1, [1500], [64]), (8, 2, [40] * 6, [24] * 6)])
def test_few_tokens(dev, dtype, kind, kv, group, ctx, new):
    # up to 64 rows of a kv head: tiles that end inside a token's heads
    cache, step, q = setup(dev, kind, dtype, 32, 128, kv, group, ctx, new)
    lens = [c + n for c, n in zip(ctx, new)]
    hinted = at.Step(step.tables, step.seq_lens, step.cu_new, None, None, page_size=32, num_tokens=step.num_tokens, max_len=max(lens), max_new=max(new))
    check(q, cache, step)
    check(q, cache, hinted)
    check(q, cache, hinted, window=37)
    check(q, cache, hinted, causal=False)


def test_bad_rows(dev):
    # cu_new that is no list of rows: nothing out of bounds is written
    cache, step, q = setup(dev, "int8", torch.float32, 16, 64, 1, 2, [30, 30], [4, 70], pad=0)
    out = torch.full((200, 2, 64), 7.0, device=dev)
    for cu in ([0, 4, 900], [-5, 4, 74], [74, 4, 0], [0, 90, 74]):
        bad = at.Step(step.tables, step.seq_lens, i32(cu, dev), None, None, page_size=16, num_tokens=74)
        at.paged_attention(q, cache, bad, out=out[:74])
        assert (out[74:] == 7.0).all()


def test_pages_behind_four_gib(dev):
    pages, page, h, dim = 70000, 64, 8, 128
    k = torch.zeros(pages, h, page, dim, dtype=torch.int8, device=dev)
    v = torch.zeros(pages, h, dim, page, dtype=torch.int8, device=dev)
    s = torch.zeros(pages, h, device=dev)
    used = [pages - 1, 3, 40000, 65535]
    small, step, q = setup(dev, "int8", torch.float32, page, dim, h, 4, [200], [1], pad=0, slack=0)
    src = step.tables[0].long()
    at_ = torch.tensor(used, device=dev)
    k[at_], v[at_] = small.k[src], small.v[src]
    ks, vs = s.clone(), s.clone()
    ks[at_], vs[at_] = small.k_scales[src], small.v_scales[src]
    far = at.Step(i32([used], dev), step.seq_lens, step.cu_new, None, None, page_size=page, num_tokens=1)
    want = check(q, small, step)
    assert torch.equal(at.paged_attention(q, at.KvCache.wrap(k, v, ks, vs), far), want)


def test_captured_beside_eager_calls(dev):
    # two graphs and eager calls of one cache and step: each has a workspace of its own
    cache, step, q = setup(dev, "int8", torch.float32, 64, 128, 2, 4, [5000, 100, 900], [1, 1, 60], pad=0)
    qs = [q, q * 0.5, q.flip(1).contiguous()]
    want = [at.paged_attention(x, cache, step) for x in qs]
    graphs, outs = [], []
    for x in qs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(at.paged_attention(x, cache, step))
        graphs.append(g)
    side = torch.cuda.Stream()
    for _ in range(3):
        for o in outs:
            o.fill_(3.0)
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
            eager = at.paged_attention(qs[2], cache, step)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*outs, eager), want))


@pytest.mark.parametrize("dtype", DTYPES)
def test_bounds_that_do_not_hold(dev, dtype):
    # max_len below a length: the keys behind it are not seen (a single token then sees what a step of that
    # length shows to all its rows)
    cache, step, q = setup(dev, "int8", dtype, 16, 64, 2, 4, [300, 20, 2500], [1, 1, 1], pad=0)
    for most in (10, 130, 2000):
        low = at.Step(step.tables, step.seq_lens, step.cu_new, None, None, page_size=16, num_tokens=3, max_len=most, max_new=1)
        cut = at.Step(step.tables, step.seq_lens.clamp(max=most), step.cu_new, None, None, page_size=16, num_tokens=3)
        check(q, cache, cut, causal=False, got=at.paged_attention(q, cache, low))
    # max_new below a sequence's rows: the others' are right, and nothing else is touched
    cache, step, q = setup(dev, "int8", dtype, 16, 64, 2, 4, [300, 20, 100], [4, 40, 3], pad=2)
    few = at.Step(step.tables, step.seq_lens, step.cu_new, None, None, page_size=16, num_tokens=49, max_new=4)
    out = torch.full(q.shape, 7.0, dtype=dtype, device=dev)
    at.paged_attention(q, cache, few, out=out)
    rest = at.Step(step.tables[[0, 2]], step.seq_lens[[0, 2]], i32([0, 4, 7], dev), None, None, page_size=16, num_tokens=7)
    check(torch.cat([q[:4], q[44:47]]), cache, rest, got=torch.cat([out[:4], out[44:47]]))
    assert (out[4:44] == 7.0).all() and (out[47:] == 7.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 256])
def test_more_rows_than_the_bound_gives_tiles(dev, dtype, dim):
    # a bound of 20 new tokens, which one sequence breaks: its rows are right or left as they were, the others' are right
    new = [20, 90, 7, 20]
    cache, step, q = setup(dev, "int8", dtype, 16, dim, 2, 4, [300, 20, 100, 0], new, pad=2)
    out = torch.full(q.shape, 7.0, dtype=dtype, device=dev)
    at.paged_attention(q, cache, at.Step(step.tables, step.seq_lens, step.cu_new, None, None, page_size=16, num_tokens=139, max_new=20), out=out)
    left = (out[:137] == 7.0).flatten(1).all(1)
    assert not left[:20].any() and not left[110:].any()
    filled = torch.where(left[:, None, None], check(q, cache, step)[:137], out[:137])
    check(q, cache, step, got=torch.cat([filled, out[137:]]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,new", [(33, 5), (7, 70), (3, 200)])
def test_sequences_of_one_length(dev, dtype, batch, new):
    cache, step, q = setup(dev, "e4m3", dtype, 32, 128, 2, 4, [(i * 37) % 150 for i in range(batch)], [new] * batch, pad=0)
    check(q, cache, at.Step(step.tables, step.seq_lens, step.cu_new, None, None, page_size=32, num_tokens=batch * new, max_new=new))


@pytest.mark.parametrize("new", [[1, 3, 2], [70, 3, 50]])
def test_queries_of_stride_zero(dev, new):
    # one query for all heads, one row for all tokens
    cache, step, q = setup(dev, "int8", torch.float32, 16, 64, 2, 4, [30, 200, 5], new, pad=0)
    for part in (q[:, :1].expand(q.shape), q[:1].expand(q.shape), q[:1, :1].expand(q.shape)):
        assert torch.equal(at.paged_attention(part, cache, step), at.paged_attention(part.contiguous(), cache, step))


def test_most_sequences(dev):
    # 65536 rows of a table, most of them idle
    batch, page, dim = 65536, 16, 64
    small, one, q = setup(dev, "int8", torch.float32, page, dim, 1, 2, [30, 5, 90], [1, 2, 20], pad=0)
    tables = torch.full((batch, one.tables.shape[1]), -1, dtype=torch.int32, device=dev)
    lens, new = torch.zeros(batch, dtype=torch.int32, device=dev), torch.zeros(batch, dtype=torch.int32, device=dev)
    at_ = torch.tensor([0, 40000, 65535], device=dev)
    tables[at_], lens[at_], new[at_] = one.tables, one.seq_lens, i32([1, 2, 20], dev)
    cu = torch.cat([i32([0], dev), new.cumsum(0).to(torch.int32)])
    step = at.Step(tables, lens, cu, None, None, page_size=page, num_tokens=23)
    check(q, small, one, got=at.paged_attention(q, small, step))


def test_refusals(dev):
    cache, step, q = setup(dev, "int8", torch.float32, 16, 64, 2, 2, [3], [1], pad=0)
    for bad in (q[:, :3], q.double(), q[..., :32], q[0], q.cpu(), torch.cat([q, q])):
        with pytest.raises(ValueError):
            at.paged_attention(bad, cache, step)
    for out in (torch.empty_like(q).half(), torch.empty(2, 4, 64, device=dev)[:1].expand(1, 4, 64)[:, :2], q.cpu()):
        with pytest.raises(ValueError, match="out"):
            at.paged_attention(q, cache, step, out=out)
    with pytest.raises(ValueError, match="window"):
        at.paged_attention(q, cache, step, window=-1)
    with pytest.raises(ValueError, match="window"):
        at.paged_attention(q, cache, step, causal=False, window=3)
    from lightbulb_amd._lib import LbqError
    with pytest.raises(LbqError, match="overlap"):
        at.paged_attention(q, cache, step, out=q)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def make_layer(dev, hidden, heads, kv, dim, types, rotary, window=0, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    def linear(n, k, t):
        w = torch.randn(n, k, generator=g, device=dev) * k ** -0.5
        return qz.QuantizableLinear.from_qmatmul(qz.QMatMul.from_qtensor(qz.QTensor.quantize(w, t)))
    q, k, v = linear(heads * dim, hidden, types[0]), linear(kv * dim, hidden, types[1]), linear(kv * dim, hidden, types[2])
    return at.Attention(q, k, v, linear(hidden, heads * dim, types[3]), heads, kv, dim, rotary, window=window)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("types", [(qz.GgmlDType.Q4K, qz.GgmlDType.Q4K, qz.GgmlDType.Q6K, qz.GgmlDType.Q4K), (qz.GgmlDType.Q8_0,) * 4])
def test_layer_over_steps(dev, kind, types):
    # prompts and token steps of a batch of requests through the tables, the append, the attention and
    # the projections, each step against the definitions from the same projections
    hidden, heads, kv, dim, page = 256, 4, 2, 64, 16
    rotary = at.Rotary.from_theta(dim, 16 * 12, device=dev)
    layer = make_layer(dev, hidden, heads, kv, dim, types, rotary)
    table, cache = at.PageTable(40, page, 3, 12, dev), at.KvCache(40, page, kv, dim, kind, dev)
    gen = torch.Generator(device=dev).manual_seed(11)
    lens = [0, 0, 0]
    for new in ([40, 0, 7], [1, 33, 1], [1, 1, 1], [1, 1, 1], [0, 1, 90]):
        t = sum(new)
        step = table.step(i32(lens, dev), i32(new, dev), t)
        x = torch.randn(t, hidden, generator=gen, device=dev)
        before = [cache.k.double().cpu(), cache.v.double().cpu(), cache.k_scales.double().cpu(), cache.v_scales.double().cpu()]
        got = layer.forward(x, cache, step)
        q, k, v = (p.forward(x).view(t, -1, dim) for p in (layer.q_proj, layer.k_proj, layer.v_proj))
        pos, cos, sin = step.positions.long().cpu(), rotary.cos.cpu(), rotary.sin.cpu()
        qr, kr = (kv_ref.rotate(y.cpu(), pos, cos, sin, False) for y in (q, k))
        want = kv_ref.append(*before, kind, kr, v.cpu(), step.slots.tolist(), page)
        for a, b in zip((cache.k, cache.v, cache.k_scales, cache.v_scales), want):
            assert torch.equal(a.cpu().double(), b)
        o, mag, most, reach = kv_ref.attention(qr.to(dev), *(w.to(dev) for w in want), step.tables, step.seq_lens.tolist(), step.cu_new.tolist(), dim ** -0.5)
        mine = at.paged_attention(qr.to(dev), cache, step)
        assert ((mine.double() - o).abs() <= kv_ref.attention_bound(torch.float32, mag, most, o, reach, 200)).all()
        assert torch.equal(got, layer.o_proj.forward(mine.view(t, heads * dim)))
        lens = [a + b for a, b in zip(lens, new)]


def test_layer_captured(dev):
    # a token step captured once and replayed: lengths, tables, cache and output move on by themselves
    hidden, heads, kv, dim, page, b = 256, 4, 2, 64, 16, 3
    rotary = at.Rotary.from_theta(dim, 16 * 8, device=dev)
    layer = make_layer(dev, hidden, heads, kv, dim, (qz.GgmlDType.Q8_0,) * 4, rotary, window=20)
    gen = torch.Generator(device=dev).manual_seed(12)
    xs = torch.randn(30, b, hidden, generator=gen, device=dev)

    def fresh():
        table, cache = at.PageTable(30, page, b, 8, dev), at.KvCache(30, page, kv, dim, "int8", dev)
        lens = i32([0] * b, dev)
        step = table.step(lens, i32([5, 17, 1], dev), 23)
        layer.forward(torch.randn(23, hidden, generator=torch.Generator(device=dev).manual_seed(13), device=dev), cache, step)
        return table, cache, lens.add_(i32([5, 17, 1], dev))

    one = i32([1] * b, dev)
    table, cache, lens = fresh()
    want = []
    for x in xs:
        want.append(layer.forward(x, cache, table.step(lens, one, b, max_new=1)))
        lens.add_(one)
    table2, cache2, lens2 = fresh()
    x = xs[0].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer.forward(x, cache2, table2.step(lens2, one, b, max_new=1))
        lens2.add_(one)
    for i in range(30):
        x.copy_(xs[i])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i]), i
    assert torch.equal(cache.k, cache2.k) and torch.equal(cache.v_scales, cache2.v_scales) and torch.equal(table.tables, table2.tables)


def test_layer_of_dense_and_biased_projections(dev):
    # f16 weights, regular weights with a bias, padding, and a step without tokens
    hidden, heads, kv, dim, page = 128, 4, 2, 64, 16
    g = torch.Generator(device=dev).manual_seed(5)
    rotary = at.Rotary.from_theta(dim, 200, device=dev)
    w = [torch.randn(n, hidden if i < 3 else heads * dim, generator=g, device=dev) * 0.1 for i, n in enumerate((heads * dim, kv * dim, kv * dim, hidden))]
    bias = [torch.randn(x.shape[0], generator=g, device=dev) for x in w]
    dense = [qz.QuantizableLinear.from_qmatmul(qz.QMatMul.from_qtensor(qz.QTensor(x.half().view(torch.uint8).reshape(-1), qz.GgmlDType.F16, tuple(x.shape)))) for x in w[:3]]
    regular = [qz.QuantizableLinear.from_linear(x, b) for x, b in zip(w, bias)]
    for projs in ([*dense, regular[3]], regular):
        layer = at.Attention(*projs, heads, kv, dim, rotary)
        table, cache, other = at.PageTable(20, page, 2, 8, dev), at.KvCache(20, page, kv, dim, device=dev), at.KvCache(20, page, kv, dim, device=dev)
        step = table.step(i32([0, 0], dev), i32([21, 3], dev), 30)
        x = torch.randn(1, 30, hidden, generator=g, device=dev)
        y = layer(x, cache, step)
        q, k, v = (p.forward(x).view(30, -1, dim) for p in projs[:3])
        q = other.append(k, v, step, rotary=rotary, q=q)
        want = projs[3].forward(at.paged_attention(q, other, step).view(1, 30, heads * dim))
        assert y.shape == (1, 30, hidden) and torch.allclose(y[:, :24], want[:, :24], rtol=1e-4, atol=1e-4)
        assert torch.equal(cache.k, other.k) and torch.equal(cache.v_scales, other.v_scales)
        none = table.step(i32([21, 3], dev), i32([0, 0], dev), 0)
        assert layer(x[:, :0], cache, none).shape == (1, 0, hidden)
