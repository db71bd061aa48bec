"""Attention over the 8-bit cache where calls are allowed and seldom made: bounds that do not hold while the
keys are cut into parts, value scales far apart, queries with one large channel, queries that are
not finite, and the defaults of a step across other sequences."""
import ctypes
import math

import pytest
import torch

import kv_ref
from lightbulb_amd import attention as at
from test_gpu_attention import DTYPES, check, i32, setup

pytestmark = pytest.mark.gpu


def attend_with_workspace(lbq, q, cache, step, out, fill):
    """The C call with a workspace of the asked size, full of one value."""
    n = ctypes.c_size_t()
    assert lbq.lbq_kv_attention_workspace(cache._ctx, cache._struct, step._struct, q.shape[1], n) == 0
    ws = torch.full((n.value // 4,), fill, device=q.device)
    assert lbq.lbq_kv_attention(cache._ctx, cache._struct, step._struct, at._DTYPES[q.dtype], q.data_ptr(), q.stride(0), q.stride(1), q.shape[1],
                                cache.head_dim ** -0.5, 1, 0, out.data_ptr(), ws.data_ptr() if n.value else None, n.value,
                                torch.cuda.current_stream(q.device).cuda_stream) == 0
    return n.value


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,batch", [(64, 2), (128, 2), (256, 2), (128, 9)])
def test_rows_behind_the_bound_are_not_joined(dev, lbq, dtype, dim, batch):
    # a bound of 60 new tokens, one tile (two above 128 channels) for each sequence, and one of 100 tokens
    # over contexts whose keys are cut into parts: rows of no tile stay as they were, whatever the workspace held
    new = [60] * batch
    new[1] = 100
    cache, step, q = setup(dev, "int8", dtype, 64, dim, 1, 4, [2000] * batch, new, pad=2)
    few = at.Step(step.tables, step.seq_lens, step.cu_new, None, None, page_size=64, num_tokens=step.num_tokens, max_new=60)
    out = torch.full(q.shape, 7.0, dtype=dtype, device=dev)
    assert attend_with_workspace(lbq, q, cache, few, out, 1e30) > 0
    first, served = 60, 64  # the sequence's first row, and its tokens in whole tiles: 256 rows of 4 heads
    assert (out[first + served: first + 100] == 7.0).all()
    filled = out.clone()
    filled[first + served: first + 100] = at.paged_attention(q, cache, step)[first + served: first + 100]
    check(q, cache, step, got=filled)


QUERY_STEP = 2.0 ** -31  # of the row's largest: what a query's channel may be off by, at the least


def row_bound(q, cache, step, scale, causal=True, window=0):
    """(out, bound) of f32, f16 or bf16 rows, element by element and from what a row itself sees, in 64 bits.

    A key's logit: its operands are held to 2^-22 and QUERY_STEP of the row's largest, and its running sum is rounded
    at most 20 times.  The exponent that it enters, with the base and the value scale's logarithm, is rounded at most 6 times,
    each half a step of the magnitudes in it.  So its weight is off by e = (2^-22 + 20 * 2^-24) sum |q k| scale
    + QUERY_STEP max |q| sum |k| scale + ln 2 * 6 * 2^-24 (|logit| + |base| + |log scale| + 15) + 16 * 2^-24 for the
    exponential's last bits, in parts of itself, and the result, to the first order, by sum p e |v| + (sum p e) |out|.
    Values: one rounding for each 16 keys and each join, 2^-24 each.  f16 parts of a weight are off by half the smallest f16
    step where the row's largest weight with its value scale is at least 2^9: 2^-34 |code| of the largest p s, for each
    key; bf16 weights are one f16 part: 2^-11.  The result is rounded once, by half a step of its type at most.  A page's scale below 2^-80 of the largest counts as that."""
    codes, scales = [cache.k.double(), cache.v.double()], [cache.k_scales.double(), cache.v_scales.double()]
    heads, kv, page, ln2 = q.shape[1], cache.kv_heads, cache.page_size, math.log(2)
    g, out, bound = heads // kv, torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lens, cu = step.seq_lens.tolist(), step.cu_new.tolist()
    half = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[q.dtype]
    tiny = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}[q.dtype]
    for b, n in enumerate(lens):
        t0, t1 = cu[b], cu[b + 1]
        if t0 == t1:
            continue
        pages = step.tables[b, : -(-n // page)].long()
        j, pos = torch.arange(n, device=q.device), n - (t1 - t0) + torch.arange(t1 - t0, device=q.device)[:, None]
        seen = (j <= pos) & ((j > pos - window) if window else (j >= 0)) if causal else torch.ones(t1 - t0, n, dtype=torch.bool, device=q.device)
        for h in range(kv):
            k = (codes[0][pages, h] * scales[0][pages, h][:, None, None]).reshape(-1, q.shape[2])[:n]
            c = codes[1][pages, h].transpose(1, 2).reshape(-1, q.shape[2])[:n]
            s = scales[1][pages, h].repeat_interleave(page)[:n]
            rows = q[t0:t1, h * g:(h + 1) * g].double()
            x = (rows @ k.t() * scale).masked_fill(~seen[:, None], -math.inf)
            p = torch.softmax(x, -1)
            logs = torch.log2(s.clamp(min=2.0 ** -80 * s.max().item())) - math.log2(s.max().item())
            base = (x / ln2 + logs).amax(-1, keepdim=True).abs()
            reach = (rows.abs() @ k.abs().t()) * abs(scale)
            ends = rows.abs().amax(-1, keepdim=True) * k.abs().sum(-1) * abs(scale)
            exponent = x.nan_to_num(neginf=0.0).abs() / ln2 + base + logs.abs() + 15
            e = (2.0 ** -22 + 20 * 2.0 ** -24) * reach + QUERY_STEP * ends + ln2 * 6 * 2.0 ** -24 * exponent + 16 * 2.0 ** -24
            assert (p * e).max() < 0.01
            v = c * s[:, None]
            o, mag = p @ v, p @ v.abs()
            most, code = (p * s).amax(-1, keepdim=True), 127.0 if cache.kind == "int8" else 448.0
            off = 1.01 * ((p * e) @ v.abs() + (p * e).sum(-1, keepdim=True) * o.abs())
            off = off + ((n / 16 + 64) * 2.0 ** -24 + (2.0 ** -11 if q.dtype == torch.bfloat16 else 0.0)) * mag
            off = off + n * 2.0 ** -34 * code * most + n * 2.0 ** -80 * code * s.max()
            out[t0:t1, h * g:(h + 1) * g] = o
            step_half = half * torch.exp2(torch.floor(torch.log2(o.abs() + off)))  # of the result's own binade
            bound[t0:t1, h * g:(h + 1) * g] = off + step_half.nan_to_num(0.0) + tiny
    return out, bound


def check_rows(q, cache, step, **kw):
    got = at.paged_attention(q, cache, step, **kw)
    want, bound = row_bound(q, cache, step, cache.head_dim ** -0.5, **kw)
    off = (got.double() - want).abs()
    assert (off <= bound).all(), f"off by {(off / bound).max().item():.3g} of the bound"
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,new", [(64, 1), (128, 1), (128, 5), (64, 100), (128, 100), (256, 40)])
@pytest.mark.parametrize("power", [-60, -40, -20])
def test_scales_of_pages_without_weight(dev, dtype, kind, dim, new, power):
    # the page that decides a row has a value scale far below that of pages whose weights are next to nothing: one
    # before it and one behind it, and short and long contexts, whole and in parts
    for ctx in (200, 3000):
        cache, step, q = setup(dev, kind, dtype, 16, dim, 1, 2, [ctx], [new], pad=0)
        pages = step.tables[0, : -(-(ctx + new) // 16)].long()
        cache.v_scales[pages] = 2.0 ** (power if dtype != torch.float16 else power / 4 - 8)
        if dtype == torch.float16:  # (the result has to be a normal number of its type)
            cache.v_scales[pages] *= 8
        # keys of the loud pages against the queries: logits lower by 40 and more
        q[:, :, 0] = 60.0
        cache.k.view(torch.int8)[pages, :, :, 0] = 0
        loud = pages[[1, len(pages) // 2, len(pages) - 2 - new // 16]]
        cache.v_scales[loud] = 1.0
        cache.k_scales[loud] = 0.25
        cache.k.view(torch.int8)[loud, :, :, 0] = -127 if kind == "int8" else -2  # (e4m3: -448)
        got = check_rows(q, cache, step)
        assert got.float().abs().max() > 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,ctx,new", [(64, 0, 64), (128, 0, 300), (256, 10, 90), (128, 2000, 40)])
def test_scales_of_pages_of_later_rows(dev, dtype, dim, ctx, new):
    # value scales that grow from page to page: a causal row is as exact as if the later pages were not there
    cache, step, q = setup(dev, "int8", dtype, 16, dim, 1, 2, [ctx], [new], pad=0)
    pages = step.tables[0, : -(-(ctx + new) // 16)].long()
    low, high = (-20, 6) if dtype == torch.float16 else (-60, 10)
    cache.v_scales[pages, 0] = torch.exp2(torch.linspace(low, high, len(pages), device=dev))
    check_rows(q, cache, step)
    cache.v_scales[pages, 0] = cache.v_scales[pages, 0].flip(0)
    check_rows(q, cache, step)
    check_rows(q, cache, step, window=30)
    check_rows(q, cache, step, causal=False)


@pytest.mark.parametrize("new", [1, 90])
def test_pages_of_zeros_first(dev, new):
    # pages whose scale is 0 stand for zeros whatever codes they hold, also where all of the first steps' are
    cache, step, q = setup(dev, "int8", torch.float32, 64, 64, 1, 2, [30000], [new], pad=0)
    pages = step.tables[0, : -(-(30000 + new) // 64)].long()
    cache.v_scales[pages] = 0.0
    assert (at.paged_attention(q, cache, step) == 0).all()
    cache.v_scales[pages[-3:]] = 2.0 ** -100
    check_rows(q, cache, step)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("new", [1, 5, 90])
def test_scales_that_grow_late(dev, kind, new):
    # whole pages of large logits under scales of 2^-70 and 0, then a single page of scale 1, which some rows weigh and
    # others do not, at any place of the steps that are looked up at once
    for place in (0, 1, 3, 40, 256, 400):
        cache, step, q = setup(dev, kind, torch.float32, 64, 64, 1, 4, [30000], [new], pad=0)
        pages = step.tables[0, : -(-(30000 + new) // 64)].long()
        cache.v_scales[pages] = 2.0 ** -70
        cache.v_scales[pages[::3]] = 0.0
        cache.v_scales[pages[place]] = 1.0
        q[:, :, 0] = torch.linspace(-60, 60, 4, device=dev)  # for the page, or against it, by the head
        cache.k.view(torch.int8)[pages, :, :, 0] = 0
        cache.k_scales[pages[place]] = 0.25
        cache.k.view(torch.int8)[pages[place], :, :, 0] = 127 if kind == "int8" else 0x7e
        check_rows(q, cache, step)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,ctx,new", [(64, 300, 1), (96, 40, 3), (128, 3000, 1), (192, 90, 5), (256, 500, 1), (128, 100, 90)])
@pytest.mark.parametrize("loud", [200.0, 8000.0, 50000.0])
def test_queries_with_one_large_channel(dev, dtype, kind, dim, ctx, new, loud):
    # a channel far above the others in which the keys are zero, or a code of 1: the other channels decide, to the same bits
    cache, step, q = setup(dev, kind, dtype, 16, dim, 2, 2, [ctx, 0, 77], [new] * 3, pad=0)
    q[:, ::2, 5] = loud
    q[:, 1::2, dim - 3] = -loud
    codes = cache.k.view(torch.int8)
    codes[..., 5] = 0
    codes[..., dim - 3] = 0
    check_rows(q, cache, step)
    codes[::7, :, ::5, 5] = 1  # (e4m3: 2^-9)
    check_rows(q, cache, step)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("new", [[1, 1], [5, 2], [66, 5]])
def test_rows_that_are_not_finite(dev, dtype, kind, new):
    # NaN whatever the keys' signs: also where all of a row's logits are -infinity, and in every form alike
    for bad, sign in ((math.inf, 0x80), (-math.inf, 0), (math.inf, 0), (math.nan, 0)):
        cache, step, q = setup(dev, kind, dtype, 64, 64, 1, 4, [100, 30], new, pad=0)
        codes = cache.k.view(torch.uint8)
        codes[..., 9] = (codes[..., 9] & 0x3f | 1) if kind == "e4m3" or not sign else 1
        if sign:
            codes[..., 9] = codes[..., 9] | 0x80
        q *= 0.1  # (so that no other channel's products are infinite)
        clean = at.paged_attention(q, cache, step)
        q[0, 2, 9] = bad
        got = at.paged_attention(q, cache, step)
        assert torch.isnan(got[0, 2]).all()
        got[0, 2] = clean[0, 2]
        assert torch.equal(got, clean)
        step.seq_lens[0] = 0  # it sees nothing: zero
        assert (at.paged_attention(q, cache, step)[0] == 0).all()


@pytest.mark.parametrize("new", [[1, 1], [90, 3]])
def test_a_step_across_sees_all_of_the_source(dev, new):
    # without a word about the mask: a decoder's rows over longer and shorter sources
    cache, source, _ = setup(dev, "int8", torch.float32, 16, 64, 2, 2, [200, 2], [0, 0])
    t = sum(new)
    mine = at.Step(torch.zeros(2, 1, dtype=torch.int32, device=dev), i32(new, dev), i32([0, new[0], t], dev), None, None, page_size=64, num_tokens=t)
    q = torch.randn(t, 4, 64, device=dev)
    want = at.paged_attention(q, cache, mine.across(source), causal=False)
    assert torch.equal(at.paged_attention(q, cache, mine.across(source)), want)
    # (a single row's causal mask is none: it is at the source's last position)
    assert torch.equal(at.paged_attention(q, cache, mine.across(source), causal=True), want) == (t == 2)
    with pytest.raises(ValueError, match="window"):
        at.paged_attention(q, cache, mine.across(source), window=5)


def test_workspace_is_bounded_beside_a_prompt(dev, lbq):
    # many single tokens beside a chunk, and a table for far longer sequences: parts for a few workgroups a CU at most,
    # of 64 rows a sequence and 130 values a row (without limit 16 parts: 68 MB for 64 sequences, 204 MB for 256)
    for batch in (8, 64, 256):
        cache, step, _ = setup(dev, "int8", torch.float32, 64, 128, 8, 4, [100] * batch, [512] + [1] * (batch - 1), pad=0)
        wide = at.Step(step.tables, step.seq_lens, step.cu_new, None, None, page_size=64, num_tokens=step.num_tokens, max_new=512)
        wide._struct.max_blocks = wide._struct.table_stride = 2048  # sequences of up to 131072 tokens; nothing is read
        n = ctypes.c_size_t()
        assert lbq.lbq_kv_attention_workspace(cache._ctx, cache._struct, wide._struct, 32, n) == 0
        cus = torch.cuda.get_device_properties(dev).multi_processor_count
        short = max(1, 4 * cus // (batch * 8)) * batch * 4 * 32
        long = max(1, 256 // ((512 + batch) * 4 // 256 * 8)) * step.num_tokens * 32
        assert n.value <= (short + long) * 130 * 4


@pytest.mark.parametrize("kv,group,ctx,new", [(8, 4, [4000] * 12, [1] * 12), (2, 4, [5000, 70], [1, 1]), (8, 4, [3000] * 6, [1, 5, 1, 3, 1, 1]), (1, 17, [9000, 10, 0], [1, 2, 1])])
def test_parts_without_a_bound_on_new_tokens(dev, lbq, kv, group, ctx, new):
    # the parts go by the tokens that are there, not by the most that a sequence could have of them
    cache, step, q = setup(dev, "int8", torch.float32, 64, 128, kv, group, ctx, new, pad=0, slack=0)
    out = torch.full(q.shape, 7.0, device=dev)
    assert attend_with_workspace(lbq, q, cache, step, out, math.nan) > 0
    check(q, cache, step, got=out)


def test_bounds_beyond_32_bits(dev):
    cache, step, q = setup(dev, "int8", torch.float32, 16, 64, 2, 2, [300, 2], [1, 20], pad=0)
    want = at.paged_attention(q, cache, step)
    free = at.Step(step.tables, step.seq_lens, step.cu_new, None, None, page_size=16, num_tokens=21, max_len=2 ** 32 + 10, max_new=2 ** 32 + 1)
    assert torch.equal(at.paged_attention(q, cache, free), want)
    table = at.PageTable(8, 16, 1, 8, dev)
    step = table.step(i32([0], dev), i32([100], dev), 100, max_len=2 ** 32 + 10, max_new=2 ** 32 + 1)
    assert step._struct.max_len == step._struct.max_new == 2 ** 31 - 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,ctx,new", [(64, 700, 1), (128, 90, 1), (128, 3000, 4), (64, 10, 130), (128, 0, 300), (192, 40, 70)])
def test_rows_by_what_they_see(dev, dtype, kind, dim, ctx, new):
    # ordinary rows by the narrow bound (f16 results from weights of one f16 part are outside it)
    cache, step, q = setup(dev, kind, dtype, 32, dim, 2, 2, [ctx, 50], [new, 2], pad=0, spread=1.0)
    check_rows(q, cache, step)
    check_rows(q, cache, step, window=40)
