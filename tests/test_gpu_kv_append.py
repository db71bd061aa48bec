"""Appends to the 8-bit cache against their definition in 64 bits: codes and scales are equal, bit for bit."""
import math

import pytest
import torch

import kv_ref
from lightbulb_amd import attention as at

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def values(cache):
    """The cache's codes as 64-bit values, and its scales, on the CPU."""
    return [cache.k.cpu().double(), cache.v.cpu().double(), cache.k_scales.cpu().double(), cache.v_scales.cpu().double()]


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=-7e77), torch.nan_to_num(b.to(a.dtype), nan=-7e77))


def rows(gen, t, h, d, dtype, dev, spread=1.0):
    x = torch.randn(t, h, d, generator=gen) * spread * torch.exp2(torch.randint(-3, 4, (t, h, 1), generator=gen).float())
    return x.to(dtype).to(dev)


def append_and_check(cache, step, k, v, rotary=None, q=None):
    before = values(cache)
    got = cache.append(k, v, step, rotary=rotary, q=q)
    slots, kr = step.slots.tolist(), k.float().cpu()
    live = torch.tensor([s >= 0 for s in slots], dtype=torch.bool)
    if rotary is not None:
        pos = step.positions.cpu().long().clamp(min=0)
        cos, sin = rotary.cos.cpu(), rotary.sin.cpu()
        kr = kv_ref.rotate(kr, pos, cos, sin, rotary.interleaved)
        if q is not None:
            want = kv_ref.rotate(q.float().cpu(), pos, cos, sin, rotary.interleaved).to(q.dtype)
            assert torch.equal(got.cpu()[live], want[live])
    want = kv_ref.append(*before, cache.kind, kr, v.float().cpu(), slots, cache.page_size)
    for name, a, b in zip(("k", "v", "k_scales", "v_scales"), values(cache), want):
        assert same(a, b), name
    return got


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,dim,heads", [(16, 64, 1), (16, 128, 8), (32, 96, 3), (64, 128, 2), (64, 192, 1), (128, 256, 2), (128, 64, 5)])
def test_prompts_then_tokens(dev, kind, dtype, page, dim, heads):
    # prompts of odd lengths, then a few tokens at a time into partly filled pages, whose scales
    # grow now and then
    gen = torch.Generator().manual_seed(page + dim)
    table = at.PageTable(24, page, 4, 5, dev)
    cache = at.KvCache(24, page, heads, dim, kind, dev)
    lens = [0, 0, 0, 0]
    for new in ([page + 3, 1, 0, 2 * page], [1, 1, 7, 1], [1, page - 2, 1, 0], [3, 1, page + 1, page - 1]):
        t = sum(new)
        step = table.step(i32(lens, dev), i32(new, dev), t + 5)
        pad = lambda x: torch.cat([x, x[:1].expand(5, -1, -1)])  # noqa: E731  (rows behind the last sequence)
        k, v = pad(rows(gen, t, heads, dim, dtype, dev)), pad(rows(gen, t, heads, dim, dtype, dev, 0.1))
        append_and_check(cache, step, k, v)
        lens = [a + b for a, b in zip(lens, new)]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 128), (128, 64), (96, 20), (256, 2)])
def test_rotation(dev, kind, dtype, interleaved, dim, rot):
    gen = torch.Generator().manual_seed(rot)
    table = at.PageTable(40, 16, 3, 20, dev)
    cache = at.KvCache(40, 16, 2, dim, kind, dev)
    rotary = at.Rotary.from_theta(rot, 320, 10000.0, interleaved, dev)
    lens = [0, 0, 0]
    for new in ([33, 0, 200], [1, 5, 1], [2, 1, 19]):
        t = sum(new)
        step = table.step(i32(lens, dev), i32(new, dev), t + 3, max_new=max(new))
        pad = lambda x: torch.cat([x, x[:1].expand(3, -1, -1)])  # noqa: E731
        k, v, q = (pad(rows(gen, t, h, dim, dtype, dev)) for h in (2, 2, 6))
        append_and_check(cache, step, k, v, rotary, q)
        lens = [a + b for a, b in zip(lens, new)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rot", [(128, 128), (64, 32)])
def test_views_of_one_projection(dev, dtype, dim, rot):
    # q, k and v as slices of one row, at an odd offset of it, heads and channels apart
    gen = torch.Generator().manual_seed(9)
    t, hq, h = 37, 4, 2
    wide = torch.randn(t, (hq + 2 * h) * dim + 3, generator=gen).to(dtype).to(dev)
    q, k, v = wide[:, 1: 1 + (hq + 2 * h) * dim].split([hq * dim, h * dim, h * dim], 1)
    q, k, v = q.unflatten(1, (hq, dim)), k.unflatten(1, (h, dim)), v.unflatten(1, (h, dim))
    by_heads = torch.randn(h, t, dim, generator=gen).to(dtype).to(dev).transpose(0, 1)
    rotary = at.Rotary.from_theta(rot, 64, 500.0, False, dev)
    for keys in (k, by_heads, by_heads[:, :1].expand(t, h, dim)):  # the last: one head's row for both
        table, cache = at.PageTable(8, 16, 1, 4, dev), at.KvCache(8, 16, h, dim, "int8", dev)
        append_and_check(cache, table.step(i32([0], dev), i32([t], dev), t), keys, v, rotary, q)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_ties_and_extremes(dev, kind):
    # quotients that lie on or next to a tie, the largest and smallest magnitudes, zeros
    page, dim = 16, 64
    table, cache = at.PageTable(16, page, 1, 12, dev), at.KvCache(16, page, 1, dim, kind, dev)
    gen = torch.Generator().manual_seed(4)
    blocks = []
    for top in (127.0, 1.0, 3.3e38, 1e-37, 1.5e-45, 448.0, 392.0, 0.1):
        x = torch.randint(-254, 255, (page, dim), generator=gen).double() / 2 * (top / 127)
        near = torch.randint(-1, 2, (page, dim), generator=gen)
        x = x.float()
        x = torch.where(near > 0, torch.nextafter(x, torch.tensor(math.inf)), torch.where(near < 0, torch.nextafter(x, torch.tensor(-math.inf)), x))
        x = x.clamp(-top, top)
        x[3, 5] = top
        blocks.append(x)
    blocks.append(torch.zeros(page, dim))
    k = torch.cat(blocks)[:, None].to(dev)
    t = k.shape[0]
    append_and_check(cache, table.step(i32([0], dev), i32([t], dev), t), k, k.flip(0).contiguous())


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_growing_scales(dev, kind):
    # token by token, each larger than the last: every append codes the page again; then smaller
    # ones, which leave it
    page, dim, h = 32, 64, 2
    table, cache = at.PageTable(4, page, 1, 2, dev), at.KvCache(4, page, h, dim, kind, dev)
    gen = torch.Generator().manual_seed(5)
    for i in range(40):
        k, v = (torch.randn(1, h, dim, generator=gen) * (1.37 ** min(i, 25)) for _ in range(2))
        append_and_check(cache, table.step(i32([i], dev), i32([1], dev), 1), k.to(dev), v.to(dev))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite(dev, kind, bad):
    # the (page, head) they fall into reads as NaN from then on; other heads and pages do not
    table, cache = at.PageTable(6, 16, 1, 4, dev), at.KvCache(6, 16, 2, 64, kind, dev)
    gen = torch.Generator().manual_seed(6)
    lens = 0
    for n, where in ((20, None), (3, (1, 0, 7)), (2, None), (12, None)):
        k, v = torch.randn(n, 2, 64, generator=gen), torch.randn(n, 2, 64, generator=gen)
        if where:
            k[where] = bad
        append_and_check(cache, table.step(i32([lens], dev), i32([n], dev), n), k.to(dev), v.to(dev))
        lens += n
    page = int(table.tables[0, 1])
    assert math.isnan(cache.k_scales[page, 0].item()) and not torch.isnan(cache.k_scales[page, 1])
    assert not torch.isnan(cache.v_scales).any() and int(torch.isnan(cache.k_scales).sum()) == 1


def test_position_behind_the_angles(dev):
    table, cache = at.PageTable(4, 16, 1, 4, dev), at.KvCache(4, 16, 1, 64, "int8", dev)
    rotary = at.Rotary.from_theta(32, 20, device=dev)
    x = torch.randn(24, 1, 64, device=dev)
    q = cache.append(x, x, table.step(i32([0], dev), i32([24], dev), 24), rotary=rotary, q=x)
    assert torch.isfinite(q[:20]).all() and torch.isnan(q[20:, :, :32]).all() and torch.equal(q[20:, :, 32:], x[20:, :, 32:])
    pages = table.tables[0, :2].long()
    assert torch.isfinite(cache.k_scales[pages[0]]) and torch.isnan(cache.k_scales[pages[1]]) and torch.isfinite(cache.v_scales).all()


def test_sequences_without_slots_leave_the_cache(dev):
    # not granted, idle, and bad slots made by hand: nothing outside the granted pages changes
    table, cache = at.PageTable(3, 16, 3, 4, dev), at.KvCache(3, 16, 1, 64, "int8", dev)
    x = torch.randn(60, 1, 64, device=dev)
    step = table.step(i32([0, 0, 0], dev), i32([20, 40, 0], dev), 60)
    assert step.granted.tolist() == [1, 0, 1]
    append_and_check(cache, step, x, x)
    before = values(cache)
    n = 4
    for slots in ([-1] * n, [48, 49, 50, 51], [1 << 40] * n, [-9] * n, [17, 18, 19, 20]):  # none, behind the last page, misplaced
        bad = at.Step(step.tables, i32([n, 0, 0], dev), i32([0, n, n, n], dev), torch.tensor(slots, device=dev), i32(range(n), dev),
                      page_size=16, num_tokens=n)
        cache.append(x[:n], x[:n], bad)
        assert all(same(a, b) for a, b in zip(values(cache), before)), slots
    for cu, lens in (([0, n + 9, n, n], [n + 9, 0, 0]), ([-3, n, n, n], [n, 0, 0]), ([n, 0, 0, 0], [n, n, n]), ([0, n, n, n], [2, 0, 0])):
        bad = at.Step(step.tables, i32(lens, dev), i32(cu, dev), torch.arange(n, device=dev), i32(range(n), dev), page_size=16, num_tokens=n)
        cache.append(x[:n], x[:n], bad)
        assert all(same(a, b) for a, b in zip(values(cache), before)), cu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 96])
def test_rows_of_stride_zero(dev, dtype, dim):
    # one head's keys for all heads, one token's values for all tokens
    table, cache = at.PageTable(9, 32, 2, 4, dev), at.KvCache(9, 32, 3, dim, "int8", dev)
    step = table.step(i32([0, 0], dev), i32([70, 5], dev), 75)
    k = torch.randn(75, 1, dim, device=dev).to(dtype).expand(75, 3, dim)
    v = torch.randn(1, 3, dim, device=dev).to(dtype).expand(75, 3, dim)
    rotary = at.Rotary.from_theta(dim, 80, device=dev)
    got = cache.append(k, v, step, rotary=rotary, q=k)
    other = at.KvCache(9, 32, 3, dim, "int8", dev)
    want = other.append(k.contiguous(), v.contiguous(), step, rotary=rotary, q=k.contiguous())
    assert torch.equal(got, want) and all(same(a, b) for a, b in zip(values(cache), values(other)))


def test_more_tokens_than_the_bound(dev):
    # max_new is the caller's word: a sequence that breaks it is not served, and nothing else is touched
    table, cache = at.PageTable(8, 16, 2, 4, dev), at.KvCache(8, 16, 1, 64, "int8", dev)
    step = table.step(i32([0, 0], dev), i32([30, 2], dev), 32, max_new=2)
    x = torch.randn(32, 1, 64, device=dev)
    cache.append(x, x, step)
    first, second = table.tables[0, :2].long(), table.tables[1, :1].long()
    assert (cache.k_scales[first] == 0).all() and (cache.k[first] == 0).all()
    want = kv_ref.block_scale(x[30:, 0].cpu(), "int8")
    assert cache.k_scales[second].item() == cache.v_scales[second].item() == want


def test_pages_behind_four_gib(dev):
    # codes whose offsets pass 32 bits
    pages, page, h, dim = 70000, 64, 8, 128
    cache = at.KvCache.wrap(torch.empty(pages, h, page, dim, dtype=torch.int8, device=dev), torch.empty(pages, h, dim, page, dtype=torch.int8, device=dev),
                            torch.zeros(pages, h, device=dev), torch.zeros(pages, h, device=dev))
    # (the pool is the cache's: three of its pages are free)
    free = torch.cat([i32([5, pages - 1, 40000], dev), i32([0] * (pages - 3), dev)])
    table = at.PageTable.wrap(torch.full((1, 4), -1, dtype=torch.int32, device=dev), free, i32([3], dev), page)
    x = torch.randn(130, h, dim, device=dev)
    cache.append(x, x, table.step(i32([0], dev), i32([130], dev), 130))
    gen = table.tables[0, :3].tolist()
    assert gen == [40000, pages - 1, 5]
    xs = x.cpu()
    for j, pg in enumerate(gen):
        part = xs[64 * j: 64 * (j + 1)]
        for i in (0, 7):
            s = kv_ref.block_scale(part[:, i], "int8")
            want = kv_ref.codes(part[:, i].double(), s, "int8")
            assert torch.equal(cache.k[pg, i, : part.shape[0]].cpu().double(), want)
            assert torch.equal(cache.v[pg, i, :, : part.shape[0]].cpu().double(), want.t())


def test_python_refusals(dev):
    table, cache = at.PageTable(4, 16, 2, 4, dev), at.KvCache(4, 16, 2, 64, "int8", dev)
    step = table.step(i32([0, 0], dev), i32([3, 2], dev), 5)
    x = torch.zeros(5, 2, 64, device=dev)
    for k, v, q in ((x[:4], x, None), (x, x[:, :1], None), (x.double(), x.double(), None), (x, x.half(), None), (x, x, x.half()),
                    (x.cpu(), x, None), (x.transpose(1, 2).contiguous().transpose(1, 2), x, None), (x.view(5, -1), x, None),
                    (x, x, x[..., :32])):
        with pytest.raises(ValueError):
            cache.append(k, v, step, q=q)
    with pytest.raises(ValueError, match="pages"):
        at.KvCache(4, 32, 2, 64, "int8", dev).append(x, x, step)
    with pytest.raises(ValueError, match="slots"):
        cache.append(x, x, step.across(step))
    with pytest.raises(ValueError, match="channels"):
        cache.append(x, x, step, rotary=at.Rotary.from_theta(128, 9, device=dev))
    with pytest.raises(ValueError, match="angles"):
        cache.append(x, x, step, rotary=at.Rotary.from_theta(64, 9, device="cpu"))
    with pytest.raises(ValueError, match="batch"):
        table.step(i32([0] * 3, dev), i32([1] * 3, dev), 3)
    with pytest.raises(ValueError, match="new_lens"):
        table.step(i32([0], dev), i32([1, 1], dev), 3)
    with pytest.raises(ValueError, match="ctx_lens"):
        table.step(torch.zeros(2, device=dev), i32([1, 1], dev), 3)
    with pytest.raises(ValueError, match="negative"):
        table.step(i32([0], dev), i32([1], dev), -1)
    with pytest.raises(ValueError, match="which"):
        table.release(i32([0, 0], dev), i32([1], dev))
