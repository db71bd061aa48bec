"""Block tables, slot maps and positions from request lengths against the definition, one sequence at a
time (whole numbers: equal), and releases."""
import random

import pytest
import torch

import kv_ref
from lightbulb_amd import attention as at

pytestmark = pytest.mark.gpu


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def pool(dev, ctx, page, blocks, spare, seed=1, rows=None):
    """A PageTable whose sequences hold ctx tokens in random pages, and `spare` free pages."""
    held = [max(0, -(-c // page)) for c in ctx]
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(held) + max(spare, 1), generator=g).to(torch.int32)
    tables = torch.full((rows or len(ctx), blocks), -1, dtype=torch.int32)
    at0 = 0
    for b, n in enumerate(held):
        n = min(n, blocks)
        tables[b, :n] = order[at0: at0 + n]
        at0 += n
    free = order.roll(-sum(held)).contiguous()
    return at.PageTable.wrap(tables.to(dev), free.to(dev), i32([spare], dev), page), tables, free


def check(p, tables, free, ctx, new, page, tokens, spare, dev, commit=True):
    s = p.step(i32(ctx, dev), i32(new, dev), tokens, commit=commit)
    n = len(ctx)
    want = kv_ref.step(ctx, new, tables[:n], free, spare, page, tokens)
    assert torch.equal(s.tables.cpu(), want[0])
    assert s.seq_lens.tolist() == want[1]
    assert s.cu_new.tolist() == want[2]
    assert s.granted.tolist() == want[3]
    assert s.slots.tolist() == want[4]
    assert s.positions.tolist() == want[5]
    assert s.free_count.item() == want[6]
    assert p.free_count.item() == (want[6] if commit else spare) and p._ticket.item() == 0
    return s, want


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("batch,most_ctx,most_new,idle", [
    (1, 0, 1, 0), (1, 100, 1, 0), (1, 0, 5000, 0), (3, 130, 40, 0), (16, 1000, 1, 0.5), (16, 300, 700, 0.3),
    (255, 50, 3, 0.2), (1024, 40, 2, 0.1), (1025, 40, 2, 0), (2500, 70, 20, 0.4)])
def test_step(dev, page, batch, most_ctx, most_new, idle):
    rng = random.Random(batch * 7 + page)
    ctx = [rng.randint(0, most_ctx) for _ in range(batch)]
    new = [0 if rng.random() < idle else rng.randint(1, most_new) for _ in range(batch)]
    blocks = max(1, max(-(-(c + n) // page) for c, n in zip(ctx, new)))
    p, tables, free = pool(dev, ctx, page, blocks, 9000)
    check(p, tables, free, ctx, new, page, sum(new), 9000, dev, commit=False)
    p, tables, free = pool(dev, ctx, page, blocks, 9000)
    check(p, tables, free, ctx, new, page, sum(new) + 77, 9000, dev)


def test_no_tokens(dev):
    p, tables, free = pool(dev, [5, 0], 16, 2, 3)
    check(p, tables, free, [5, 0], [0, 0], 16, 0, 3, dev)


@pytest.mark.parametrize("spare", [0, 1, 2, 5, 6, 100])
def test_pages_run_out(dev, spare):
    # needs are 1, 0, 2, 3, 0, 1: whoever asks first is served, and one that needs none always is
    ctx, new = [16, 3, 0, 40, 7, 0], [1, 5, 30, 50, 1, 16]
    p, tables, free = pool(dev, ctx, 16, 8, spare)
    s, want = check(p, tables, free, ctx, new, 16, sum(new) + 3, spare, dev)
    assert want[3][1] == want[3][4] == 1


def test_lengths_that_do_not_fit(dev):
    # a negative length, a table row that is too short, rows behind num_tokens, and lengths
    # whose sums pass 32 bits
    top = 2 ** 31 - 1
    for ctx, new, tokens in (([3, -1, 4], [2, 3, 1], 5), ([3, 5, 4], [2, -3, 1], 5), ([3, 30, 4], [2, 40, 1], 60),
                             ([3, 5, 4, 0], [2, 9, 1, 0], 6), ([top, 0, 4], [top, 1, 1], 10), ([0, 0, 0, 4], [top, top, top, 1], 10),
                             ([16, 16], [17, 1], 17)):
        p, tables, free = pool(dev, [min(c, 64) for c in ctx], 16, 4, 7)
        check(p, tables, free, ctx, new, 16, tokens, 7, dev)


def test_entry_that_is_no_page(dev):
    # a sequence's partly filled page is missing from its table: no slot there
    p, tables, free = pool(dev, [20, 20], 16, 4, 5)
    p.tables[0, 1] = -1
    s = p.step(i32([20, 20], dev), i32([2, 2], dev), 4)
    assert s.slots[:2].tolist() == [-1, -1] and s.positions[:2].tolist() == [-1, -1]
    assert s.slots[2:].tolist() == [int(tables[1, 1]) * 16 + 4, int(tables[1, 1]) * 16 + 5]


def test_fewer_sequences_than_rows_and_strided_tables(dev):
    big = torch.full((5, 12), -1, dtype=torch.int32, device=dev)
    p = at.PageTable.wrap(big[:, 2:9], torch.arange(20, dtype=torch.int32, device=dev), i32([20], dev), 16)
    s = p.step(i32([0, 0, 0], dev), i32([17, 1, 33], dev), 51)
    assert p.tables[:3, :3].tolist() == [[19, 18, -1], [17, -1, -1], [16, 15, 14]]
    assert (big[:, :2] == -1).all() and (big[:, 9:] == -1).all() and (big[3:] == -1).all()
    assert s.free_count.item() == 14


def test_steps_and_releases_in_turn(dev):
    # a serving loop: steps are taken, finished sequences give their pages back, and every page
    # is held once or free once throughout
    rng = random.Random(3)
    page, rows, blocks, pages = 16, 7, 6, 30
    p = at.PageTable(pages, page, rows, blocks, dev)
    lens = [0] * rows
    for turn in range(40):
        new = [rng.choice((0, 1, 1, 1, 20)) for _ in range(rows)]
        s = p.step(i32(lens, dev), i32(new, dev), sum(new))
        lens = [c + n if g else c for c, n, g in zip(lens, new, s.granted.tolist())]
        done = [int(n > 60 or rng.random() < 0.1) for n in lens]
        p.release(i32(lens, dev), i32(done, dev))
        lens = [0 if d else n for n, d in zip(lens, done)]
        held = p.tables[p.tables >= 0].tolist()
        free = p.free[: p.free_count.item()].tolist()
        assert sorted(held + free) == list(range(pages)), turn
        assert [int((p.tables[b] >= 0).sum()) for b in range(rows)] == [-(-n // page) for n in lens]
    p.release(i32(lens, dev), i32([1] * rows, dev))
    p.release(i32(lens, dev), i32([1] * rows, dev))  # twice: nothing is freed again
    assert p.free_count.item() == pages and sorted(p.free.tolist()) == list(range(pages)) and (p.tables == -1).all()


def test_release_of_many(dev):
    # more than a workgroup's rows and blocks, in order
    rows, blocks, page = 1500, 3, 16
    g = torch.Generator().manual_seed(2)
    tables = torch.randperm(rows * blocks, generator=g).to(torch.int32).view(rows, blocks)
    lens = [(i * 7) % 49 for i in range(rows)]
    which = [int(i % 3 != 0) for i in range(rows)]
    p = at.PageTable.wrap(tables.to(dev), torch.full((rows * blocks,), -5, dtype=torch.int32, device=dev), i32([0], dev), page)
    p.release(i32(lens, dev), i32(which, dev))
    want = [int(tables[b, j]) for b in range(rows) if which[b] for j in range(-(-lens[b] // page))]
    assert p.free_count.item() == len(want) and p.free[: len(want)].tolist() == want
    left = p.tables.cpu()
    for b in range(rows):
        n = -(-lens[b] // page) if which[b] else 0
        assert left[b].tolist() == [-1] * n + tables[b, n:].tolist()
    one = at.PageTable.wrap(torch.arange(5000, dtype=torch.int32, device=dev)[None], torch.full((5000,), -1, dtype=torch.int32, device=dev),
                            i32([0], dev), page)
    one.release(i32([5000 * 16], dev), i32([1], dev))
    assert one.free.tolist() == list(range(5000)) and one.free_count.item() == 5000


def test_release_of_long_and_empty_sequences(dev):
    # rows of more entries than a workgroup has threads, rows without any between them, entries that are no pages
    rows, blocks, page = 1030, 1500, 16
    lens = [(0, 0, 1500 * 16, 1, 0, 24000 - 1, 0, 16 * 1100)[i % 8] if i < 24 or i > 1020 else 0 for i in range(rows)]
    which = [int(i % 5 != 2) for i in range(rows)]
    tables = torch.arange(rows * blocks, dtype=torch.int32).view(rows, blocks)
    tables[:, 7] = -1
    tables[:, 9] = rows * blocks
    p = at.PageTable.wrap(tables.to(dev), torch.full((rows * blocks,), -5, dtype=torch.int32, device=dev), i32([3], dev), page)
    p.release(i32(lens, dev), i32(which, dev))
    want = torch.cat([tables[b, : -(-lens[b] // page)] for b in range(rows) if which[b]])
    want = want[(want >= 0) & (want < rows * blocks)]
    assert p.free_count.item() == 3 + len(want)
    assert torch.equal(p.free[3: 3 + len(want)].cpu(), want) and (p.free[3 + len(want):] == -5).all() and (p.free[:3] == -5).all()
    left = tables.clone()
    for b in range(rows):
        if which[b]:
            left[b, : -(-lens[b] // page)] = -1
    assert torch.equal(p.tables.cpu(), left)


def test_replays_take_pages_each_time(dev):
    p = at.PageTable(64, 16, 4, 16, dev)
    lens, new = i32([0, 0, 0, 0], dev), i32([16, 1, 0, 33], dev)
    p.step(lens, i32([0] * 4, dev), 2500)  # (the library is loaded and warm)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s = p.step(lens, new, 2500)  # several workgroups
        lens.add_(new)
    tables, free, count, held = torch.full((4, 16), -1, dtype=torch.int32), torch.arange(63, -1, -1), 64, [0] * 4
    for _ in range(4):
        g.replay()
        torch.cuda.synchronize()
        want = kv_ref.step(held, [16, 1, 0, 33], tables, free, count, 16, 2500)
        tables, count = want[0], want[6]
        held = [h + n for h, n in zip(held, [16, 1, 0, 33])]
        assert torch.equal(p.tables.cpu(), tables) and s.slots.tolist() == want[4] and s.positions.tolist() == want[5]
        assert s.seq_lens.tolist() == want[1] and p.free_count.item() == count and lens.tolist() == held
