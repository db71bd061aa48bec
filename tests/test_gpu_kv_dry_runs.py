"""Steps that are worked out without taking their pages: what follows them finds tables, free pages and cache as if
they had not been."""
import random

import pytest
import torch

from lightbulb_amd import attention as at
from test_gpu_kv_step import i32

pytestmark = pytest.mark.gpu


def test_nothing_is_appended_to_a_dry_run(dev):
    table, cache = at.PageTable(8, 16, 2, 4, dev), at.KvCache(8, 16, 1, 64, "int8", dev)
    lens, new, x = i32([0, 0], dev), i32([20, 3], dev), torch.randn(23, 1, 64, device=dev)
    dry = table.step(lens, new, 23, commit=False)
    assert not dry.taken and dry.granted.tolist() == [1, 1]
    with pytest.raises(ValueError, match="took no pages"):
        cache.append(x, x, dry)
    assert (cache.k == 0).all() and (cache.k_scales == 0).all()
    step = table.step(lens, new, 23)  # the same one, taken
    assert step.taken and torch.equal(step.slots, dry.slots)
    cache.append(x, x, step)
    assert (cache.k_scales[table.tables[0, :2].long()] > 0).all()


def test_other_steps_after_dry_runs(dev):
    # a scheduler that asks for many steps and takes another: each page is held by one sequence or free, and every
    # taken step and release is what a table without dry runs gives
    rng = random.Random(5)
    page, rows, blocks, pages = 16, 6, 6, 24
    asked, plain = at.PageTable(pages, page, rows, blocks, dev), at.PageTable(pages, page, rows, blocks, dev)
    lens = [0] * rows
    for turn in range(40):
        for _ in range(rng.randint(1, 3)):
            new = [rng.choice((0, 1, 20, 50)) for _ in range(rows)]
            asked.step(i32(lens, dev), i32(new, dev), sum(new), commit=False)
        new = [rng.choice((0, 1, 1, 20)) for _ in range(rows)]
        a, b = (p.step(i32(lens, dev), i32(new, dev), sum(new)) for p in (asked, plain))
        for name in ("seq_lens", "cu_new", "granted", "slots", "positions"):
            assert torch.equal(getattr(a, name), getattr(b, name)), (turn, name)
        lens = [c + n if g else c for c, n, g in zip(lens, new, a.granted.tolist())]
        done = [int(n > 60 or rng.random() < 0.1) for n in lens]
        for p in (asked, plain):
            p.release(i32(lens, dev), i32(done, dev))
        lens = [0 if d else n for n, d in zip(lens, done)]
        held = [asked.tables[i, j].item() for i in range(rows) for j in range(-(-lens[i] // page))]
        free = asked.free[: asked.free_count.item()]
        assert torch.equal(free, plain.free[: plain.free_count.item()])
        assert sorted(held + free.tolist()) == list(range(pages)), turn
