"""What the cache operators refuse, without a device: the C entry points check before any HIP call,
and the Python ones before they reach the library."""
import ctypes

import pytest
import torch

from lightbulb_amd import _lib
from lightbulb_amd import attention as at

D = 256  # an address that is aligned and never read


def cache(**kw):
    f = dict(d_k=D, d_v=D, d_k_scales=D, d_v_scales=D, num_pages=4, kind=0, page_size=16, kv_heads=2, head_dim=64)
    f.update(kw)
    return _lib.KvCacheStruct(**f)


def step(**kw):
    f = dict(d_tables=D, table_stride=8, d_seq_lens=D, d_cu_new=D, d_slots=D, d_positions=D, num_tokens=3, batch=2, max_blocks=8,
             max_len=0, max_new=0)
    f.update(kw)
    return _lib.KvStepStruct(**f)


def attend(lbq, c, s, dtype=0, q=D, ts=128, hs=64, heads=2, causal=1, window=0, out=1 << 20, ws=None, ctx=D):
    return lbq.lbq_kv_attention(ctx, c, s, dtype, q, ts, hs, heads, 1.0, causal, window, out, ws, 0, None)


def append(lbq, c, s, dtype=0, k=D, v=D, q=None, heads=2, cos=D, sin=D, max_pos=10, rot=64, q_out=1 << 20, strides=(128, 64)):
    return lbq.lbq_kv_append(D, c, s, dtype, k, *strides, v, *strides, q, *strides, heads, cos, sin, max_pos, rot, 0, q_out, None)


def build(lbq, **kw):
    f = dict(ctx=D, ctx_lens=D, new_lens=D, batch=2, tables=D, stride=8, blocks=8, page=16, free=D, pages=4, count=D, count_out=D + 4,
             ticket=D, tokens=3, seq=D, cu=D, granted=D, slots=D, positions=D, stream=None)
    f.update(kw)
    return lbq.lbq_kv_step_build(*f.values())


INVALID, TYPE, SHAPE, LIMIT = -1, -2, -3, -6


@pytest.mark.parametrize("kw,status", [
    (dict(d_k=None), INVALID), (dict(d_v_scales=None), INVALID), (dict(d_k=D + 8), INVALID), (dict(d_k_scales=D + 2), INVALID),
    (dict(kind=2), TYPE), (dict(page_size=8), SHAPE), (dict(page_size=48), SHAPE), (dict(page_size=256), SHAPE),
    (dict(head_dim=80), SHAPE), (dict(head_dim=512), SHAPE), (dict(kv_heads=0), SHAPE), (dict(num_pages=0), SHAPE),
    (dict(kv_heads=2000), LIMIT), (dict(num_pages=1 << 40), LIMIT)])
def test_cache_is_checked(lbq, kw, status):
    heads = 2000 if kw.get("kv_heads") == 2000 else 2
    assert attend(lbq, cache(**kw), step(), heads=heads) == status
    assert append(lbq, cache(**kw), step()) == status
    n = ctypes.c_size_t()
    assert lbq.lbq_kv_attention_workspace(D, cache(**kw), step(), heads, n) == status
    assert lbq.lbq_last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(d_tables=None), INVALID), (dict(d_seq_lens=None), INVALID), (dict(d_cu_new=D + 1), INVALID), (dict(d_tables=D + 2), INVALID),
    (dict(batch=0), SHAPE), (dict(batch=70000), LIMIT), (dict(max_blocks=0), SHAPE), (dict(table_stride=7), SHAPE),
    (dict(num_tokens=-1), SHAPE), (dict(max_len=-1), SHAPE), (dict(max_new=-1), SHAPE), (dict(num_tokens=1 << 40), LIMIT)])
def test_step_is_checked(lbq, kw, status):
    assert attend(lbq, cache(), step(**kw)) == status
    assert append(lbq, cache(), step(**kw)) == status


def test_attention_arguments(lbq):
    assert attend(lbq, None, step()) == INVALID and attend(lbq, cache(), None) == INVALID
    assert attend(lbq, cache(), step(), ctx=None) == INVALID
    assert attend(lbq, cache(), step(), dtype=8) == TYPE
    assert attend(lbq, cache(), step(), q=None) == INVALID and attend(lbq, cache(), step(), out=None) == INVALID
    assert attend(lbq, cache(), step(), q=D + 2) == INVALID and attend(lbq, cache(), step(), out=(1 << 20) + 2) == INVALID
    assert attend(lbq, cache(), step(), ts=-1) == SHAPE
    assert attend(lbq, cache(), step(), heads=3) == SHAPE and attend(lbq, cache(), step(), heads=0) == SHAPE
    assert attend(lbq, cache(), step(), heads=2048) == LIMIT
    assert attend(lbq, cache(), step(), window=-1) == SHAPE and attend(lbq, cache(), step(), causal=0, window=5) == SHAPE
    assert attend(lbq, cache(), step(), out=D + 4 * (2 * 128 + 64)) == INVALID  # the last row of q
    assert attend(lbq, cache(), step(), ws=D + 8) == INVALID
    assert attend(lbq, cache(), step(max_blocks=1 << 30, table_stride=1 << 30)) == LIMIT
    assert attend(lbq, cache(kv_heads=1024), step(batch=65536), heads=1024) == LIMIT
    assert attend(lbq, cache(), step(num_tokens=1 << 24), heads=1024) == LIMIT
    assert attend(lbq, cache(), step(num_tokens=0), q=None, out=None) == 0  # nothing to do


def test_append_arguments(lbq):
    assert append(lbq, cache(), step(d_slots=None)) == INVALID and append(lbq, cache(), step(d_positions=None)) == INVALID
    assert append(lbq, cache(), step(d_slots=D + 4)) == INVALID
    assert append(lbq, cache(), step(), dtype=12) == TYPE
    assert append(lbq, cache(), step(), k=None) == INVALID and append(lbq, cache(), step(), v=D + 1) == INVALID
    assert append(lbq, cache(), step(), rot=66) == SHAPE and append(lbq, cache(), step(), rot=-2) == SHAPE
    assert append(lbq, cache(), step(), rot=33) == SHAPE
    assert append(lbq, cache(), step(), cos=None) == INVALID and append(lbq, cache(), step(), sin=D + 2) == INVALID
    assert append(lbq, cache(), step(), max_pos=0) == SHAPE
    assert append(lbq, cache(), step(), q=1 << 22, q_out=None) == INVALID
    assert append(lbq, cache(), step(), q=1 << 22, heads=0) == SHAPE and append(lbq, cache(), step(), q=1 << 22, heads=2000) == LIMIT
    for other in ("q", "k", "v"):
        assert append(lbq, cache(), step(), **{"q": 1 << 22, other: (1 << 20) + 64}) == INVALID
    assert append(lbq, cache(), step(), strides=(128, -1)) == SHAPE
    assert append(lbq, cache(kv_heads=1024), step(batch=65536)) == LIMIT
    assert append(lbq, cache(), step(num_tokens=0, d_slots=None, d_positions=None), k=None, v=None) == 0


def test_step_build_arguments(lbq):
    for name in ("ctx", "ctx_lens", "new_lens", "free", "count", "count_out", "seq", "cu", "granted", "slots", "positions", "tables"):
        assert build(lbq, **{name: None}) == INVALID, name
    assert build(lbq, count_out=D, ticket=None) == INVALID
    assert build(lbq, slots=D + 4) == INVALID and build(lbq, new_lens=D + 1) == INVALID
    assert build(lbq, batch=0) == SHAPE and build(lbq, batch=1 << 20) == LIMIT
    assert build(lbq, blocks=9) == SHAPE and build(lbq, page=24) == SHAPE and build(lbq, pages=0) == SHAPE
    assert build(lbq, tokens=-1) == SHAPE and build(lbq, tokens=1 << 40) == LIMIT and build(lbq, pages=1 << 40) == LIMIT


def test_release_arguments(lbq):
    def release(**kw):
        f = dict(ctx=D, lens=D, which=D, batch=2, tables=D, stride=8, blocks=8, page=16, free=D, pages=4, count=D, stream=None)
        f.update(kw)
        return lbq.lbq_kv_release(*f.values())
    for name in ("ctx", "lens", "which", "tables", "free", "count"):
        assert release(**{name: None}) == INVALID, name
    assert release(lens=D + 2) == INVALID and release(batch=0) == SHAPE and release(page=0) == SHAPE
    assert release(pages=0) == SHAPE and release(pages=1 << 40) == LIMIT and release(blocks=9) == SHAPE


def _step(**kw):
    f = dict(tables=torch.zeros(2, 3, dtype=torch.int32), seq_lens=torch.zeros(2, dtype=torch.int32),
             cu_new=torch.zeros(3, dtype=torch.int32), slots=None, positions=None, page_size=16, num_tokens=4)
    f.update(kw)
    return at.Step(**f)


def test_python_step_is_checked():
    _step()
    with pytest.raises(ValueError, match="block tables"):
        _step(tables=torch.zeros(2, 3))
    with pytest.raises(ValueError, match="block tables"):
        _step(tables=torch.zeros(3, 2, dtype=torch.int32).t())
    with pytest.raises(ValueError, match="seq_lens"):
        _step(seq_lens=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="cu_new"):
        _step(cu_new=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="slots"):
        _step(slots=torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="positions"):
        _step(positions=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="negative"):
        _step(max_new=-1)
    with pytest.raises(ValueError, match="page_size"):
        _step(page_size=20)
    with pytest.raises(ValueError, match="across"):
        _step().across(_step(tables=torch.zeros(1, 3, dtype=torch.int32), seq_lens=torch.zeros(1, dtype=torch.int32),
                             cu_new=torch.zeros(2, dtype=torch.int32)))


def test_python_cache_and_angles_are_checked():
    k = torch.zeros(3, 2, 16, 64, dtype=torch.int8)
    s = torch.zeros(3, 2)
    with pytest.raises(ValueError, match="GPU"):
        at.KvCache.wrap(k, k.transpose(2, 3).contiguous(), s, s)  # there is no CPU form
    with pytest.raises(ValueError, match="codes"):
        at.KvCache.wrap(k.float(), k, s, s)
    with pytest.raises(ValueError, match="among"):
        at.KvCache.wrap(k[:, :, :8], k, s, s)
    with pytest.raises(ValueError, match="is not"):
        at.KvCache.wrap(k, k, s, s)
    with pytest.raises(ValueError, match="k_scales"):
        at.KvCache.wrap(k, k.transpose(2, 3).contiguous(), s[:2], s)
    with pytest.raises(ValueError, match="kind"):
        at.KvCache(3, 16, 2, 64, kind="int4", device="cpu")
    with pytest.raises(ValueError, match="angles"):
        at.Rotary(torch.zeros(4, 3), torch.zeros(4, 2))
    with pytest.raises(ValueError, match="cos"):
        at.Rotary(torch.zeros(4, 3).double(), torch.zeros(4, 3))
    with pytest.raises(ValueError, match="GPU"):
        at.PageTable(4, 16, 2, 3, device="cpu")
    with pytest.raises(ValueError, match="needs"):
        at.PageTable(0, 16, 2, 3, device="cpu")
    with pytest.raises(ValueError, match="query heads"):
        at.Attention(None, None, None, None, 5, 2, 64)
