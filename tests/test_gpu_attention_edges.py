"""Attention over the 8-bit cache where calls are allowed and seldom made: bounds that do not hold while the
keys are cut into parts."""
import ctypes

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
