"""The cache's objects hold addresses and sizes of the tensors they were made of: attributes that the library would
not see again are not set anew, and sizes that its fields do not hold are not cut."""
import pytest
import torch

from lightbulb_amd import attention as at


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.fixture
def no_device(monkeypatch):
    monkeypatch.setattr(at, "context", lambda device="cuda": 256)  # (nothing is launched)


def test_attributes_are_fixed(no_device):
    codes, scales = torch.zeros(3, 2, 16, 64, dtype=torch.int8), torch.zeros(3, 2)
    step = at.Step(i32(2, 3), i32(2), i32(3), torch.zeros(4, dtype=torch.int64), i32(4), page_size=16, num_tokens=4)
    made = [
        (at.PageTable.wrap(i32(2, 3), i32(4), i32(1), 16), ("tables", "free", "free_count", "page_size", "device")),
        (at.KvCache.wrap(codes, codes.transpose(2, 3).contiguous(), scales, scales.clone()),
         ("k", "v", "k_scales", "v_scales", "kind", "page_size", "kv_heads", "head_dim", "device")),
        (step, ("tables", "seq_lens", "cu_new", "slots", "positions", "page_size", "num_tokens", "max_len", "max_new", "granted", "crosses")),
        (step.across(step), ("tables", "seq_lens", "crosses")),
        (at.Rotary(torch.zeros(9, 32), torch.zeros(9, 32)), ("cos", "sin", "interleaved", "max_pos", "rot_dim")),
    ]
    for obj, names in made:
        for name in names:
            kept = getattr(obj, name)
            new = kept.clone() if isinstance(kept, torch.Tensor) else kept
            with pytest.raises(AttributeError, match=f"{type(obj).__name__}'s {name} is fixed"):
                setattr(obj, name, new)
            assert getattr(obj, name) is kept
    assert step.across(step).crosses and not step.crosses


@pytest.mark.parametrize("most", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 10 ** 18])
def test_bounds_beyond_32_bits_stay_bounds(most):
    # (their low 32 bits would be another bound, and keys beyond it unseen)
    step = at.Step(i32(2, 3), i32(2), i32(3), None, None, page_size=16, num_tokens=4, max_len=most, max_new=most)
    assert step._struct.max_len == step._struct.max_new == 2 ** 31 - 1
    assert (step.max_len, step.max_new) == (most, most)
    across = step.across(step)
    assert across._struct.max_len == across._struct.max_new == 2 ** 31 - 1
