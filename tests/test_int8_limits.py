"""The integer linears' and norms' stated limits, results laid over what a call reads, and tokens' attributes, without a device: the C
entry points check before any HIP call."""
import pytest
import torch

from lightbulb_amd import int8
from test_int8_refusals import D, FAR, INVALID, LIMIT, gate_up, linear, norm, residual_norm, weight

MOST = (1 << 22) - 1  # tokens


def far(n, i):
    """A weight of n channels whose memory is apart from all else."""
    return weight(n=n, d_codes=(16 + i) * FAR, d_scales=(32 + i) * FAR)


@pytest.mark.parametrize("m,ns", [(448, [1 << 24] * 4), (MOST, [8100]), (MOST, [1, 1, 1, 8188]), (1, [1 << 24] * 4), (511, [1 << 24] * 4), (2048, [(1 << 24) - 1])])
def test_sizes_inside_the_limit(lbq, m, ns):
    # tokens times channels below 2^35: what is refused is the output that is not there, which is looked at last
    assert m * sum(ns) < 1 << 35
    assert linear(lbq, [far(n, i) for i, n in enumerate(ns)], m=m, k=1, stride=1, codes=8 * FAR, scales=9 * FAR, ys=[None] * 8) == INVALID
    if len(set(ns)) == 1 and 2 * ns[0] * m < 1 << 35:
        assert gate_up(lbq, far(ns[0], 0), far(ns[0], 1), m=m, k=1, stride=1, codes=8 * FAR, scales=9 * FAR, y=None) == INVALID


@pytest.mark.parametrize("m,ns", [(512, [1 << 24] * 4), (MOST, [1 << 14]), (MOST, [8193]), (2048, [1 << 24]), (MOST, [1 << 24] * 4)])
def test_sizes_beyond_the_limit(lbq, m, ns):
    assert m * sum(ns) >= 1 << 35
    kw = dict(m=m, k=1, stride=1, codes=8 * FAR, scales=9 * FAR)
    assert linear(lbq, [far(n, i) for i, n in enumerate(ns)], ys=[None] * 8, **kw) == LIMIT and b"in one call" in lbq.lbq_last_error()
    if 2 * ns[0] * m >= 1 << 35:
        assert gate_up(lbq, far(ns[0], 0), far(ns[0], 1), y=None, **kw) == LIMIT


def test_outputs_over_what_is_read(lbq):
    # 5 tokens over 64 channels of 100 values: 1280 bytes of outputs
    w = weight(d_codes=16 * FAR, d_scales=17 * FAR, d_bias=18 * FAR)
    for y in (16 * FAR, 16 * FAR + 64 * 128 - 4, 16 * FAR - 1276, 17 * FAR + 252, 18 * FAR - 4):
        assert linear(lbq, [w], ys=[y]) == INVALID and b"weight" in lbq.lbq_last_error(), hex(y)
        assert linear(lbq, [weight(), w], ys=[3 * FAR, y]) == INVALID and linear(lbq, [weight(), w], ys=[y, 3 * FAR]) == INVALID
        assert gate_up(lbq, w, y=y) == INVALID and gate_up(lbq, None, w, y=y) == INVALID
    # the tokens' codes, where the call writes them
    for kw in (dict(codes=16 * FAR + 128), dict(scales=17 * FAR), dict(scales=18 * FAR - 16)):
        assert linear(lbq, [weight(), w], **kw) == INVALID and b"weight" in lbq.lbq_last_error()
        assert gate_up(lbq, w, **kw) == INVALID and gate_up(lbq, None, w, **kw) == INVALID
    # beside it, and codes that are read only (the null output is looked at last)
    for y in (16 * FAR + 64 * 128, 16 * FAR - 1280, 17 * FAR + 256):
        assert linear(lbq, [w, w], ys=[y, None]) == INVALID and b"null output" in lbq.lbq_last_error()
    assert linear(lbq, [w], x=None, codes=16 * FAR, scales=17 * FAR, ys=[None]) == INVALID and b"null output" in lbq.lbq_last_error()


def test_norms_results_over_their_vectors(lbq):
    n = norm(d_weight=16 * FAR, d_bias=17 * FAR)
    for kw in (dict(r=16 * FAR), dict(y=16 * FAR + 396), dict(r=17 * FAR - 1196), dict(y=17 * FAR), dict(y=None, codes=16 * FAR + 112, scales=5 * FAR),
               dict(y=None, codes=4 * FAR, scales=17 * FAR + 396)):
        assert residual_norm(lbq, pre=n, **kw) == INVALID and b"norm" in lbq.lbq_last_error(), kw
        assert residual_norm(lbq, post=n, **kw) == INVALID and b"norm" in lbq.lbq_last_error(), kw


def test_tokens_keep_what_they_were_made_with():
    # a scale for every row of codes, as the products read them: other tensors cannot take their places
    t = int8.Int8Tokens(torch.ones(2, 128, dtype=torch.int8), torch.full((2,), 0.5), torch.Size((2, 100)), torch.bfloat16, torch.device("cpu"))
    assert t.shape == (2, 100) and t.dtype == torch.bfloat16 and t.device == torch.device("cpu") and t.codes.shape == (2, 100)
    for name, value in dict(scales=torch.ones(1), codes=torch.ones(1, 100, dtype=torch.int8), shape=torch.Size((4, 100)), dtype=torch.float32,
                            device=torch.device("meta")).items():
        with pytest.raises(AttributeError):
            setattr(t, name, value)
    t.scales.mul_(2)
    assert torch.equal(t.dequantize(), torch.ones(2, 100)) and "(2, 100)" in repr(t)
