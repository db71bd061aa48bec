"""The integer linears' and norms' stated limits, and results laid over what a call reads, without a device: the C entry points check
before any HIP call."""
import pytest

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
