"""Attention over the paged cache where what rows see is not finite: values of shares whose weight is
nothing."""
import numpy as np
import pytest

from test_gpu_paged_attention import Case

pytestmark = pytest.mark.gpu


def steep(c, length, dims):
    """Keys whose scores rise from -64 (log2 -92) before token `length` / 3 to 64 in the last third: the first
    weigh 2^-184 of the last, nothing in 32 bits."""
    c.q.fill_(1.0)
    slots = c.slots(0, length)
    size = 64 / np.sqrt(dims)
    for i, x in enumerate((-size, 0.0, size)):
        c.k[slots[i * length // 3:(i + 1) * length // 3]] = x


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("length,rows,heads", [(4200, 1, 4), (70001, 1, 4), (4200, 40, 2), (16000, 130, 1), (300, 1, 4), (300, 40, 2)])
def test_a_value_that_weighs_nothing_counts_where_it_is_seen(torch_cuda, qctx, length, rows, heads, d):
    """NaN at an early token: its share of the keys has a factor of 0 in the join, the output is NaN all the same;
    in a window without it, it does not count."""
    c = Case(torch_cuda, qctx, [length], [rows], heads, 1, d, 64)
    steep(c, length, d)
    slots = c.slots(0, length)
    c.v[slots[5], 0, 3] = c.v[slots[length - 1], 0, 7] = float("nan")
    c.put()
    for kw in (dict(), dict(causal=False), dict(window=length - 100), dict(window=length - 100, sinks=9)):
        c.check(**kw)
    c.free()
