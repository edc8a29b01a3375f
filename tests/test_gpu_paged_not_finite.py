"""Attention over the paged cache where what rows see is not finite: values of shares whose weight is
nothing, scores of minus infinity."""
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


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv,rows", [(4, 2, [1, 1, 1, 1, 1, 1]), (3, 3, [1, 5, 20, 1, 40, 2]), (8, 2, [3, 50, 300, 60, 129, 1])])
def test_scores_of_minus_infinity(torch_cuda, qctx, heads, kv, rows, d):
    """A row all of whose scores are minus infinity has no weights: NaN, as the formula gives, not the zeros of a
    row that sees nothing. Among finite scores they weigh nothing."""
    torch, inf = torch_cuda, float("inf")
    lengths = [1, 20, 200, 700, 4200, 33]
    c = Case(torch, qctx, lengths, rows, heads, kv, d, 32, seed=heads)
    c.q[..., 0] = 1.0
    for r, n in enumerate(lengths):
        c.k[c.slots(r, n), 0, 0] = -inf         # of key head 0 every score
    for r in (2, 4):
        n = lengths[r]
        c.k[c.slots(r, n)[n // 2:], 0, 0] = 0.5  # but here of the first half of the keys alone,
    c.k[c.slots(3, 700)[:650], kv - 1, 0] = -inf  # and of another head's all but the last 50
    c.put()
    for kw in (dict(), dict(causal=False), dict(window=30), dict(window=600, sinks=40)):
        c.check(**kw)
    # keys without a page are not seen: nothing is left of one request, minus infinity of another
    c.tables[0, :1] = -1
    c.tables[3, 3:] = -1
    c.check()
    c.free()
