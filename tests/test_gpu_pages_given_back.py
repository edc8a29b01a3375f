"""Pages given back that the ring of free pages has no room for, which lengths larger than a request's
or pages of several requests bring about: what is free stays as it is."""
import numpy as np
import pytest

import paged_ref
import qimm
from gpu_util import stream
from test_gpu_pages import Plan, a_case

pytestmark = pytest.mark.gpu


def plan(page, pages, tables, lengths, added, queue, state, max_rows):
    """paged_ref.plan, but of the pages given back only as many as the ring has room for go into it."""
    back = added < 0
    got = paged_ref.plan(page, pages, tables, lengths, np.where(back, 0, added), queue, state, max_rows)
    have = np.minimum(-(-np.maximum(lengths, 0) // page), tables.shape[1])
    given = np.concatenate([tables[r, :have[r]] for r in np.flatnonzero(back)])
    head, free = int(state[0]) % pages, min(max(int(state[1]), 0), pages)
    given = given[:pages - free]
    got["queue"][(head + free + np.arange(len(given))) % pages] = given
    got["lengths"][back] = 0
    got["state"][1] += len(given)
    return got


@pytest.mark.parametrize("free", [5, 4, 3, 99])
def test_a_full_ring(torch_cuda, qctx, free):
    """Two requests give back three pages each, of which 0, 1 and 2 have room; two others take the free ones."""
    torch = torch_cuda
    tables = np.array([[4, 4, 4], [-9, -9, -9], [4, 2, 1], [-9, -9, -9]], np.int32)
    case = (tables, np.array([33, 0, 48, 0], np.int32), np.array([-1, 17, -2, 1], np.int32), np.array([3, 1, 4, 0, 2], np.int32),
            np.array([2, free, 0, 0], np.int32), 20)
    p = Plan(torch, 16, *case)
    qctx.page_plan(p.call, stream(torch))
    p.check(plan(16, 5, *case))


@pytest.mark.parametrize("n,most_new", [(40, 20), (700, 3), (1500, 7), (9000, 1)])
def test_lengths_larger_than_the_requests(torch_cuda, qctx, n, most_new):
    """Three of four requests are given back, with lengths past their table's end: more pages come back than
    there is room for."""
    torch = torch_cuda
    case = list(a_case(np.random.default_rng(n), n, 16, 60, most_new))
    case[2][np.arange(n) % 4 != 1] = -1
    back = case[2] < 0
    case[1][back] = case[0].shape[1] * 16 + 5
    assert back.sum() * case[0].shape[1] > len(case[3]) - case[4][1]
    p = Plan(torch, 16, *case)
    qctx.page_plan(p.call, stream(torch))
    p.check(plan(16, len(case[3]), *case))
