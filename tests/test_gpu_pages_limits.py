"""Steps of the page tables at the limits of their numbers and arrays: tokens past 31 bits, scratch anywhere."""
import numpy as np
import pytest

import paged_ref
import qimm
from gpu_util import host, stream
from test_gpu_pages import Plan, a_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_rows", [40, 3000])
def test_a_table_wider_than_a_length_can_be(torch_cuda, qctx, max_rows):
    """Tables of 2^31 tokens and more: a request that would have more than 2^31 - 1 is refused, one that
    comes up to it is served; both forms of the step."""
    torch, page, pages, most = torch_cuda, 512, 8, 2 ** 31 - 1
    width = 2 ** 31 // page + 3
    lengths = np.array([most - 5, most - 5, most, most - 1, 0], np.int32)
    added = np.array([3, 10, 1, 1, 2], np.int32)
    tables = np.full((5, width), -7, np.int32)
    tables[:, width - 4] = [5, 6, 1, 2, -7]  # the page of tokens 2^31 - 512 .. 2^31 - 1
    queue = np.array([3, 4, 0, 7, -1, -1, -1, -1], np.int32)
    p = Plan(torch, page, tables, lengths, added, queue, np.array([0, 4, 0, 0], np.int32), max_rows)
    qctx.page_plan(p.call, stream(torch))
    first = np.arange(most - 5, most - 2)
    slots, positions = np.full(max_rows, -1), np.zeros(max_rows, int)
    slots[:3], positions[:3] = 5 * page + first % page, first
    slots[14], positions[14] = 2 * page + page - 2, most - 1
    slots[15:17], positions[15:17] = 3 * page + np.arange(2), np.arange(2)
    tables[4, 0] = 3
    p.check(dict(tables=tables, lengths=np.array([most - 2, most - 5, most, most, 2]), queue=queue, state=np.array([1, 3, 17, 2]),
                 starts=np.array([0, 3, 13, 14, 15, 17]), slots=slots, positions=positions))


@pytest.mark.parametrize("at", [1, 2, 3])
@pytest.mark.parametrize("n", [60, 1025, 5000])
def test_scratch_on_any_int32(torch_cuda, qctx, n, at):
    """work begins 4, 8 and 12 bytes behind a multiple of 16; what lies around it stays."""
    torch = torch_cuda
    case = a_case(np.random.default_rng(n), n, 16, 60, 9)
    p = Plan(torch, 16, *case)
    size = qimm.page_plan_work(n)
    room = torch.full((size + 8,), -99, dtype=torch.int32, device="cuda")
    p.call.work = room[at:].data_ptr()
    qctx.page_plan(p.call, stream(torch))
    p.check(paged_ref.plan(16, len(case[3]), *case))
    assert (host(room)[:at] == -99).all() and (host(room)[at + size:] == -99).all()
