"""A cache that the card has no room for is refused, and the calls after it are as ever."""
import numpy as np
import pytest

import paged_ref
import qimm
from gpu_util import stream
from test_gpu_paged_attention import Case
from test_gpu_pages import Plan, a_case

pytestmark = pytest.mark.gpu


def refused(ctx):
    with pytest.raises(qimm.QimmError) as e:
        ctx.pages_create(16, 2 ** 20, 64, 8, 128)  # 4 TiB
    assert "QIMM_ERR_OOM" in str(e.value)


def test_calls_after_a_cache_too_large(torch_cuda, qctx):
    """The allocation's error is not reported again by the next launch, the library's or another's."""
    torch = torch_cuda
    case = a_case(np.random.default_rng(0), 9, 16, 60, 9)
    p = Plan(torch, 16, *case)
    c = Case(torch, qctx, [40, 700], [3, 1], 4, 2, 64, 16)
    refused(qctx)
    qctx.page_plan(p.call, stream(torch))
    p.check(paged_ref.plan(16, len(case[3]), *case))
    refused(qctx)
    c.check()
    refused(qctx)
    c.put()
    refused(qctx)
    assert float(torch.ones(5, device="cuda").sum()) == 5
    pg = qctx.pages_create(1, 4, 16, 2, 64)
    pg.free()
    c.free()
