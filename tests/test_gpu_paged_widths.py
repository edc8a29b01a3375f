"""Attention over the paged cache with tables whose rows are said to be as wide as an int64 can say."""
import pytest

from gpu_util import stream
from paged_ref import assert_near
from test_gpu_paged_attention import Case

pytestmark = pytest.mark.gpu


def test_a_table_of_any_width(torch_cuda, qctx):
    """One request's entries lie behind each other, however wide its row is said to be."""
    torch = torch_cuda
    c = Case(torch, qctx, [700], [3], 4, 2, 64, 16)
    for wide in (2 ** 31, 2 ** 59, 2 ** 60 + 3, 2 ** 62):
        a = c.call()
        a.max_pages = wide
        c.pg.attention(0, a, stream(torch))
        assert_near(torch, c.out, *c.want())
    c.free()
