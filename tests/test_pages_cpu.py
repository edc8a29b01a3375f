"""The paged cache's plain forms on known steps, and its calls' refusals without a device."""
import ctypes as C

import numpy as np
import pytest

import paged_ref
import qimm


def i32(*x):
    return np.array(x, np.int32)


def test_a_known_step():
    """Pages of 16 tokens: 15 + 2 tokens take a page, 16 + 16 one, a request gives two back, 0 + 0 nothing."""
    tables = np.array([[5, 9, 9, 9], [2, 9, 9, 9], [7, 1, 9, 9], [9, 9, 9, 9]], np.int32)
    got = paged_ref.plan(16, 8, tables, i32(15, 16, 20, 0), i32(2, 16, -1, 0), i32(0, 3, -9, -9, -9, -9, 4, 6), i32(6, 4, 0, 0), 20)
    assert got["starts"].tolist() == [0, 2, 18, 18, 18] and got["lengths"].tolist() == [17, 32, 0, 0]
    assert got["tables"][0].tolist() == [5, 4, 9, 9] and got["tables"][1].tolist() == [2, 6, 9, 9]
    assert got["slots"].tolist() == [95, 64] + list(range(96, 112)) + [-1, -1]
    assert got["positions"].tolist() == [15, 16] + list(range(16, 32)) + [0, 0]
    assert got["queue"].tolist() == [0, 3, 7, 1, -9, -9, 4, 6] and got["state"].tolist() == [0, 4, 18, 0]


def test_refusals_of_a_step():
    """The second request asks for more than is free and the third after it; the fourth needs no page;
    the fifth's table is full."""
    tables = np.zeros((5, 2), np.int32)
    got = paged_ref.plan(16, 4, tables, i32(16, 0, 0, 3, 32), i32(1, 32, 1, 5, 1), i32(1, 2, 3, -1), i32(0, 2, 0, 0), 99)
    assert got["lengths"].tolist() == [17, 0, 0, 8, 32] and got["state"].tolist() == [1, 1, 40, 3]
    assert (got["slots"][1:34] == -1).all() and got["slots"][34:39].tolist() == [3, 4, 5, 6, 7]


def test_attention_over_known_pages():
    torch = pytest.importorskip("torch")
    k = torch.zeros(64, 1, 4)
    v = torch.arange(64.0)[:, None, None].expand(64, 1, 4)
    tables = torch.tensor([[3, 1]])
    out, _ = paged_ref.attention(torch, torch.ones(2, 1, 4), k, v, tables, [18], [0, 2], 16, True)
    # keys of no direction: the mean of the slots 48 .. 63 and 16 (, 17)
    assert out[0, 0, 0] == pytest.approx((sum(range(48, 64)) + 16) / 17) and out[1, 0, 0] == pytest.approx((sum(range(48, 64)) + 33) / 18)
    out, _ = paged_ref.attention(torch, torch.ones(2, 1, 4), k, v, tables, [18], [0, 2], 16, True, 2, 1)
    assert out[1, 0, 0] == pytest.approx((48 + 16 + 17) / 3)
    out, _ = paged_ref.attention(torch, torch.ones(2, 1, 4), k, v, tables, [1], [0, 2], 16, True)
    assert not out[0].any() and out[1, 0, 0] == 48


def test_null_arguments():
    lib = qimm.load()
    h = C.c_void_p()
    assert lib.qimm_page_plan(None, None, None) == 1
    assert lib.qimm_pages_create(None, 1, 1, 16, 1, 128, C.byref(h)) == 1
    assert lib.qimm_pages_destroy(None) == 1
    assert lib.qimm_pages_device_bytes(None) == -1
    assert lib.qimm_pages_store(None, 0, None, None, 0, 0, 0, 0, 0, 0, None, None) == 1
    assert lib.qimm_pages_load(None, 0, None, None, 0, None, None) == 1
    assert lib.qimm_attention_paged(None, 0, None, None) == 1


def test_work_of_a_plan():
    assert qimm.page_plan_work(1) >= 4 and qimm.page_plan_work(65536) >= 4 * 65536
    for n in (0, -1, 65537):
        assert qimm.load().qimm_page_plan_work(n) == -1
        with pytest.raises(qimm.QimmError):
            qimm.page_plan_work(n)
