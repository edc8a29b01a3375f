"""The attention over a 4-bit cache where a head's keys are split into shares that a second launch
joins: padded batches whose hidden keys fill whole shares, rows that see nothing, numbers that are
none, a key that takes nearly all, and the most shares there are. The bar is test_gpu_kv4's; the
join adds f32 roundings."""
import numpy as np
import pytest

import kv4_ref
import qimm
from gpu_util import dev, host, stream
from test_gpu_kv4 import assert_near, attn_case, bf16, stored

pytestmark = pytest.mark.gpu


def shares(torch, b, h, sq, p, so):
    """How many the call is split into: two workgroups per CU, a tile for every wave, at most 64."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    items, wgs = -(-p // 128) + -(-so // 64), b * h * -(-sq // 16)
    return 1 if items <= 16 else max(1, min(2 * cus // wgs, (items + 3) // 4, 64))


@pytest.mark.parametrize("fill", [None, float("nan"), float("inf"), -3.0e38])
@pytest.mark.parametrize("h,sq,p,so", [(1, 3, 5000, 0), (2, 17, 4300, 65), (1, 1, 9000, 1), (8, 40, 2500, 40)])
def test_padded_batches(torch_cuda, qctx, h, sq, p, so, fill):
    assert shares(torch_cuda, 3, h, sq, p, so) > 1
    valid = np.ones((3, p + so), np.uint8)
    valid[0, p // 3:p] = 0  # whole shares of the cache
    valid[1] = np.random.default_rng(p).random(p + so) < 0.5
    valid[1, :1500] = 0
    valid[2] = 0  # one key alone
    valid[2, p - 130] = 1
    assert_near(*attn_case(torch_cuda, qctx, 3, h, sq, p, so, seed=p + sq, valid=valid, fill=fill))


@pytest.mark.parametrize("sq,p,so", [(1, 4000, 0), (5, 2300, 3), (30, 6001, 100)])
def test_a_row_without_a_visible_key_is_nan(torch_cuda, qctx, sq, p, so):
    assert shares(torch_cuda, 2, 2, sq, p, so) > 1
    valid = np.ones((2, p + so), np.uint8)
    valid[1] = 0
    got, want, a = attn_case(torch_cuda, qctx, 2, 2, sq, p, so, seed=so, valid=valid)
    assert np.isnan(got[1]).all() and np.isnan(want[1]).all()
    assert_near(got[:1], want[:1], a[:1])


@pytest.mark.parametrize("keys", [[5500], range(700)])
def test_a_nan_query_or_key_stays_in_its_rows(torch_cuda, qctx, keys):
    """One key of the last share, or every key of the first ones; hidden ones do not show."""
    torch, p = torch_cuda, 6000
    assert shares(torch, 1, 2, 4, p, 0) > 1
    rng = np.random.default_rng(8)
    q_d, _ = bf16(torch, rng.standard_normal((1, 2, 4, 128)))
    k_d, _ = bf16(torch, rng.standard_normal((1, 2, p, 128)))
    v_d = k_d.clone()
    q_d[0, 0, 2, 100] = float("nan")
    k_d[0, 1, list(keys), 3] = float("nan")
    kv = stored(torch, qctx, k_d, v_d)
    out = torch.empty(1, 4, 256, dtype=torch.bfloat16, device="cuda")
    args = (q_d.data_ptr(), 1, 2, 4, kv, 0, None, None, 0, 0.088, out.data_ptr())
    qctx.attention(*args, stream=stream(torch))
    nan = np.isnan(host(out.float())).reshape(4, 2, 128)
    assert nan[2, 0].all() and not nan[[0, 1, 3], 0].any() and nan[:, 1].all()
    ok = np.ones((1, p), np.uint8)
    ok[0, list(keys)] = 0
    ok = dev(torch, ok)
    qctx.attention_masked(*args, key_valid=ok.data_ptr(), stream=stream(torch))
    nan = np.isnan(host(out.float())).reshape(4, 2, 128)
    assert nan[2, 0].all() and not nan[[0, 1, 3]].any() and not nan[2, 1].any()
    kv.free()


@pytest.mark.parametrize("at", [40, 2900])
@pytest.mark.parametrize("bits", [16.5, 24.0, 40.0])
def test_a_key_that_takes_nearly_all_leaves_the_others_their_precision(torch_cuda, qctx, at, bits):
    """A key of value 0 with 2^bits the probability of each other one, in the first share or the last."""
    torch, p, sq, rng = torch_cuda, 3000, 2, np.random.default_rng(3)
    assert shares(torch, 1, 1, sq, p, 0) > 1
    q_d, q = bf16(torch, np.where(np.arange(128) == 0, 1.0, 0.0) * np.ones((1, 1, sq, 1)))
    k = np.zeros((1, 1, p, 128))
    k[0, 0, at, 0] = 6.0
    v = np.abs(rng.standard_normal((1, 1, p, 128))) + 0.5
    v[0, 0, at] = 0.0
    (k_d, k), (v_d, v) = bf16(torch, k), bf16(torch, v)
    pk, pv = kv4_ref.near_kv(k, v)
    scale = bits * np.log(2.0) / 6.0
    kv = stored(torch, qctx, k_d, v_d)
    out = torch.empty(1, sq, 128, dtype=torch.bfloat16, device="cuda")
    qctx.attention(q_d.data_ptr(), 1, 1, sq, kv, 0, None, None, 0, scale, out.data_ptr(), stream(torch))
    kv.free()
    got = host(out.float()).reshape(1, sq, 1, 128).astype(np.float64)
    want, a = kv4_ref.attention(q, pk, pv, scale, None)
    tile = pv[0, 0, at // 128 * 128:at // 128 * 128 + 128]
    tol = 2.0 ** -8 * (a + np.abs(want)) + 2.0 ** -9 * a + 2.0 ** -23 * np.abs(tile).sum(0)
    worst = np.max(np.abs(got - want) / tol)
    assert np.isfinite(got).all() and worst <= 1.0, worst


@pytest.mark.parametrize("sq,so", [(1, 0), (2, 33)])
def test_the_most_shares(torch_cuda, qctx, sq, so):
    assert shares(torch_cuda, 1, 1, sq, 32500, so) == 64
    assert_near(*attn_case(torch_cuda, qctx, 1, 1, sq, 32500, so, seed=11, sharp=3.0))
    valid = np.ones((1, 32500 + so), np.uint8)
    valid[0, 600:32000] = 0  # nearly every share
    assert_near(*attn_case(torch_cuda, qctx, 1, 1, sq, 32500, so, seed=12, valid=valid, fill=float("nan")))
