"""Adapters where their numbers are at a limit: f32 outputs that keep 24 bits of t on every route,
ranks up to the largest, and scales that are no numbers.

f32 outputs carry t as three bf16 parts, 24 bits, where the matrix pipe multiplies it. Here x, A and B
are such that t has 21 significant bits, every sum is exact and every output is one t: off by at most
the roundings of the three additions that join the parts and the projection, 3 * 2^-24 of it. Two
parts would be off by up to 2^-17.
"""
import numpy as np
import pytest

import oracle as O
import qimm
import synth
from gpu_util import bf16_dev, dev, host, stream
from test_gpu_adapters import Case
from test_gpu_block import SMALL, block_tensors, make_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k,ranks,way", [
    (20, 256, 256, (16, 40), "rows"), (200, 512, 256, (16,), "rows"), (300, 256, 1024, (16, 40), "pass"),
    (514, 512, 2048, (40, 16), "pass"), (700, 12288, 128, (40, 16), "steps"), (1030, 12288, 256, (16, 12), "steps"),
    (4299, 4096, 256, (33, 40), "steps")])
def test_f32_outputs_keep_24_bits_of_t(torch_cuda, qctx, m, n, k, ranks, way):
    torch = torch_cuda
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    route = qimm.qmatmul_route(synth.BF16, n, k, m, cus)
    if way != "rows":
        assert (route.kernel == qimm.GEMM_BF16_ROWS and route.splits == 1) == (way == "steps")
    rng = np.random.default_rng(m)
    w = qctx.upload(synth.BF16, n, k, bytes(2 * n * k))  # zeros
    given, scale = [], (1.0, -2.0)
    for r, s in zip(ranks, scale):
        a, b = np.zeros((r, k)), np.zeros((n, r))
        a[np.repeat(np.arange(r), 3), np.arange(3 * r)] = 1.0  # t of a rank: the sum of three of x
        b[np.arange(n), np.arange(n) % r] = 1.0
        given.append((s, qimm.BF16, *(bf16_dev(torch, t)[0].cpu().view(torch.uint8).numpy().tobytes() for t in (a, b))))
    ad = qctx.adapters_create(n, k, given)
    # 8, 8 and 4 bits, 2^8 apart: from below 2 down to 2^-19
    x = rng.choice([-1.0, 1.0], (m, k)) * np.where(np.arange(k) % 3 == 2, (1 + rng.integers(0, 8, (m, k)) / 8) * 2.0 ** -16,
                                                   (1 + rng.integers(0, 128, (m, k)) / 128) * 2.0 ** (-8.0 * (np.arange(k) % 3)))
    x_d, xv = bf16_dev(torch, x)
    assert np.array_equal(xv, x)
    ids = np.arange(m) * 4 // m % 3 - (m > 4)  # runs of one adapter, the other and none
    ids_d, y = dev(torch, ids.astype(np.int32)), torch.full((m, n), 3.0, device="cuda")
    qctx.qmatmul_adapters(w, ad, ids_d.data_ptr(), x_d.data_ptr(), m, k, y.data_ptr(), qimm.F32, stream(torch))
    got = host(y).astype(np.float64)
    want, two = np.zeros((m, n)), np.zeros((m, n))
    for i, r in enumerate(ranks):
        rows = ids == i
        t = x[rows, :3 * r].reshape(-1, r, 3).sum(-1)
        hi = O.bf16_round(t.astype(np.float32)).astype(np.float64)
        lo = O.bf16_round((t - hi).astype(np.float32)).astype(np.float64)
        want[rows], two[rows] = scale[i] * t[:, np.arange(n) % r], scale[i] * (hi + lo)[:, np.arange(n) % r]
    bar = 3 * 2.0 ** -24 * np.abs(want)
    assert (np.abs(two - want) > 8 * bar).any()  # it tells two parts from three
    assert (np.abs(got - want) <= bar).all(), np.max(np.abs(got - want) / np.maximum(np.abs(want), 1e-9))
    ad.free()
    w.free()


@pytest.mark.parametrize("m,n,k,ranks", [(1, 256, 512, (1024,)), (5, 384, 256, (1023, 1024)), (64, 256, 1024, (1024, 7, 1000)),
                                         (70, 256, 512, (1024, 1)), (300, 256, 512, (900, 1024)), (1500, 512, 512, (1024,)),
                                         (4299, 4096, 256, (1024, 30))])
def test_ranks_up_to_the_largest(torch_cuda, qctx, m, n, k, ranks):
    c = Case(torch_cuda, qctx, synth.BF16, n, k, ranks, seed=m)
    rng = np.random.default_rng(m)
    x_d, x = bf16_dev(torch_cuda, rng.standard_normal((m, k)))
    ids = np.arange(m) * 3 // m % (len(ranks) + 1) - (m > 70)
    ids_d = dev(torch_cuda, ids.astype(np.int32))
    at = np.arange(m) if m <= 1500 else np.arange(0, m, 29)
    for out_type in (qimm.F32, qimm.BF16):
        y = c.call(x_d, m, ids_d, out_type)
        c.check(host(y.float())[at], x[at], ids[at], out_type)
    c.free()


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf")])
def test_a_scale_that_is_no_number_is_refused(torch_cuda, qctx, scale):
    """In a block it would reach the projections that the adapter leaves alone."""
    hid = SMALL["hidden"]
    a, b, keep = bytes(2 * hid * 2), bytes(hid * 2 * 2), []
    with pytest.raises(qimm.QimmError, match="QIMM_ERR_ARG"):
        qctx.adapters_create(hid, hid, [(1.0, qimm.BF16, a, b), (scale, qimm.BF16, a, b)])
    w = make_case(5, SMALL, 1, 4, 0, synth.Q8_0, synth.Q8_0)[0]
    blk = qctx.block_create(qimm.BlockConfig(hid, SMALL["heads"], 128, SMALL["mlp"]), block_tensors(w, keep))
    for pairs in ({"to_q": (qimm.BF16, hid, hid, 2, a, b)}, {}):
        with pytest.raises(qimm.QimmError, match="QIMM_ERR_ARG"):
            blk.set_adapters([(1.0, {}), (scale, pairs)])
    blk.free()
