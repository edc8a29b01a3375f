"""Low-rank adapters of many requests beside a projection (qimm_qmatmul_adapters) against 64
bits. The weight's values are the bf16 rows that the products multiply (exact for BF16 weights).

Bar per output, with X = sum |x| |w|, T_r = sum |x| |a_r|, all f32 sums in steps of 32 terms:
e(K) = (K / 32 + 32) 2^-24 of the sum's absolute terms for each of W, A; t = hi + lo of two bf16
numbers is off by at most 2^-16 of itself; the second product's f32 sum by e(rank). A bf16 output
adds 2^-8 of itself.
"""
import numpy as np
import pytest

import oracle as O
import qimm
import synth
from gpu_util import bf16_dev, dev, host, stream

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, torch, ctx, t, n, k, ranks, seed, kind=qimm.BF16):
        rng = np.random.default_rng(seed)
        self.torch, self.ctx, self.n, self.k, self.ranks = torch, ctx, n, k, ranks
        _, raw, _, _ = synth.weight(rng, t, n, k, 0.02)
        self.w = ctx.upload(t, n, k, raw.tobytes())
        self.wv = O.bf16_round(O.dequantize(t, raw, n * k).reshape(n, k)).astype(np.float64)
        self.a, self.b, self.scale, given = [], [], [], []
        for i, r in enumerate(ranks):
            a, b = rng.standard_normal((r, k)) / np.sqrt(k), rng.standard_normal((n, r)) * 0.3
            ad, av = bf16_dev(torch, a)
            bd, bv = bf16_dev(torch, b)
            self.a.append(av.astype(np.float64))
            self.b.append(bv.astype(np.float64))
            self.scale.append((0.5 + i) / r * (-1) ** i)
            store = {qimm.BF16: lambda d: d.cpu().view(torch.uint8).numpy().tobytes(),
                     qimm.F32: lambda d: d.float().cpu().numpy().tobytes()}[kind]
            given.append((self.scale[-1], kind, store(ad), store(bd)))
        self.ad = ctx.adapters_create(n, k, given)

    def free(self):
        self.ad.free()
        self.w.free()

    def call(self, x_d, m, ids_d, out_type, lda=None, fill=5.0):
        torch = self.torch
        y = torch.full((m, self.n), fill, dtype=torch.float32 if out_type == qimm.F32 else torch.bfloat16, device="cuda")
        self.ctx.qmatmul_adapters(self.w, self.ad, ids_d.data_ptr(), x_d.data_ptr(), m, lda or self.k, y.data_ptr(), out_type,
                                  stream(torch))
        return y

    def check(self, got, x, ids, out_type):
        def e(n):
            return (n / 32 + 32) * 2.0 ** -24
        x = x.astype(np.float64)
        want, tol = x @ self.wv.T, e(self.k) * (np.abs(x) @ np.abs(self.wv).T)
        for i, (a, b, s) in enumerate(zip(self.a, self.b, self.scale)):
            rows = np.asarray(ids) == i
            if rows.any():
                t, tt = s * (x[rows] @ a.T), abs(s) * (np.abs(x[rows]) @ np.abs(a).T)
                want[rows] += t @ b.T
                tol[rows] += (e(self.k) * tt + (2.0 ** -16 + e(len(a))) * np.abs(t)) @ np.abs(b).T
        tol += e(32) * np.abs(want)
        if out_type == qimm.BF16:
            tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(want)
        worst = np.max(np.abs(got.astype(np.float64) - want) / tol)
        assert np.isfinite(got).all() and worst <= 1.0, worst


def ids_of(kind, m, count, rng):
    if kind == "one":
        return np.full(m, count - 1)
    if kind == "requests":  # runs of rows, one of them without
        return (np.arange(m) * 5 // m) % (count + 1) - 1
    if kind == "none":
        return np.where(np.arange(m) % 2, -1, 2 ** 31 - 1)
    return rng.integers(-2, count + 2, m)  # any, next to each other


@pytest.mark.parametrize("kind", ["one", "requests", "any", "none"])
@pytest.mark.parametrize("m,n,k,ranks", [
    (1, 128, 256, (4,)), (1, 256, 4096, (16, 1)), (7, 384, 512, (8, 3, 16)), (16, 256, 1024, (33,)), (17, 128, 64, (5, 64)),
    (48, 512, 2048, (16, 8, 40, 1)), (64, 256, 512, (64, 128)), (65, 256, 512, (16,)), (129, 384, 320, (7, 31, 32)),
    (300, 256, 1024, (12, 200)), (514, 512, 512, (16, 64)), (1030, 512, 1024, (8, 96, 65)), (2100, 256, 384, (16, 130))])
def test_against_64_bits(torch_cuda, qctx, kind, m, n, k, ranks):
    c = Case(torch_cuda, qctx, synth.BF16, n, k, ranks, seed=m + n)
    rng = np.random.default_rng(m)
    x_d, x = bf16_dev(torch_cuda, rng.standard_normal((m, k)))
    ids = ids_of(kind, m, len(ranks), rng)
    ids_d = dev(torch_cuda, ids.astype(np.int32))
    for out_type in (qimm.F32, qimm.BF16):
        c.check(host(c.call(x_d, m, ids_d, out_type).float()), x, ids, out_type)
    c.free()


@pytest.mark.parametrize("codes_only", [False, True])
@pytest.mark.parametrize("t", [synth.Q8_0, synth.Q4_K, synth.Q6_K])
@pytest.mark.parametrize("m", [2, 40, 200, 1500, 2560])
def test_quantized_weights(torch_cuda, qctx, qctx_codes, t, m, codes_only):
    """On every route of the shared product, with and without its bf16 rows. Up to 16 rows a
    Q4_K product takes the exact weights instead of their bf16 rounding: its outputs are
    compared with those of the product without adapters."""
    torch = torch_cuda
    ctx = qctx_codes if codes_only else qctx
    c = Case(torch, ctx, t, 512, 1024, (16, 24), seed=t + m)
    rng = np.random.default_rng(m)
    x_d, x = bf16_dev(torch, rng.standard_normal((m, 1024)))
    ids = ids_of("requests", m, 2, rng)
    ids_d = dev(torch, ids.astype(np.int32))
    if t == synth.Q4_K and m <= 16:
        y = torch.empty(m, 512, dtype=torch.float32, device="cuda")
        ctx.qmatmul(c.w, x_d.data_ptr(), m, 1024, y.data_ptr(), qimm.F32, stream(torch))
        c.wv = np.zeros_like(c.wv)
        got = host(c.call(x_d, m, ids_d, qimm.F32)).astype(np.float64) - host(y)
        want = np.zeros((m, 512))
        for i in (0, 1):
            want[ids == i] = c.scale[i] * (x[ids == i].astype(np.float64) @ c.a[i].T) @ c.b[i].T
        assert np.abs(got - want).max() <= 2.0 ** -16 * (np.abs(want).max() + np.abs(host(y)).max())
    else:
        c.check(host(c.call(x_d, m, ids_d, qimm.F32)), x, ids, qimm.F32)
    c.free()


@pytest.mark.parametrize("m,ranks", [
    (65, (64,) * 3), (100, (40, 41) * 60), (128, (64,) * 128), (129, (64,) * 8), (200, (16, 20) * 100), (256, (16,) * 256),
    (256, (32,) * 300), (257, (16,) * 257)])
def test_an_adapter_for_every_row(torch_cuda, qctx, m, ranks):
    """By rows and by tiles, on both sides of the bounds between them."""
    c = Case(torch_cuda, qctx, synth.BF16, 256, 256, ranks, seed=m)
    rng = np.random.default_rng(m)
    x_d, x = bf16_dev(torch_cuda, rng.standard_normal((m, 256)))
    ids = rng.permutation(max(m, len(ranks)))[:m]
    ids_d = dev(torch_cuda, ids.astype(np.int32))
    for out_type in (qimm.F32, qimm.BF16):
        c.check(host(c.call(x_d, m, ids_d, out_type).float()), x, ids, out_type)
    c.free()


@pytest.mark.parametrize("out_type", [qimm.F32, qimm.BF16])
@pytest.mark.parametrize("m,n,k,ranks", [
    (4096, 4096, 256, (64,)), (700, 12288, 128, (16, 3)), (1030, 12288, 256, (8, 65, 130)), (4299, 4096, 256, (33, 16)),
    (2051, 4096, 512, tuple([1, 2, 5] * 100)), (6889, 4096, 128, (16,) * 7)])
def test_steps_of_the_product_over_bf16_rows(torch_cuda, qctx, m, n, k, ranks, out_type):
    """Large and small tiles, tails, several adapters and up to a tile's worth of them, an odd
    number of steps; rows that are no numbers stay alone."""
    torch = torch_cuda
    rng = np.random.default_rng(m)
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    route = qimm.qmatmul_route(qimm.BF16, n, k, m, cus)
    route = qimm.qmatmul_route(qimm.BF16, n, k, m - route.tail, cus)
    assert route.kernel == qimm.GEMM_BF16_ROWS and route.splits == 1
    c = Case(torch, qctx, synth.BF16, n, k, ranks, seed=m + k)
    x_d, _ = bf16_dev(torch, rng.standard_normal((m, k)))
    for kind in ("requests", "any", "one", "none"):
        ids = ids_of(kind, m, len(ranks), rng)
        ids_d = dev(torch, ids.astype(np.int32))
        got = c.call(x_d, m, ids_d, out_type)
        # the bar of Case.check, on the device
        x, w = x_d.double(), dev(torch, c.wv)
        want, tol = x @ w.t(), (k / 32 + 32) * 2.0 ** -24 * (x.abs() @ w.abs().t())
        for i in np.unique(ids):
            if 0 <= i < len(ranks):
                rows = dev(torch, np.flatnonzero(ids == i))
                a, b, s = dev(torch, c.a[i]), dev(torch, c.b[i]), c.scale[i]
                t = s * (x[rows] @ a.t())
                want[rows] += t @ b.t()
                tol[rows] += ((k / 32 + 32) * 2.0 ** -24 * abs(s) * (x[rows].abs() @ a.abs().t()) +
                              (2.0 ** -16 + (len(a) / 32 + 32) * 2.0 ** -24) * t.abs()) @ b.abs().t()
        tol += 33 * 2.0 ** -24 * want.abs()
        if out_type == qimm.BF16:
            tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()
        worst = float(((got.double() - want).abs() / tol).max())
        assert worst <= 1.0, (kind, worst)
        bad = x_d.clone()
        bad[5], bad[min(m - 1, 300), 7] = float("inf"), float("nan")
        after = c.call(bad, m, ids_d, out_type)
        keep = torch.ones(m, dtype=torch.bool, device="cuda")
        keep[5] = keep[min(m - 1, 300)] = False
        assert torch.equal(got[keep], after[keep]) and bool(after[min(m - 1, 300)].isnan().all()), kind
    c.free()


def test_rows_without_adapters_equal_the_plain_product_within_rounding(torch_cuda, qctx):
    torch = torch_cuda
    c = Case(torch, qctx, synth.Q8_0, 512, 1024, (16,), seed=1)
    for m in (3, 50, 100, 700, 2304):
        x_d, _ = bf16_dev(torch, np.random.default_rng(m).standard_normal((m, 1024)))
        ids = torch.full((m,), -1, dtype=torch.int32, device="cuda")
        y = torch.empty(m, 512, dtype=torch.float32, device="cuda")
        qctx.qmatmul(c.w, x_d.data_ptr(), m, 1024, y.data_ptr(), qimm.F32, stream(torch))
        got = c.call(x_d, m, ids, qimm.F32)
        assert float((got - y).abs().max()) <= 2e-5 * float(y.abs().max())
    c.free()


def test_strided_rows_f32_adapters_and_rows_behind_the_last(torch_cuda, qctx):
    torch = torch_cuda
    c = Case(torch, qctx, synth.BF16, 256, 512, (20, 4), seed=3, kind=qimm.F32)
    for m in (5, 90, 600):
        rng = np.random.default_rng(m)
        x_d, x = bf16_dev(torch, rng.standard_normal((m, 520)))
        x_d[:, 512:] = float("nan")
        ids = rng.integers(-1, 2, m)
        y = torch.full((m + 2, 256), 9.0, dtype=torch.float32, device="cuda")
        c.ctx.qmatmul_adapters(c.w, c.ad, dev(torch, ids.astype(np.int32)).data_ptr(), x_d.data_ptr(), m, 520, y.data_ptr(),
                               qimm.F32, stream(torch))
        c.check(host(y[:m]), x[:, :512], ids, qimm.F32)
        assert (host(y[m:]) == 9.0).all()
    c.free()


def test_a_row_that_is_no_number_stays_alone(torch_cuda, qctx):
    """Rows are independent, whichever adapters share their tile."""
    torch = torch_cuda
    c = Case(torch, qctx, synth.BF16, 256, 512, (16, 16), seed=4)
    for m in (16, 300, 2304):
        x_d, _ = bf16_dev(torch, np.random.default_rng(m).standard_normal((m, 512)))
        ids = dev(torch, (np.arange(m) % 3 - 1).astype(np.int32))
        before = host(c.call(x_d, m, ids, qimm.F32))
        x_d[5] = float("inf")
        x_d[7, 3] = float("nan")
        after = host(c.call(x_d, m, ids, qimm.F32))
        keep = np.ones(m, bool)
        keep[[5, 7]] = False
        assert np.array_equal(before[keep], after[keep]) and np.isnan(after[7]).all()
    c.free()


def test_replays_of_a_graph_equal_eager_calls(torch_cuda, qctx):
    torch = torch_cuda
    c = Case(torch, qctx, synth.Q4_K, 512, 1024, (16, 8, 40), seed=6)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for m in (4, 150, 1100):
        x = torch.randn(m, 1024, device="cuda", generator=gen).to(torch.bfloat16)
        ids = torch.randint(-1, 3, (m,), device="cuda", generator=gen, dtype=torch.int32)
        y = torch.empty(m, 512, dtype=torch.bfloat16, device="cuda")

        def step():
            qctx.qmatmul_adapters(c.w, c.ad, ids.data_ptr(), x.data_ptr(), m, 1024, y.data_ptr(), qimm.BF16, stream(torch))

        qctx.qmatmul_adapters_reserve(c.w, c.ad, m, qimm.BF16)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for i in range(3):
            x.copy_(torch.randn(m, 1024, device="cuda", generator=gen).to(torch.bfloat16))
            ids.copy_(torch.randint(-1, 3, (m,), device="cuda", generator=gen, dtype=torch.int32))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = y.clone()
            y.zero_()
            step()
            torch.cuda.synchronize()
            assert torch.equal(got, y), (m, i)
        del graph
    c.free()


def test_refusals(torch_cuda, qctx):
    torch = torch_cuda
    c = Case(torch, qctx, synth.BF16, 256, 512, (16,), seed=7)
    other = qctx.upload(qimm.BF16, 128, 512, bytes(128 * 512 * 2))
    x = torch.zeros(4 * 512 + 8, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(4 * 256 + 8, dtype=torch.float32, device="cuda")
    ids = torch.zeros(5, dtype=torch.int32, device="cuda")
    a, b = bytes(16 * 512 * 2), bytes(256 * 16 * 2)

    def refused(status, call):
        with pytest.raises(qimm.QimmError, match=status):
            call()

    def product(w=c.w, i=ids.data_ptr(), xp=x.data_ptr(), m=4, lda=512, yp=y.data_ptr(), t=qimm.F32):
        qctx.qmatmul_adapters(w, c.ad, i, xp, m, lda, yp, t, stream(torch))

    refused("QIMM_ERR_SHAPE", lambda: product(w=other))
    refused("QIMM_ERR_ARG", lambda: product(i=None))
    refused("QIMM_ERR_ARG", lambda: product(i=ids.data_ptr() + 2))
    refused("QIMM_ERR_ARG", lambda: product(xp=x.data_ptr() + 2))
    refused("QIMM_ERR_ARG", lambda: product(m=-1))
    refused("QIMM_ERR_SHAPE", lambda: product(lda=504))
    refused("QIMM_ERR_TYPE", lambda: product(t=qimm.F16))
    product(m=0)
    refused("QIMM_ERR_SHAPE", lambda: qctx.adapters_create(250, 512, [(1.0, qimm.BF16, a, b)]))
    refused("QIMM_ERR_SHAPE", lambda: qctx.adapters_create(256, 520, [(1.0, qimm.BF16, a, b)]))
    refused("QIMM_ERR_ARG", lambda: qctx.adapters_create(256, 512, [(1.0, qimm.BF16, b"\x80\x7f" + a[2:], b)]))  # an infinity
    refused("QIMM_ERR_ARG", lambda: qctx.adapters_create(256, 512, [(1.0, qimm.BF16, a, b[:-2] + b"\xc0\x7f")]))  # a NaN
    refused("QIMM_ERR_SHAPE", lambda: qctx.adapters_create(256, 512, []))
    refused("QIMM_ERR_SHAPE", lambda: qctx.adapters_create(256, 512, [(1.0, qimm.BF16, a, b[:-2])]))
    refused("QIMM_ERR_TYPE", lambda: qctx.adapters_create(256, 512, [(1.0, qimm.Q8_0, a, b)]))
    refused("QIMM_ERR_ARG", lambda: product(yp=None))
    refused("QIMM_ERR_SHAPE", lambda: qctx.qmatmul_adapters_reserve(other, c.ad, 4, qimm.F32))
    assert c.ad.device_bytes() >= len(a) + len(b)
    other.free()
    c.free()
    torch.cuda.synchronize()
