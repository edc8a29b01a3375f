"""Calls of the batched-request operators that are allowed and out of the ordinary: as many adapters
as there may be, rows far apart, one token of one request through a block, two contexts at work at
once on one weight, masked attention in shares replayed from a graph, many heads."""
import numpy as np
import pytest

import kv4_ref
import oracle as O
import qimm
import synth
from gpu_util import bf16_dev, cos_sim, dev, host, max_abs_rel, stream
from test_gpu_adapters import Case
from test_gpu_block import SMALL, block_tensors, make_case
from test_gpu_block_adapters import ALL, make_adapters, merged
from test_gpu_kv4 import assert_near, stored

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [40, 300, 2500])
def test_as_many_adapters_as_there_may_be(torch_cuda, qctx, m):
    """65535 of rank 1, y = s x a for a row's own: the last ids, and the first past them."""
    torch, n, k, count = torch_cuda, 128, 64, 65535
    w = qctx.upload(synth.BF16, n, k, bytes(2 * n * k))
    one = bf16_dev(torch, np.ones((n, 1)))[0].cpu().view(torch.uint8).numpy().tobytes()
    a = bf16_dev(torch, np.eye(k))[0].cpu().view(torch.uint8).numpy()
    ad = qctx.adapters_create(n, k, [(1.0 + i % 7, qimm.BF16, a[i % k].tobytes(), one) for i in range(count)])
    rng = np.random.default_rng(m)
    x_d, x = bf16_dev(torch, rng.standard_normal((m, k)))
    ids = rng.integers(0, count, m)
    ids[:4] = (count - 1, count, 0, -2 ** 31)
    y = torch.full((m, n), 3.0, device="cuda")
    ids_d = dev(torch, ids.astype(np.int32))
    qctx.qmatmul_adapters(w, ad, ids_d.data_ptr(), x_d.data_ptr(), m, k, y.data_ptr(), qimm.F32, stream(torch))
    want = np.where((ids >= 0) & (ids < count), x[np.arange(m), ids % count % k] * (1.0 + ids % count % 7), 0.0)[:, None]
    assert (np.abs(host(y) - want) <= 2.0 ** -22 * np.abs(want)).all()
    ad.free()
    w.free()


@pytest.mark.parametrize("m", [3, 70, 300])
def test_rows_far_apart(torch_cuda, qctx, m):
    """A row stride above what the kernel over bf16 rows takes."""
    torch, n, k, lda = torch_cuda, 512, 256, (1 << 22) + 8
    c = Case(torch, qctx, synth.BF16, n, k, (16, 33), seed=m)
    x = torch.zeros((m - 1) * lda + k, dtype=torch.bfloat16, device="cuda")
    x_d, xv = bf16_dev(torch, np.random.default_rng(m).standard_normal((m, k)))
    torch.as_strided(x, (m, k), (lda, 1)).copy_(x_d)
    ids = np.arange(m) % 3 - 1
    ids_d = dev(torch, ids.astype(np.int32))
    qctx.qmatmul_adapters_reserve(c.w, c.ad, m, qimm.F32)
    for out_type in (qimm.F32, qimm.BF16):
        c.check(host(c.call(x, m, ids_d, out_type, lda=lda).float()), xv, ids, out_type)
    c.free()


@pytest.mark.parametrize("codes_only", [False, True])
@pytest.mark.parametrize("b,s", [(1, 1), (3, 1), (1, 65), (5, 13)])
def test_few_tokens_through_a_block(torch_cuda, qctx, qctx_codes, b, s, codes_only):
    torch, hid, mlp = torch_cuda, SMALL["hidden"], SMALL["mlp"]
    w, x, mod, pe, kpre, vpre = make_case(b + s, SMALL, b, s, 40, synth.Q4_K, synth.Q6_K)
    given, deltas = make_adapters(torch, np.random.default_rng(s), (ALL, ("to_v", "mlp_out")))
    ids, keep = np.arange(b) % 2, []
    ctx = qctx_codes if codes_only else qctx
    blk = ctx.block_create(qimm.BlockConfig(hid, SMALL["heads"], 128, mlp), block_tensors(w, keep))
    blk.set_adapters(given)
    blk.set_act_mode(qimm.ACT_BF16)
    ids_d = dev(torch, ids.astype(np.int32))
    blk.set_adapter_ids(ids_d.data_ptr())
    x_d, mod_d, pe_d = dev(torch, x), dev(torch, mod), dev(torch, pe)
    kv = ctx.kv_create(1, b, SMALL["heads"], 40)
    k_d, v_d = dev(torch, kpre.view(np.int16)), dev(torch, vpre.view(np.int16))
    kv.store(0, k_d.data_ptr(), v_d.data_ptr(), stream(torch))
    blk.forward(x_d.data_ptr(), x_d.data_ptr(), b, s, mod_d.data_ptr(), pe_d.data_ptr(), kv, 0, None, None, stream(torch))  # in place
    got = host(x_d)
    blk.free()
    kv.free()
    want = np.concatenate([O.block_forward(SMALL, merged(w, deltas[a]), x[i:i + 1], mod[i:i + 1], pe, kpre[i:i + 1],
                                           vpre[i:i + 1], mode=O.EXACT)[0] for i, a in enumerate(ids)])
    assert cos_sim(got, want) >= 0.9999 and cos_sim(got - x, want - x) >= 0.9999 and max_abs_rel(got, want) <= 2e-2


def test_two_contexts_at_once(torch_cuda):
    """One weight, its adapters and two 4-bit caches, used through two contexts on two streams."""
    torch, n, k, heads, p = torch_cuda, 1024, 1024, 8, 3000
    ctxs = [qimm.Context(0), qimm.Context(0)]
    c = Case(torch, ctxs[0], synth.Q4_K, n, k, (16, 40), seed=5)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    gen = torch.Generator(device="cuda").manual_seed(3)

    def draw(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(torch.bfloat16)

    work = []
    for ctx, m in zip(ctxs, (700, 2100)):
        kv = ctx.kv_create_q4(1, 1, heads, p)
        kk, vv, q, x = draw(1, heads, p, 128), draw(1, heads, p, 128), draw(1, heads, 5, 128), draw(m, k)
        ids = torch.randint(-1, 2, (m,), device="cuda", generator=gen, dtype=torch.int32)
        y, o = torch.empty(m, n, dtype=torch.bfloat16, device="cuda"), torch.empty(1, 5, heads * 128, dtype=torch.bfloat16, device="cuda")
        ctx.qmatmul_adapters_reserve(c.w, c.ad, m, qimm.BF16)
        work.append((ctx, kv, kk, vv, q, x, ids, y, o, m))

    def step(i):
        ctx, kv, kk, vv, q, x, ids, y, o, m = work[i]
        s = streams[i].cuda_stream
        kv.store(0, kk.data_ptr(), vv.data_ptr(), s)
        ctx.attention(q.data_ptr(), 1, heads, 5, kv, 0, None, None, 0, 0.088, o.data_ptr(), s)
        ctx.qmatmul_adapters(c.w, c.ad, ids.data_ptr(), x.data_ptr(), m, k, y.data_ptr(), qimm.BF16, s)

    torch.cuda.synchronize()
    alone = []
    for i in (0, 1):
        step(i)
        torch.cuda.synchronize()
        alone.append((work[i][7].clone(), work[i][8].clone()))
    for _ in range(4):
        for w in work:
            w[7].zero_(), w[8].zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            for i in (0, 1):
                step(i)
        torch.cuda.synchronize()
        for i in (0, 1):
            assert torch.equal(work[i][7], alone[i][0]) and torch.equal(work[i][8], alone[i][1])
    for w in work:
        w[1].free()
    c.free()
    for ctx in ctxs:
        ctx.close()


def test_masked_shares_from_a_graph(torch_cuda, qctx):
    torch, b, h, sq, p, so = torch_cuda, 2, 2, 3, 5000, 20
    gen = torch.Generator(device="cuda").manual_seed(1)

    def draw(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(torch.bfloat16)

    k, v, q, ko, vo = draw(b, h, p, 128), draw(b, h, p, 128), draw(b, h, sq, 128), draw(b, h, so, 128), draw(b, h, 128, so)
    ok, out = torch.ones(b, p + so, dtype=torch.uint8, device="cuda"), torch.empty(b, sq, h * 128, dtype=torch.bfloat16, device="cuda")
    kv = qctx.kv_create_q4(1, b, h, p)
    kv.store(0, k.data_ptr(), v.data_ptr(), stream(torch))

    def step():
        qctx.attention_masked(q.data_ptr(), b, h, sq, kv, 0, ko.data_ptr(), vo.data_ptr(), so, 0.088, out.data_ptr(),
                              key_valid=ok.data_ptr(), stream=stream(torch))

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(4):
        ok.fill_(1)
        ok[0, 1000 * i + 7:p] = 0
        ok[1, :1200 * i] = 0
        q.copy_(draw(*q.shape))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.zero_()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, out) and bool(got.isfinite().all()), i
    kv.free()


def test_many_heads(torch_cuda, qctx):
    """As many heads as a cache may have, one row of each over a few keys."""
    torch, b, h, p, so = torch_cuda, 4369, 15, 3, 1
    gen = torch.Generator(device="cuda").manual_seed(9)
    k, v, q, ko, vt = (torch.randn(b, h, *shape, device="cuda", generator=gen).to(torch.bfloat16)
                       for shape in ((p, 128), (p, 128), (1, 128), (so, 128), (128, so)))
    kv, out = stored(torch, qctx, k, v), torch.empty(b, 1, h * 128, dtype=torch.bfloat16, device="cuda")
    qctx.attention(q.data_ptr(), b, h, 1, kv, 0, ko.data_ptr(), vt.data_ptr(), so, 0.088, out.data_ptr(), stream(torch))
    got = host(out.float()).reshape(b, 1, h, 128)
    kv.free()
    for at in (0, 1, 2730, b - 1):  # every head of an entry
        f = [host(t[at:at + 1].float()).astype(np.float64) for t in (k, v, q, ko, vt)]
        pk, pv = kv4_ref.near_kv(f[0], f[1])
        want, a = kv4_ref.attention(f[2], np.concatenate([pk, f[3]], 2), np.concatenate([pv, np.swapaxes(f[4], 2, 3)], 2), 0.088)
        assert_near(got[at:at + 1].astype(np.float64), want, a)
