"""The prefix cache held in 4 bits: what it stores, bit for bit; the attention of few queries
over its codes, against 64 bits; and every call that reads it expanded, against the same call
on a bf16 cache of the same values.

Bar of the attention over codes, per output with A = sum p |v| (p the exact probabilities):
- a query is the sum of two e4m3 numbers, exact but for values below 2^-15 of the row's
  largest (error 2^-22 of it), so scores are off by f32 roundings: e^s by less than 2^-12;
- a prefix key's probability is hi + lo, hi off by half a step 2^-4, lo by 2^-4 of that: 2^-8;
  an own key's is rounded to bf16: 2^-8; what falls below the e4m3 range of lo, 2^-23 of the
  largest of its 128 keys each: less than 2^-16 in all of keys of equal values;
- the output is rounded to bf16: 2^-8 of it.
Together 2^-8 (A + |out|) + 2^-9 A.
"""
import numpy as np
import pytest

import kv4_ref
import oracle as O
import qimm
import synth
from gpu_util import bf16_dev, cos_sim, dev, host, kv_close, max_abs_rel, stream
from test_gpu_block import SMALL, block_tensors, make_case

pytestmark = pytest.mark.gpu


def bf16(torch, x):
    """The bf16 device tensor of x and its values in f64."""
    t, v = bf16_dev(torch, np.asarray(x, np.float32))
    return t, v.astype(np.float64)


def stored(torch, qctx, k, v, layers=1, layer=0):
    b, h, p, _ = k.shape
    kv = qctx.kv_create_q4(layers, b, h, p)
    kv.store(layer, k.data_ptr(), v.data_ptr(), stream(torch))
    return kv


def read_back(torch, kv, like, layer=0):
    k, v = torch.full_like(like, 99.0), torch.full_like(like, 99.0)
    kv.load(layer, k.data_ptr(), v.data_ptr(), stream(torch))
    return k, v


# ---------------------------------------------------------------- storing

@pytest.mark.parametrize("b,h,p", [(1, 1, 1), (1, 2, 7), (2, 1, 31), (1, 2, 32), (1, 1, 33), (2, 2, 127), (1, 1, 128),
                                   (1, 2, 129), (2, 3, 300), (1, 1, 1023)])
def test_store_and_load_give_the_format(torch_cuda, qctx, b, h, p):
    torch = torch_cuda
    rng = np.random.default_rng(p)
    scale = 2.0 ** rng.integers(-12, 12, (b, h, p, 4, 1)).repeat(32, -1).reshape(b, h, p, 128)
    k_d, k = bf16(torch, rng.standard_normal((b, h, p, 128)) * scale)
    v_d, v = bf16(torch, rng.integers(-14, 15, (b, h, p, 128)) * 0.25 * 2.0 ** rng.integers(-1, 2, (b, h, p, 128)))
    kv = stored(torch, qctx, k_d, v_d)
    assert kv.bits == 4 and not kv.is_host and kv.prefix_len == p
    gk, gv = read_back(torch, kv, k_d)
    wk, wv = kv4_ref.near_kv(k, v)
    assert np.array_equal(host(gk.float()), wk) and np.array_equal(host(gv.float()), wv)
    kv.free()


def test_store_extremes(torch_cuda, qctx):
    """Zeros, the smallest and the largest bf16 numbers, powers of two around 7 2^s, signed zeros."""
    torch = torch_cuda
    x = np.zeros((1, 1, 64, 128), np.float32)
    x[0, 0, 0, :32] = 3.3895e38
    x[0, 0, 1, :32] = 1e-40
    x[0, 0, 2, 0], x[0, 0, 2, 1] = 2.0 ** -118 * 7, 2.0 ** -120
    for i, e in enumerate(range(-126, 127, 9)):
        x[0, 0, 3 + i, 32:64] = np.linspace(-1, 1, 32, dtype=np.float32) * np.float32(2.0 ** e) * np.float32(1.75)
    x[0, 0, 40, 64:96] = -0.0
    k_d, k = bf16(torch, x)
    kv = stored(torch, qctx, k_d, k_d)
    gk, gv = read_back(torch, kv, k_d)
    wk, wv = kv4_ref.near_kv(k, k)
    assert np.array_equal(host(gk.float()), wk) and np.array_equal(host(gv.float()), wv)
    kv.free()


def test_numbers_that_are_none(torch_cuda, qctx):
    torch = torch_cuda
    rng = np.random.default_rng(5)
    x = rng.standard_normal((1, 1, 96, 128)).astype(np.float32)
    y = x.copy()
    k_d, v_d = bf16(torch, x)[0], bf16(torch, y)[0]
    k_d[0, 0, 3, 40] = float("nan")
    k_d[0, 0, 70, 5] = -float("inf")
    v_d[0, 0, 8, 9] = float("nan")
    v_d[0, 0, 40, 10], v_d[0, 0, 41, 10] = float("inf"), -float("inf")
    v_d[0, 0, 64:, 127] = float("inf")
    kv = stored(torch, qctx, k_d, v_d)
    gk, gv = (host(t.float())[0, 0] for t in read_back(torch, kv, k_d))
    wk = kv4_ref.near(np.nan_to_num(host(k_d.float())[0, 0].astype(np.float64), posinf=0, neginf=0))
    bad = np.zeros((96, 128), bool)
    bad[3, 32:64] = bad[70, :32] = True
    assert np.isnan(gk[bad]).all() and np.array_equal(gk[~bad], wk[~bad])
    clean = host(v_d.float())[0, 0].astype(np.float64)
    inf = np.isinf(clean)
    wv = kv4_ref.near_kv(np.zeros((1, 1, 96, 128)), np.where(np.isfinite(clean), clean, 0)[None, None])[1][0, 0]
    assert np.array_equal(gv[~inf], wv[~inf])
    assert gv[40, 10] == -gv[41, 10] > 0 and gv[40, 10] >= np.abs(gv[32:64, 10]).max()
    assert np.isfinite(gv).all() and (gv[64:, 127] == 6 * 2.0 ** -120).all()
    kv.free()


def test_layers_beyond_32_bit_offsets(torch_cuda, qctx):
    """The last of ten layers of 583 MB: every offset into it is above 2^32."""
    torch = torch_cuda
    b, h, p = 8, 32, 16640
    gen = torch.Generator(device="cuda").manual_seed(3)
    k = torch.randn(b, h, p, 128, device="cuda", generator=gen, dtype=torch.bfloat16)
    v = torch.randn(b, h, p, 128, device="cuda", generator=gen, dtype=torch.bfloat16)
    kv = stored(torch, qctx, k, v, layers=10, layer=9)
    gk, gv = read_back(torch, kv, k, 9)
    for at in ((0, 0), (5, 17), (7, 31)):
        wk, wv = kv4_ref.near_kv(host(k[at].float())[None, None], host(v[at].float())[None, None])
        assert np.array_equal(host(gk[at].float()), wk[0, 0]) and np.array_equal(host(gv[at].float()), wv[0, 0])
    q, _ = bf16(torch, np.random.default_rng(4).standard_normal((b, h, 1, 128)))
    out = torch.empty(b, 1, h * 128, dtype=torch.bfloat16, device="cuda")
    qctx.attention(q.data_ptr(), b, h, 1, kv, 9, None, None, 0, 0.09, out.data_ptr(), stream(torch))
    s = torch.matmul(q.float(), gk.float().transpose(2, 3).contiguous()) * 0.09
    want = torch.matmul(torch.softmax(s, -1), gv.float()).transpose(1, 2).reshape(b, 1, -1)
    assert float((out.float() - want).norm() / want.norm()) < 5e-3
    kv.free()


# ---------------------------------------------------------------- attention over the codes

def attn_case(torch, qctx, b, h, sq, p, so, seed, valid=None, scale=0.088, sharp=1.0, fill=None):
    rng = np.random.default_rng(seed)
    q_d, q = bf16(torch, rng.standard_normal((b, h, sq, 128)) * sharp)
    k_d, k = bf16(torch, rng.standard_normal((b, h, p, 128)))
    v_d, v = bf16(torch, rng.standard_normal((b, h, p, 128)))
    ko_d, ko = bf16(torch, rng.standard_normal((b, h, so, 128)))
    vo_d, vo = bf16(torch, rng.standard_normal((b, h, 128, so)))
    pk, pv = kv4_ref.near_kv(k, v) if p else (k, v)
    if fill is not None:  # what hidden keys hold
        hid = torch.from_numpy(valid == 0).cuda()
        k_d.masked_fill_(hid[:, None, :p, None], fill)
        ko_d.masked_fill_(hid[:, None, p:, None], fill)
        vo_d.masked_fill_(hid[:, None, None, p:], fill)
    kv = stored(torch, qctx, k_d, v_d) if p else qctx.kv_create_q4(1, b, h, 0)
    out = torch.full((b, sq, h * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    args = (q_d.data_ptr(), b, h, sq, kv, 0, ko_d.data_ptr() if so else None, vo_d.data_ptr() if so else None, so, scale,
            out.data_ptr())
    if valid is None:
        qctx.attention(*args, stream=stream(torch))
    else:
        v_ok = dev(torch, valid.astype(np.uint8))
        qctx.attention_masked(*args, key_valid=v_ok.data_ptr(), stream=stream(torch))
    got = host(out.float()).reshape(b, sq, h, 128).astype(np.float64)
    kv.free()
    want, a = kv4_ref.attention(q, np.concatenate([pk, ko], 2), np.concatenate([pv, np.swapaxes(vo, 2, 3)], 2), scale, valid)
    return got, want, a


def assert_near(got, want, a):
    tol = 2.0 ** -8 * (a + np.abs(want)) + 2.0 ** -9 * a
    assert np.isfinite(got).all()
    worst = np.max(np.abs(got - want) / np.maximum(tol, 1e-30))
    assert worst <= 1.0, worst


@pytest.mark.parametrize("b,h,sq,p,so", [
    (1, 1, 1, 1, 0), (1, 1, 1, 1, 1), (2, 3, 1, 128, 0), (1, 2, 1, 129, 1), (1, 2, 1, 127, 3), (2, 2, 16, 300, 16),
    (1, 3, 17, 333, 17), (1, 2, 15, 64, 0), (1, 1, 32, 1000, 33), (1, 2, 33, 511, 33), (1, 2, 48, 640, 64),
    (2, 1, 64, 1025, 65), (1, 1, 64, 31, 200), (1, 2, 5, 0, 9), (1, 1, 64, 0, 64), (1, 1, 3, 8191, 0),
    (3, 5, 7, 77, 250), (1, 1, 1, 40, 2049), (2, 2, 65, 140, 65), (1, 3, 300, 333, 129), (1, 1, 1000, 600, 0)])
def test_attention_over_codes(torch_cuda, qctx, b, h, sq, p, so):
    assert_near(*attn_case(torch_cuda, qctx, b, h, sq, p, so, seed=sq * 1000 + p + so))


@pytest.mark.parametrize("scale,sharp", [(0.088, 6.0), (-0.088, 1.0), (0.0, 1.0), (0.5, 1.0), (0.088, 1e-3), (1e-30, 1e20)])
def test_attention_over_codes_scales(torch_cuda, qctx, scale, sharp):
    """Scores up to a few hundred, a negative scale, none, and queries of other ranges."""
    assert_near(*attn_case(torch_cuda, qctx, 1, 2, 19, 260, 19, seed=int(sharp) % 97 + 3, scale=scale, sharp=sharp))


@pytest.mark.parametrize("fill", [None, float("nan"), float("inf"), -3.0e38])
@pytest.mark.parametrize("sq,p,so", [(1, 200, 1), (20, 700, 70), (64, 130, 64), (9, 129, 0), (150, 400, 33)])
def test_attention_over_codes_masked(torch_cuda, qctx, sq, p, so, fill):
    """Padded prompts: the tail of one, scattered keys and whole tiles of another; hidden keys
    may hold anything."""
    rng = np.random.default_rng(sq + p)
    valid = np.ones((3, p + so), np.uint8)
    valid[0, p // 2:p] = 0
    valid[1] = rng.random(p + so) < 0.6
    valid[1, 0] = 1
    valid[2, :min(p, 128)] = 0
    assert_near(*attn_case(torch_cuda, qctx, 3, 2, sq, p, so, seed=p, valid=valid, fill=fill))


@pytest.mark.parametrize("h,sq,so", [(2, 1, 0), (2, 5, 3), (2, 64, 64), (2, 300, 40), (8, 1300, 1300)])
def test_a_row_without_a_visible_key_is_nan(torch_cuda, qctx, h, sq, so):
    """As on the other caches (the softmax of -inf); the other entries are as without it. The
    last case takes the expanded layer."""
    valid = np.ones((2, 140 + so), np.uint8)
    valid[1] = 0
    got, want, a = attn_case(torch_cuda, qctx, 2, h, sq, 140, so, seed=so, valid=valid)
    assert np.isnan(got[1]).all() and np.isnan(want[1]).all()
    if sq < 1000:
        assert_near(got[:1], want[:1], a[:1])
    else:
        kv_close(got[:1], want[:1])


@pytest.mark.parametrize("sq,bits", [(8192, 24.0), (8192, 16.5), (2, 24.0), (2, 40.0)])
def test_a_key_that_takes_nearly_all_leaves_the_others_their_precision(torch_cuda, qctx, sq, bits):
    """A key of value 0 with 2^bits the probability of each other one, in one share or many. Its own
    tile's probabilities are off by up to 2^-23 of its."""
    torch = torch_cuda
    p, at, rng = 1536, 40, np.random.default_rng(3)
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
    want, a = kv4_ref.attention(q[:, :, :1], pk, pv, scale, None)
    extra = 2.0 ** -23 * np.abs(pv[0, 0, :128]).sum(0)
    tol = 2.0 ** -8 * (a + np.abs(want)) + 2.0 ** -9 * a + extra
    worst = np.max(np.abs(got - want) / tol)
    assert np.isfinite(got).all() and worst <= 1.0, worst


def test_attention_with_many_shares_and_few(torch_cuda, qctx):
    """One head over a long cache (64 shares joined) and many heads (one share), the same head's rows."""
    got, want, a = attn_case(torch_cuda, qctx, 1, 1, 2, 7000, 2, seed=11, sharp=3.0)
    assert_near(got, want, a)
    got, want, a = attn_case(torch_cuda, qctx, 4, 160, 2, 300, 2, seed=12)
    assert_near(got, want, a)


def test_a_nan_query_or_key_stays_in_its_rows(torch_cuda, qctx):
    torch = torch_cuda
    rng = np.random.default_rng(8)
    q_d, _ = bf16(torch, rng.standard_normal((1, 2, 4, 128)))
    k_d, _ = bf16(torch, rng.standard_normal((1, 2, 200, 128)))
    q_d[0, 0, 2, 100] = float("nan")
    k_d[0, 1, 150, 3] = float("nan")
    kv = stored(torch, qctx, k_d, k_d.clone().nan_to_num())
    out = torch.empty(1, 4, 256, dtype=torch.bfloat16, device="cuda")
    qctx.attention(q_d.data_ptr(), 1, 2, 4, kv, 0, None, None, 0, 0.088, out.data_ptr(), stream(torch))
    nan = np.isnan(host(out.float())).reshape(4, 2, 128)
    assert nan[2, 0].all() and not nan[[0, 1, 3], 0].any() and nan[:, 1].all()
    kv.free()


# ---------------------------------------------------------------- the expanded layer

def two_caches(torch, qctx, b, h, p, seed):
    """A 4-bit cache and a bf16 cache of the values it stands for."""
    rng = np.random.default_rng(seed)
    k_d, _ = bf16(torch, rng.standard_normal((b, h, p, 128)))
    v_d, _ = bf16(torch, rng.standard_normal((b, h, p, 128)))
    kv4 = stored(torch, qctx, k_d, v_d)
    gk, gv = read_back(torch, kv4, k_d)
    kv16 = qctx.kv_create(1, b, h, p)
    kv16.store(0, gk.data_ptr(), gv.data_ptr(), stream(torch))
    torch.cuda.synchronize()
    assert kv16.bits == 16 and (p < 200 or kv4.device_bytes() > 0)
    return kv4, kv16


@pytest.mark.parametrize("b,h,sq,p,so,padded", [(1, 8, 1536, 333, 1536, False), (2, 8, 1200, 128, 1200, True),
                                                (1, 16, 1100, 217, 1101, True), (1, 8, 2100, 40, 2100, False)])
def test_many_queries_equal_the_bf16_cache_of_the_same_values(torch_cuda, qctx, b, h, sq, p, so, padded):
    """Where the layer is expanded the attention is the bf16 cache's, bit for bit."""
    torch = torch_cuda
    caches = two_caches(torch, qctx, b, h, p, seed=sq)
    rng = np.random.default_rng(sq + 1)
    q, _ = bf16(torch, rng.standard_normal((b, h, sq, 128)))
    ko, _ = bf16(torch, rng.standard_normal((b, h, so, 128)))
    vo, _ = bf16(torch, rng.standard_normal((b, h, 128, so)))
    ok = np.ones((b, p + so), np.uint8)
    ok[-1, p // 2:p] = 0
    ok = dev(torch, ok)
    outs = []
    for kv in caches:
        out = torch.empty(b, sq, h * 128, dtype=torch.bfloat16, device="cuda")
        args = (q.data_ptr(), b, h, sq, kv, 0, ko.data_ptr() if so else None, vo.data_ptr() if so else None, so, 0.088, out.data_ptr())
        if padded:
            qctx.attention_masked(*args, key_valid=ok.data_ptr(), stream=stream(torch))
        else:
            qctx.attention(*args, stream=stream(torch))
        outs.append(host(out.view(torch.int16)))
        kv.free()
    assert np.array_equal(*outs)


@pytest.mark.parametrize("s,p", [(64, 40), (200, 333)])
def test_block_on_a_4_bit_cache(torch_cuda, qctx, s, p):
    torch = torch_cuda
    w, x, mod, pe, _, _ = make_case(21, SMALL, 2, s, p, synth.Q4_K, synth.Q6_K)
    keep = []
    blk = qctx.block_create(qimm.BlockConfig(SMALL["hidden"], SMALL["heads"], 128, SMALL["mlp"]), block_tensors(w, keep))
    x_d, mod_d, pe_d = dev(torch, x), dev(torch, mod), dev(torch, pe)
    outs = []
    for kv in two_caches(torch, qctx, 2, SMALL["heads"], p, seed=5):
        out = torch.empty_like(x_d)
        blk.forward(x_d.data_ptr(), out.data_ptr(), 2, s, mod_d.data_ptr(), pe_d.data_ptr(), kv, 0, None, None, stream(torch))
        outs.append(host(out) - x)
        kv.free()
    blk.free()
    # the same values, but the attention's fixed softmax reference is the cache's own bound
    kv_close(*outs)


# ---------------------------------------------------------------- streams, graphs, refusals

def test_replays_of_a_graph_equal_eager_calls(torch_cuda, qctx):
    """Store, few and many queries captured on a stream of their own, replayed on new inputs
    with the program's own work in between."""
    torch = torch_cuda
    b, h, p, so, sq = 2, 8, 700, 1500, 1500
    gen = torch.Generator(device="cuda").manual_seed(1)

    def draw(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(torch.bfloat16)

    k, v, q, ko, vo = draw(b, h, p, 128), draw(b, h, p, 128), draw(b, h, sq, 128), draw(b, h, so, 128), draw(b, h, 128, so)
    few, many = torch.empty(b, 3, h * 128, dtype=torch.bfloat16, device="cuda"), torch.empty(b, sq, h * 128, dtype=torch.bfloat16, device="cuda")
    kv = qctx.kv_create_q4(2, b, h, p)

    def step():
        s = stream(torch)
        kv.store(1, k.data_ptr(), v.data_ptr(), s)
        qctx.attention(q.data_ptr(), b, h, 3, kv, 1, ko.data_ptr(), vo.data_ptr(), so, 0.088, few.data_ptr(), s)
        qctx.attention(q.data_ptr(), b, h, sq, kv, 1, ko.data_ptr(), vo.data_ptr(), so, 0.088, many.data_ptr(), s)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(4):
        for t in (k, v, q):
            t.copy_(draw(*t.shape))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = few.clone(), many.clone()
        few.zero_(), many.zero_()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], few) and torch.equal(got[1], many), i
    kv.free()


def test_refusals(torch_cuda, qctx):
    torch = torch_cuda
    kv = qctx.kv_create_q4(2, 1, 2, 40)
    t = torch.zeros(2 * 40 * 128 + 8, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros(4 * 256, dtype=torch.bfloat16, device="cuda")
    a = t.data_ptr()

    def refused(status, call):
        with pytest.raises(qimm.QimmError, match=status):
            call()

    refused("QIMM_ERR_SHAPE", lambda: qctx.kv_create_q4(1, 1, 2, 40, head_dim=64))
    refused("QIMM_ERR_SHAPE", lambda: qctx.kv_create_q4(0, 1, 2, 40))
    refused("QIMM_ERR_SHAPE", lambda: qctx.kv_create_q4(1, 1, 2, -1))
    refused("QIMM_ERR_SHAPE", lambda: qctx.kv_create_q4(1, 65536, 1, 40))
    refused("QIMM_ERR_SHAPE", lambda: kv.store(2, a, a))
    refused("QIMM_ERR_ARG", lambda: kv.store(0, a + 2, a))
    refused("QIMM_ERR_ARG", lambda: kv.load(0, a, a + 8))
    refused("QIMM_ERR_ARG", lambda: kv.store(0, None, a))
    refused("QIMM_ERR_SHAPE", lambda: qctx.attention(a, 1, 3, 1, kv, 0, None, None, 0, 0.1, out.data_ptr()))
    refused("QIMM_ERR_SHAPE", lambda: qctx.attention(a, 1, 2, 1, kv, 2, None, None, 0, 0.1, out.data_ptr()))
    refused("QIMM_ERR_ARG", lambda: qctx.attention(a + 2, 1, 2, 1, kv, 0, None, None, 0, 0.1, out.data_ptr()))
    refused("QIMM_ERR_ARG", lambda: qctx.attention(a, 1, 2, 1, kv, 0, None, None, 4, 0.1, out.data_ptr()))
    refused("QIMM_ERR_SHAPE", lambda: qctx.attention_masked(a, 1, 2, 4, kv, 0, a, a, 4, 0.1, out.data_ptr(), image_ids=a))
    kv.free()
    empty = qctx.kv_create_q4(1, 1, 2, 0)
    empty.store(0, a, a)
    empty.load(0, a, a)
    refused("QIMM_ERR_SHAPE", lambda: qctx.attention(a, 1, 2, 1, empty, 0, None, None, 0, 0.1, out.data_ptr()))
    qctx.attention(a, 1, 2, 0, empty, 0, a, a, 4, 0.1, out.data_ptr())  # no query: nothing to do
    empty.free()
    torch.cuda.synchronize()
