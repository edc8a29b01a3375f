"""Adapters beside weights without bf16 rows, where the second product is a pass over the
projection's f32 sums: the sums of a bounded number of rows are held at a time, whatever the
batch, and every epilogue of the block takes its rows in parts.

Bars: a forward in parts against forwards of few entries each, which are taken whole, and against
the block over bf16 rows, whose adapters go another way: the block tests' bar (cosine 0.9999 of the
update, 2% of the largest). Products against 64 bits as in test_gpu_adapters.
"""
import numpy as np
import pytest

import oracle as O
import qimm
import synth
from gpu_util import bf16_dev, dev, host, stream
from test_gpu_adapters import Case
from test_gpu_block import SMALL, block_tensors

pytestmark = pytest.mark.gpu

SUMS = 1 << 29  # bytes


def used(torch, call):
    """The device memory that a call takes for good."""
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    call()
    torch.cuda.synchronize()
    return before - torch.cuda.mem_get_info()[0]


@pytest.fixture
def codes_ctx(torch_cuda):
    ctx = qimm.Context(0)
    ctx.set_bf16_rows(qimm.BF16_ROWS_NEVER)
    yield ctx
    torch_cuda.cuda.synchronize()
    ctx.close()


def block_with_adapters(torch, ctx, hid, mlp, seed, ranks=(16, 5)):
    """A block of Q4_K and Q6_K weights and two adapters on every projection."""
    rng = np.random.default_rng(seed)
    keep, given = [], []
    w = synth.block_weights(seed, hid, hid // 128, mlp, synth.Q4_K, synth.Q6_K)
    shapes = {"to_q": (hid, hid), "to_k": (hid, hid), "to_v": (hid, hid), "to_out": (hid, hid), "gate_up": (2 * mlp, hid),
              "mlp_out": (hid, mlp)}
    for r in ranks:
        pairs = {}
        for name, (rows, cols) in shapes.items():
            a, b = rng.standard_normal((r, cols)) / np.sqrt(cols), rng.standard_normal((rows, r)) * 0.25 / np.sqrt(r)
            pairs[name] = (qimm.BF16, rows, cols, r,
                           *(bf16_dev(torch, t)[0].cpu().view(torch.uint8).numpy().tobytes() for t in (a, b)))
        given.append((1.0, pairs))
    return ctx.block_create(qimm.BlockConfig(hid, hid // 128, 128, mlp), block_tensors(w, keep)), given


def test_scratch_of_a_block_is_bounded(torch_cuda, codes_ctx):
    """What the adapters of 256 x 1024 tokens add to the scratch: the sums of gate and up alone would
    be 1.6 GB."""
    torch = torch_cuda
    blk, given = block_with_adapters(torch, codes_ctx, SMALL["hidden"], SMALL["mlp"], 1)
    blk.reserve(256, 1024)
    blk.set_adapters(given)
    # beside the sums: of every row t (f32, up to 64 ranks of q, k and v), its two bf16 parts and the id
    assert used(torch, lambda: blk.reserve(256, 1024)) <= SUMS + 256 * 1024 * (256 + 256 + 4) + (8 << 20)
    blk.free()


def test_scratch_of_a_product_is_bounded(torch_cuda, codes_ctx):
    torch = torch_cuda
    c = Case(torch, codes_ctx, synth.Q8_0, 12288, 256, (16,), seed=1)
    codes_ctx.qmatmul_adapters_reserve(c.w, c.ad, 1, qimm.BF16)
    assert used(torch, lambda: codes_ctx.qmatmul_adapters_reserve(c.w, c.ad, 65536, qimm.BF16)) <= SUMS + (64 << 20)
    c.free()


@pytest.mark.parametrize("out_type", [qimm.F32, qimm.BF16])
@pytest.mark.parametrize("m,n,k,t", [(40000, 256, 512, synth.Q8_0), (16385, 512, 256, synth.Q4_K), (33000, 12288, 256, synth.Q6_K)])
def test_products_in_parts(torch_cuda, codes_ctx, m, n, k, t, out_type):
    torch = torch_cuda
    c = Case(torch, codes_ctx, t, n, k, (16, 40), seed=m)
    x = torch.randn(m, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(torch.bfloat16)
    ids = (np.arange(m) * 7 // m) % 3 - 1
    got = c.call(x, m, dev(torch, ids.astype(np.int32)), out_type)
    # around the parts' ends (8448 and 13568 rows each) and in between
    at = np.unique(np.r_[0:3, 8446:8450, 13566:13570, 16894:16898, 25342:25346, 27134:27138, m - 3:m, np.arange(0, m, 977)])
    at = at[at < m]
    rows = torch.from_numpy(at).cuda()
    c.check(host(got[rows].float()), host(x[rows].float()), ids[at], out_type)
    c.free()


def forward(torch, blk, x, mod, pe, ids):
    out = torch.empty_like(x)
    blk.set_adapter_ids(ids.data_ptr())
    blk.forward(x.data_ptr(), out.data_ptr(), x.shape[0], x.shape[1], mod.data_ptr(), pe.data_ptr(), None, 0, None, None,
                stream(torch))
    torch.cuda.synchronize()
    return out


def assert_close(got, want, x):
    """Cosine of the updates and the largest difference, on the device."""
    a, b = (got - x).double().flatten(), (want - x).double().flatten()
    cos, rel = float(a @ b / (a.norm() * b.norm())), float((got - want).abs().max() / want.abs().max())
    assert cos >= 0.9999 and rel <= 2e-2, (cos, rel)


def inputs(torch, b, s, hid, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(b, s, hid, device="cuda", generator=gen)
    mod = torch.randn(b, 1, 4 * hid, device="cuda", generator=gen) * 0.5
    rows = max(i for i in range(1, 100) if s % i == 0)
    return x, mod, dev(torch, O.rope_table([(1, rows, s // rows)], [1] * s)), torch.arange(b, device="cuda", dtype=torch.int32) % 3 - 1


@pytest.mark.parametrize("act", [qimm.ACT_BF16, qimm.ACT_CANDLE])
@pytest.mark.parametrize("b,s,group", [(1366, 1024, 16), (150, 200, 50)])
def test_a_forward_in_parts_equals_its_entries(torch_cuda, codes_ctx, b, s, group, act):
    """1366 x 1024 tokens have more than 2^31 sums of gate and up; 150 x 200 leave a last part of
    fewer rows in every projection."""
    torch, hid = torch_cuda, SMALL["hidden"]
    blk, given = block_with_adapters(torch, codes_ctx, hid, SMALL["mlp"], b)
    blk.set_adapters(given)
    blk.set_act_mode(act)
    x, mod, pe, ids = inputs(torch, b, s, hid, b)
    got = forward(torch, blk, x, mod, pe, ids)
    for i in range(0, b, group):
        n = min(group, b - i)
        one = forward(torch, blk, x[i:i + n], mod[i:i + n], pe, ids[i:i + n].clone())
        assert_close(got[i:i + n], one, x[i:i + n])
    none = forward(torch, blk, x[:9], mod[:9], pe, torch.full((9,), -1, dtype=torch.int32, device="cuda"))
    assert not torch.equal(none, got[:9]) and float((none - got[:9]).norm() / (none - x[:9]).norm()) > 0.05
    blk.free()


@pytest.mark.parametrize("mod_rows", ["one", "each"])
def test_a_sequence_longer_than_a_part(torch_cuda, codes_ctx, mod_rows):
    """Every projection of one sequence of 20008 tokens in two parts, the second from position 13568 on."""
    torch = torch_cuda
    b, s, hid, mlp = 2, 20008, SMALL["hidden"], SMALL["mlp"]
    x, mod, pe, _ = inputs(torch, b, s, hid, 3)
    ids = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    rows = 1 if mod_rows == "one" else s
    if rows > 1:
        mod = mod + 0.1 * torch.randn(b, s, 4 * hid, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    outs = []
    rows_ctx = qimm.Context(0)
    rows_ctx.set_bf16_rows(qimm.BF16_ROWS_ALWAYS)
    for ctx in (codes_ctx, rows_ctx):
        blk, given = block_with_adapters(torch, ctx, hid, mlp, 7)
        blk.set_adapters(given)
        blk.set_act_mode(qimm.ACT_BF16)
        blk.set_adapter_ids(ids.data_ptr())
        out = torch.empty_like(x)
        k, v = (torch.empty(b, hid // 128, s, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        if rows == 1:
            blk.forward(x.data_ptr(), out.data_ptr(), b, s, mod.data_ptr(), pe.data_ptr(), None, 0, k.data_ptr(), v.data_ptr(),
                        stream(torch))
        else:
            blk.forward_masked(x.data_ptr(), out.data_ptr(), b, s, mod.data_ptr(), rows, pe.data_ptr(), k_out=k.data_ptr(),
                               v_out=v.data_ptr(), stream=stream(torch))
        torch.cuda.synchronize()
        outs.append((out, k.float(), v.float()))
        blk.free()
    rows_ctx.close()
    assert_close(outs[0][0], outs[1][0], x)
    for i in (1, 2):
        assert_close(outs[0][i], outs[1][i], 0.0)
