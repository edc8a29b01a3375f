"""Low-rank adapters in the block (qimm_block_set_adapters) and under the model.

Bars: the bf16 activation mode against the oracle's exact mode on weights with each request's own
adapter added to them (f32), at the block tests' bar: cosine 0.9999 on the output and on the
update, 2% of the largest. The candle mode, whose int8 rounding no merged weight reproduces, stays
as close to that as the block without adapters stays to its own exact result (twice the distance
1 - cosine of the update).
"""
import numpy as np
import pytest

import oracle as O
import qimm
import synth
from gpu_util import bf16_dev, cos_sim, dev, host, kv_close, max_abs_rel, stream
from test_gpu_block import SMALL, block_tensors, make_case
from test_gpu_step import CH, JD, Built, model_weights, t_sin_dev

pytestmark = pytest.mark.gpu

HID, MLP = SMALL["hidden"], SMALL["mlp"]
SHAPES = {"to_q": (HID, HID), "to_k": (HID, HID), "to_v": (HID, HID), "to_out": (HID, HID), "gate_up": (2 * MLP, HID),
          "proj": (MLP, HID), "gate_layer": (MLP, HID), "mlp_out": (HID, MLP)}


def make_adapters(torch, rng, which):
    """[(scale, {projection: tensors})] for the binding and their deltas [{projection: f64}]."""
    given, deltas = [], []
    for i, names in enumerate(which):
        scale, pairs, delta = 0.5 + i, {}, {}
        for j, name in enumerate(names):
            rows, cols = SHAPES[name]
            rank = (4, 16, 33, 1)[(i + j) % 4]
            a_d, a = bf16_dev(torch, rng.standard_normal((rank, cols)) / np.sqrt(cols))
            b_d, b = bf16_dev(torch, rng.standard_normal((rows, rank)) * 0.25 / np.sqrt(rank))
            pairs[name] = (qimm.BF16, rows, cols, rank, *(t.cpu().view(torch.uint8).numpy().tobytes() for t in (a_d, b_d)))
            delta[name] = scale * b.astype(np.float64) @ a.astype(np.float64)
        given.append((scale, pairs))
        deltas.append(delta)
    return given, deltas


def merged(w, delta):
    """The block's weights as f32 tensors with an adapter's deltas added."""
    out = {}
    for name, v in w.items():
        if not isinstance(v, tuple):
            out[name] = v
            continue
        t, data, rows, cols = v
        x = O.dequantize(t, data, rows * cols).reshape(rows, cols).astype(np.float64)
        d = delta.get("mlp_out" if name == "down" else name)
        if name == "gate_up" and d is None and ("gate_layer" in delta or "proj" in delta):
            d = np.concatenate([delta.get(n, np.zeros((rows // 2, cols))) for n in ("gate_layer", "proj")])
        if d is not None:
            x = x + d
        x = np.ascontiguousarray(x.astype(np.float32))
        out[name] = (synth.F32, x.view(np.uint8).reshape(-1), rows, cols)
    return out


ALL = ("to_q", "to_k", "to_v", "to_out", "gate_up", "mlp_out")


@pytest.mark.parametrize("codes_only", [False, True])
@pytest.mark.parametrize("s", [16, 40, 400])
@pytest.mark.parametrize("types,fused,which", [
    ((synth.BF16, synth.BF16), True, (("to_q", "to_v", "to_out"), ALL)),
    ((synth.Q4_K, synth.Q6_K), True, (("to_k", "gate_layer"), ALL)),
    ((synth.Q8_0, synth.Q8_0), False, (("proj", "mlp_out"), ("to_q", "to_k", "to_v", "gate_layer", "proj"))),
    ("mixed", True, (ALL, ("to_v", "gate_up")))])
def test_block_with_adapters(torch_cuda, qctx, qctx_codes, types, fused, which, s, codes_only):
    """Three requests: the second adapter, none, the first; rows by themselves, the pass and the
    steps; q/k/v fused or of their own types."""
    torch = torch_cuda
    ctx = qctx_codes if codes_only else qctx
    b, p = 3, 24
    attn, down = (synth.Q8_0, synth.Q6_K) if types == "mixed" else types
    w, x, mod, pe, kpre, vpre = make_case(s, SMALL, b, s, p, attn, down, fused)
    if types == "mixed":
        w["to_v"] = synth.weight(np.random.default_rng(9), synth.Q6_K, HID, HID, 0.02)
    given, deltas = make_adapters(torch, np.random.default_rng(s + 1), which)
    ids = [1, -1, 0]
    keep = []
    blk = ctx.block_create(qimm.BlockConfig(HID, SMALL["heads"], 128, MLP), block_tensors(w, keep))
    blk.set_adapters(given)
    ids_d, x_d, mod_d, pe_d = dev(torch, np.array(ids, np.int32)), dev(torch, x), dev(torch, mod), dev(torch, pe)
    k_d, v_d = dev(torch, kpre.view(np.int16)), dev(torch, vpre.view(np.int16))
    kv = ctx.kv_create(1, b, SMALL["heads"], p)
    kv.store(0, k_d.data_ptr(), v_d.data_ptr(), stream(torch))

    def forward(act, with_ids):
        blk.set_act_mode(act)
        blk.set_adapter_ids(ids_d.data_ptr() if with_ids else None)
        out = torch.empty_like(x_d)
        blk.forward(x_d.data_ptr(), out.data_ptr(), b, s, mod_d.data_ptr(), pe_d.data_ptr(), kv, 0, None, None, stream(torch))
        return host(out)

    got_b, got_c, plain_c = forward(qimm.ACT_BF16, True), forward(qimm.ACT_CANDLE, True), forward(qimm.ACT_CANDLE, False)
    blk.set_adapters([])
    blk.set_adapter_ids(ids_d.data_ptr())
    blk.set_act_mode(qimm.ACT_CANDLE)
    out = torch.empty_like(x_d)
    blk.forward(x_d.data_ptr(), out.data_ptr(), b, s, mod_d.data_ptr(), pe_d.data_ptr(), kv, 0, None, None, stream(torch))
    assert np.array_equal(host(out), plain_c)  # no adapters: the block as it was
    blk.free()
    kv.free()
    want, base = np.empty_like(x), np.empty_like(x)
    for i, a in enumerate(ids):
        for dst, delta in ((want, deltas[a] if a >= 0 else {}), (base, {})):
            dst[i:i + 1] = O.block_forward(SMALL, merged(w, delta), x[i:i + 1], mod[i:i + 1], pe, kpre[i:i + 1], vpre[i:i + 1],
                                           mode=O.EXACT)[0]
    ub, uc, u0 = (cos_sim(g - x, r - x) for g, r in ((got_b, want), (got_c, want), (plain_c, base)))
    print(f"bf16 {cos_sim(got_b, want):.7f} update {ub:.7f}; candle update {uc:.7f}, without adapters {u0:.7f}; "
          f"the adapters' own {cos_sim(base - x, want - x):.4f}", flush=True)
    assert cos_sim(got_b, want) >= 0.9999 and ub >= 0.9999 and max_abs_rel(got_b, want) <= 2e-2
    assert 1 - uc <= 2 * (1 - u0) + 1e-5
    assert cos_sim(base - x, want - x) < 0.995  # they matter


def test_model_with_adapters_takes_each_request_s_own(torch_cuda, qctx):
    """Prefix fill and step of a batch equal those of its requests alone; the prompt's keys go
    through the adapters too."""
    torch = torch_cuda
    layers, text, s, rng = 2, 40, 32, np.random.default_rng(3)
    g, blocks = model_weights(51, layers)
    mdl = Built(qctx, g, blocks)
    for blk in mdl.blocks:
        blk.set_adapters(make_adapters(torch, rng, (ALL, ("to_q", "to_v")))[0])
    txt, lat = rng.standard_normal((2, text, JD)).astype(np.float32), rng.standard_normal((2, s, CH)).astype(np.float32)
    pe = O.rope_table([(1, 4, 8)], [0] * text + [1] * s)
    pe_d, step_pe, ids_d = dev(torch, pe[:text]), dev(torch, np.ascontiguousarray(pe[text:])), dev(torch, np.full(text, -1, np.int32))

    def run(rows, ads, make):
        b = len(rows)
        req = dev(torch, np.array(ads, np.int32))
        for blk in mdl.blocks:
            blk.set_adapter_ids(req.data_ptr())
        kv = make(layers, b, SMALL["heads"], text)
        t, x, pred = dev(torch, txt[rows]), dev(torch, lat[rows]), torch.empty((b, s, CH), dtype=torch.float32, device="cuda")
        mdl.model.prefix_fill(t.data_ptr(), text, None, 0, b, qimm.joint_layout_pieces(text), ids_d.data_ptr(), None,
                              pe_d.data_ptr(), kv, stream(torch))
        sin = t_sin_dev(torch, qctx, [0.4] * b)
        mdl.model.forward(x.data_ptr(), b, s, sin.data_ptr(), step_pe.data_ptr(), kv, pred.data_ptr(), None, stream(torch))
        out = host(pred)
        kv.free()
        return out

    for make in (qctx.kv_create, qctx.kv_create_q4):
        both = run([0, 1], [1, 0], make)
        for i, a in ((0, 1), (1, 0)):
            alone, other = run([i], [a], make), run([i], [1 - a], make)
            kv_close(both[i:i + 1], alone)
            # the blocks' part of this model's output is small: its own adapter's result is
            # nearer than the other's by far
            assert np.abs(both[i] - alone[0]).max() * 10 < np.abs(both[i] - other[0]).max()
    for blk in mdl.blocks:
        blk.set_adapter_ids(None)
    mdl.free()


def test_reserved_forwards_with_adapters_do_not_allocate_and_replay(torch_cuda, qctx):
    torch = torch_cuda
    b, s = 2, 600
    w, x, mod, pe, _, _ = make_case(5, SMALL, b, s, 0, synth.Q4_K, synth.Q6_K)
    ctx, keep = qimm.Context(0), []
    blk = ctx.block_create(qimm.BlockConfig(HID, SMALL["heads"], 128, MLP), block_tensors(w, keep))
    blk.set_adapters(make_adapters(torch, np.random.default_rng(1), (ALL, ALL))[0])
    blk.reserve(b, s)
    ids, x_d, mod_d, pe_d = dev(torch, np.array([0, 1], np.int32)), dev(torch, x), dev(torch, mod), dev(torch, pe)
    blk.set_adapter_ids(ids.data_ptr())
    for n in (s, 30, 200):
        out = torch.empty(b, n, HID, device="cuda")
        x_n, pe_n = x_d[:, :n].contiguous(), pe_d[:n].contiguous()

        def step():
            blk.forward(x_n.data_ptr(), out.data_ptr(), b, n, mod_d.data_ptr(), pe_n.data_ptr(), None, 0, None, None, stream(torch))

        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):  # the first forward of its size: no allocation may be needed
            step()
        for r in range(3):
            ids.copy_(torch.tensor([r % 2, -1 if r == 2 else 1], dtype=torch.int32))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            out.zero_()
            step()
            torch.cuda.synchronize()
            assert torch.equal(got, out), (n, r)
        del graph
    blk.free()
    ctx.close()


def test_refusals(torch_cuda, qctx):
    torch = torch_cuda
    w = make_case(5, SMALL, 1, 4, 0, synth.Q8_0, synth.Q8_0)[0]
    keep = []
    blk = qctx.block_create(qimm.BlockConfig(HID, SMALL["heads"], 128, MLP), block_tensors(w, keep))
    good = (qimm.BF16, HID, HID, 2, bytes(2 * HID * 2), bytes(HID * 2 * 2))
    wide = (qimm.BF16, HID, HID, 600, bytes(600 * HID * 2), bytes(HID * 600 * 2))
    gate = (qimm.BF16, MLP, HID, 2, bytes(2 * HID * 2), bytes(MLP * 2 * 2))
    both = (qimm.BF16, 2 * MLP, HID, 2, bytes(2 * HID * 2), bytes(2 * MLP * 2 * 2))

    def refused(status, pairs):
        with pytest.raises(qimm.QimmError, match=status):
            blk.set_adapters([(1.0, {"to_q": good}), (1.0, pairs)])

    refused("QIMM_ERR_SHAPE", {"to_q": gate})
    refused("QIMM_ERR_SHAPE", {"to_out": good[:3] + (1,) + good[4:]})
    refused("QIMM_ERR_TYPE", {"to_out": (qimm.Q8_0,) + good[1:]})
    refused("QIMM_ERR_ARG", {"to_out": good[:5] + (None,)})
    refused("QIMM_ERR_ARG", {"gate_up": both, "proj": gate})
    refused("QIMM_ERR_SHAPE", {"to_q": wide, "to_k": wide})
    refused("QIMM_ERR_ARG", {"to_v": good[:4] + (b"\x80\x7f" * (2 * HID), good[5])})
    with pytest.raises(qimm.QimmError, match="QIMM_ERR_ARG"):
        blk.set_adapter_ids(2)
    blk.set_adapters([(1.0, {})])
    blk.set_adapters([])
    blk.free()
