"""Adapters in the block at a size whose products take tiles of 256 tokens: their further k steps
under every epilogue of the block, tiles with the rows of two requests, and a last partial tile.
Bars as in test_gpu_block_adapters, on the entries that the oracle computes."""
import numpy as np
import pytest

import oracle as O
import qimm
import synth
from gpu_util import bf16_dev, cos_sim, dev, host, max_abs_rel, stream
from test_gpu_block import block_tensors, make_case
from test_gpu_block_adapters import ALL, merged

pytestmark = pytest.mark.gpu

CFG = dict(hidden=2048, heads=16, head_dim=128, mlp=6144)
HID, MLP = CFG["hidden"], CFG["mlp"]
SHAPES = {"to_q": (HID, HID), "to_k": (HID, HID), "to_v": (HID, HID), "to_out": (HID, HID), "gate_up": (2 * MLP, HID),
          "gate_layer": (MLP, HID), "mlp_out": (HID, MLP)}


def test_block_with_adapters_on_large_tiles(torch_cuda, qctx):
    torch = torch_cuda
    b, s, at = 41, 200, (0, 20, 40)
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    for t, rows, cols in ((synth.Q4_K, 3 * HID, HID), (synth.Q4_K, HID, HID), (synth.Q4_K, 2 * MLP, HID), (synth.Q6_K, HID, MLP)):
        route = qimm.qmatmul_route(t, rows, cols, b * s, cus)
        assert route.kernel == qimm.GEMM_BF16_ROWS and route.splits == 1 and route.large_tiles > 0
    w, x, mod, pe, _, _ = make_case(b, CFG, b, s, 0, synth.Q4_K, synth.Q6_K)
    rng = np.random.default_rng(1)
    given, deltas = [], []
    for i, (names, rank) in enumerate(((ALL, 16), (("to_q", "to_v", "gate_layer"), 64), (("to_k", "to_out", "mlp_out"), 5))):
        scale, pairs, delta = 0.5 + i, {}, {}
        for name in names:
            rows, cols = SHAPES[name]
            a_d, a = bf16_dev(torch, rng.standard_normal((rank, cols)) / np.sqrt(cols))
            b_d, bv = bf16_dev(torch, rng.standard_normal((rows, rank)) * 0.25 / np.sqrt(rank))
            pairs[name] = (qimm.BF16, rows, cols, rank, *(t.cpu().view(torch.uint8).numpy().tobytes() for t in (a_d, b_d)))
            delta[name] = scale * bv.astype(np.float64) @ a.astype(np.float64)
        given.append((scale, pairs))
        deltas.append(delta)
    ids = np.arange(b) % 4 - 1
    ids[list(at)] = (0, 1, 2)
    keep = []
    blk = qctx.block_create(qimm.BlockConfig(HID, CFG["heads"], 128, MLP), block_tensors(w, keep))
    blk.set_adapters(given)
    ids_d, x_d, mod_d, pe_d = dev(torch, ids.astype(np.int32)), dev(torch, x), dev(torch, mod), dev(torch, pe)

    def forward(act, with_ids):
        blk.set_act_mode(act)
        blk.set_adapter_ids(ids_d.data_ptr() if with_ids else None)
        out = torch.empty_like(x_d)
        blk.forward(x_d.data_ptr(), out.data_ptr(), b, s, mod_d.data_ptr(), pe_d.data_ptr(), None, 0, None, None, stream(torch))
        return host(out)

    got_b, got_c, plain_c = forward(qimm.ACT_BF16, True), forward(qimm.ACT_CANDLE, True), forward(qimm.ACT_CANDLE, False)
    blk.free()
    for i in at:
        xi = x[i:i + 1]
        want, base = (O.block_forward(CFG, merged(w, d), xi, mod[i:i + 1], pe, None, None, mode=O.EXACT)[0]
                      for d in (deltas[ids[i]], {}))
        ub, uc, u0 = (cos_sim(g[i:i + 1] - xi, r - xi) for g, r in ((got_b, want), (got_c, want), (plain_c, base)))
        print(f"entry {i}: bf16 {cos_sim(got_b[i:i + 1], want):.7f} update {ub:.7f}; candle update {uc:.7f}, without "
              f"adapters {u0:.7f}; the adapters' own {cos_sim(base - xi, want - xi):.4f}", flush=True)
        assert cos_sim(got_b[i:i + 1], want) >= 0.9999 and ub >= 0.9999 and max_abs_rel(got_b[i:i + 1], want) <= 2e-2
        assert 1 - uc <= 2 * (1 - u0) + 1e-5
        assert cos_sim(base - xi, want - xi) < 0.999  # they matter
