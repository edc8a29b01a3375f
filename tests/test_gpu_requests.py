"""The 4-bit prefix cache and the low-rank adapters as a batched step uses them together, and
the 4-bit cache under the model's prefix fill and step."""
import numpy as np
import pytest

import kv4_ref
import oracle as O
import qimm
import synth
from gpu_util import bf16_dev, cos_sim, dev, host, kv_close, max_abs_rel, stream
from test_gpu_block import SMALL
from test_gpu_step import CH, JD, Built, _prefix_case, model_weights, t_sin_dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("text,b,pad", [(21, 2, 0), (203, 2, 60), (603, 1, 0)])
def test_prefix_fill_into_a_4_bit_cache(torch_cuda, qctx, text, b, pad):
    """Every layer stands for the format's values of the bf16 cache's (a fill's keys do not depend
    on the cache), hidden tokens for zeros; a step over it is a step over those values."""
    torch = torch_cuda
    layers, rng, h = 2, np.random.default_rng(text), SMALL["heads"]
    g, blocks = model_weights(51, layers)
    mdl = Built(qctx, g, blocks)
    txt_d = dev(torch, rng.standard_normal((b, text, JD)).astype(np.float32))
    pe = O.rope_table([(1, 4, 8)], [0] * text + [1] * 32)
    pe_d, step_pe = dev(torch, pe[:text]), dev(torch, np.ascontiguousarray(pe[text:]))
    ids_d = dev(torch, np.full(text, -1, np.int32))
    ok = np.ones((b, text + 32), np.uint8)
    ok[-1, text - pad:text] = 0
    fill_ok, step_ok = dev(torch, np.ascontiguousarray(ok[:, :text])), dev(torch, ok)
    lat, tsd = dev(torch, rng.standard_normal((b, 32, CH)).astype(np.float32)), t_sin_dev(torch, qctx, [0.4] * b)
    loaded, caches = [], []
    for make in (qctx.kv_create, qctx.kv_create_q4):
        kv = make(layers, b, h, text)
        mdl.model.prefix_fill(txt_d.data_ptr(), text, None, 0, b, qimm.joint_layout_pieces(text), ids_d.data_ptr(),
                              fill_ok.data_ptr() if pad else None, pe_d.data_ptr(), kv, stream(torch))
        for i in range(layers):
            k, v = (torch.empty((b, h, text, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
            kv.load(i, k.data_ptr(), v.data_ptr(), stream(torch))
            loaded.append((k, v))
        caches.append(kv)
    hid = dev(torch, ok[:, None, :text, None] == 0)
    for (k16, v16), (k4, v4) in zip(loaded[:layers], loaded[layers:]):
        wk, wv = kv4_ref.near_kv(host(k16.float().masked_fill(hid, 0)), host(v16.float().masked_fill(hid, 0)))
        assert np.array_equal(host(k4.float()), wk) and np.array_equal(host(v4.float()), wv)
    for i, (k4, v4) in enumerate(loaded[layers:]):
        caches[0].store(i, k4.data_ptr(), v4.data_ptr(), stream(torch))
    out = []
    for kv in caches:
        pred = torch.empty_like(lat)
        mdl.model.forward(lat.data_ptr(), b, 32, tsd.data_ptr(), step_pe.data_ptr(), kv, pred.data_ptr(),
                          step_ok.data_ptr() if pad else None, stream(torch))
        out.append(host(pred))
        kv.free()
    mdl.free()
    assert np.isfinite(out[1]).all() and cos_sim(out[1], out[0]) >= 0.99999 and max_abs_rel(out[1], out[0]) <= 2e-2


def test_prefix_fill_with_an_image_into_a_4_bit_cache(torch_cuda, qctx):
    torch = torch_cuda
    b, layers = 2, 2
    g, blocks = model_weights(31, layers)
    slots, ids, P, pe, pieces, txt, cond, key_valid = _prefix_case(b, layers, 6)
    mdl = Built(qctx, g, blocks)
    txt_d, cond_d, pe_d = dev(torch, txt), dev(torch, cond), dev(torch, pe)
    ids_d, ok_d = dev(torch, np.array(ids, np.int32)), dev(torch, key_valid)
    got = []
    for make in (qctx.kv_create, qctx.kv_create_q4):
        kv = make(layers, b, SMALL["heads"], P)
        mdl.model.prefix_fill(txt_d.data_ptr(), len(slots), cond_d.data_ptr(), 16, b, pieces, ids_d.data_ptr(),
                              ok_d.data_ptr(), pe_d.data_ptr(), kv, stream(torch))
        k, v = (torch.empty((b, SMALL["heads"], P, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        kv.load(1, k.data_ptr(), v.data_ptr(), stream(torch))
        got.append((host(k.float()), host(v.float())))
        kv.free()
    mdl.free()
    seen = key_valid[:, None, :, None] != 0
    want = kv4_ref.near_kv(*(np.where(seen, x, 0) for x in got[0]))
    assert np.array_equal(got[1][0], want[0]) and np.array_equal(got[1][1], want[1])


@pytest.mark.parametrize("s,p,pad", [(1, 50, 0), (24, 333, 100), (300, 217, 60)])
def test_adapters_cache_and_attention_together(torch_cuda, qctx, s, p, pad):
    """Three requests, two of them with adapters of their own: q, k and v of the prompts into a
    4-bit cache, of the step's tokens beside it, the attention over both, and the output
    projection, against the same in 64 bits. The intermediate bf16 values may round to the other
    neighbour where a sum differs in its last bits, and with them a code of the cache: the whole
    is held to the block's bar (cosine 0.9999, 2% of the largest)."""
    torch = torch_cuda
    rng = np.random.default_rng(s + p)
    b, heads, hid, ranks = 3, 4, 512, (16, 5)
    req = np.array([1, -1, 0])
    ws, ads, ref = {}, {}, {}
    for name in ("q", "k", "v", "o"):
        _, raw, _, _ = synth.weight(rng, synth.Q8_0, hid, hid, 0.05)
        wv = O.bf16_round(O.dequantize(synth.Q8_0, raw, hid * hid).reshape(hid, hid)).astype(np.float64)
        ws[name] = qctx.upload(synth.Q8_0, hid, hid, raw.tobytes())
        given, deltas = [], []
        for r in ranks:
            ad, av = bf16_dev(torch, rng.standard_normal((r, hid)) / np.sqrt(hid))
            bd, bv = bf16_dev(torch, rng.standard_normal((hid, r)) * 0.2)
            given.append((1.5 / r, qimm.BF16, *(t.cpu().view(torch.uint8).numpy().tobytes() for t in (ad, bd))))
            deltas.append(1.5 / r * bv.astype(np.float64) @ av.astype(np.float64))
        ads[name] = qctx.adapters_create(hid, hid, given)
        ref[name] = [wv + (deltas[i] if i >= 0 else 0.0) for i in req]  # each request's own merged weight
    norm = 1 + 0.1 * rng.standard_normal(128).astype(np.float32)
    norm_d = dev(torch, norm)
    pe = O.rope_table([(1, 1, s)], [0] * p + [1] * s)

    def project(name, x_d, rows, out_type):
        y = torch.empty(b * rows, hid, dtype=torch.float32 if out_type == qimm.F32 else torch.bfloat16, device="cuda")
        ids = dev(torch, req.repeat(rows).astype(np.int32))
        qctx.qmatmul_adapters(ws[name], ads[name], ids.data_ptr(), x_d.data_ptr(), b * rows, hid, y.data_ptr(), out_type, stream(torch))
        return y

    def rope_ref(y, table):  # per-head norm, then rotation of the pairs; rounded to bf16
        y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + 1e-6) * norm
        c, sn = table[:, 0::2].astype(np.float64), table[:, 1::2].astype(np.float64)
        c, sn = c[None, :, None, :], sn[None, :, None, :]
        out = np.empty_like(y)
        out[..., 0::2] = y[..., 0::2] * c - y[..., 1::2] * sn
        out[..., 1::2] = y[..., 0::2] * sn + y[..., 1::2] * c
        return O.bf16_round(out.astype(np.float32)).astype(np.float64).transpose(0, 2, 1, 3)

    def heads_ref(name, x):
        return np.stack([x[i].astype(np.float64) @ ref[name][i].T for i in range(b)]).reshape(b, -1, heads, 128)

    def roped(name, x_d, rows, table):
        out = torch.empty(b, heads, rows, 128, dtype=torch.bfloat16, device="cuda")
        y, pe_d = project(name, x_d, rows, qimm.F32), dev(torch, table)
        qctx.qk_norm_rope(y.data_ptr(), b, rows, heads, norm_d.data_ptr(), pe_d.data_ptr(), out.data_ptr(), stream(torch))
        torch.cuda.synchronize()
        return out

    xp_d, xp = bf16_dev(torch, rng.standard_normal((b, p, hid)))
    xs_d, xs = bf16_dev(torch, rng.standard_normal((b, s, hid)))
    pe_p, pe_s = np.ascontiguousarray(pe[:p]), np.ascontiguousarray(pe[p:])
    kp = roped("k", xp_d, p, pe_p)
    vp = project("v", xp_d, p, qimm.F32).reshape(b, p, heads, 128).permute(0, 2, 1, 3).contiguous().to(torch.bfloat16)
    kv = qctx.kv_create_q4(1, b, heads, p)
    kv.store(0, kp.data_ptr(), vp.data_ptr(), stream(torch))
    q, k = roped("q", xs_d, s, pe_s), roped("k", xs_d, s, pe_s)
    vt = torch.empty(b, heads, 128, s, dtype=torch.bfloat16, device="cuda")
    vs = project("v", xs_d, s, qimm.F32)
    qctx.v_transpose(vs.data_ptr(), b, s, heads, vt.data_ptr(), stream(torch))
    ok = np.ones((b, p + s), np.uint8)
    ok[-1, p - pad:p] = 0
    ok_d, att = dev(torch, ok), torch.empty(b, s, hid, dtype=torch.bfloat16, device="cuda")
    qctx.attention_masked(q.data_ptr(), b, heads, s, kv, 0, k.data_ptr(), vt.data_ptr(), s, 128 ** -0.5, att.data_ptr(),
                          key_valid=ok_d.data_ptr(), stream=stream(torch))
    got = host(project("o", att, s, qimm.F32)).reshape(b, s, hid)

    def rounded(y):
        return O.bf16_round(y.astype(np.float32)).astype(np.float64).transpose(0, 2, 1, 3)

    rk, rv = kv4_ref.near_kv(rope_ref(heads_ref("k", xp), pe_p), rounded(heads_ref("v", xp)))
    kk = np.concatenate([rk, rope_ref(heads_ref("k", xs), pe_s)], 2)
    vv = np.concatenate([rv, rounded(heads_ref("v", xs))], 2)
    a, _ = kv4_ref.attention(rope_ref(heads_ref("q", xs), pe_s), kk, vv, 128 ** -0.5, ok)
    want = np.stack([O.bf16_round(a[i].reshape(s, hid).astype(np.float32)).astype(np.float64) @ ref["o"][i].T for i in range(b)])
    kv_close(got, want)
    kv.free()
    for x in (*ws.values(), *ads.values()):
        x.free()
