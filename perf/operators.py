"""The operators of a batched step over many requests: a prefix K/V cache held in 4 bits, the
attention that reads it, and low-rank adapters beside a shared projection. Each in its plain form
(elementary torch operations in 32 bits), through the public binding, and in 64 bits.

A case is a dict of plain values; its "kind" names the call:

- "store": one layer of keys and values stored into a 4-bit prefix cache and read back as bf16
  (KvCache.store and load), as the prefix fill writes it and a host program saves it;
- "attn": the attention of queries over [4-bit prefix ; own bf16 keys], over the cache alone
  (own 0: cross attention to the prompt's states), and with padded prompts (key validity);
- "lora": y = x W^T + s (x A^T) B^T, each row with the adapter of its own request, or none
  (Context.qmatmul_adapters) beside a quantized or bf16 projection of the block.

The cache's format: blocks of 32 values, e2m1 codes and one power of two 2^s each; along a key's
dimensions for K, along 32 consecutive keys of one dimension for V. s is the smallest integer with
max|x| <= 7 2^s, within [-120, 125]; a value stands for the nearest of
+-{0, 0.5, 1, 1.5, 2, 3, 4, 6} 2^s, ties to the even code.

Sizes: hidden 4096 (32 heads of 128) with MLP 12288 is the model's block; an image of H x W pixels
is H/16 x W/16 tokens; prompts have any number of tokens, a reference image adds its own.
"""
import math
import os
import sys
import weakref

import torch

own = False

HD = 128


def listed():
    return [
        # the prefix fill of a text-to-image prompt writes a layer
        {"name": "store_prompt_217", "kind": "store", "batch": 1, "heads": 32, "prefix": 217},
        # an edit with two 1024x1024 reference images
        {"name": "store_edit_8395", "kind": "store", "batch": 1, "heads": 32, "prefix": 8395},
        # the smallest call: one token over an ordinary prompt
        {"name": "attn_token_333", "kind": "attn", "batch": 1, "heads": 32, "prefix": 333, "sq": 1, "own": 1,
         "padded": False},
        # one token of each of eight requests over long multi-reference prefixes, padded to the longest
        {"name": "attn_tokens_b8_16640", "kind": "attn", "batch": 8, "heads": 32, "prefix": 16640, "sq": 1,
         "own": 1, "padded": True},
        # a few tokens (cross attention of learned queries) to the prompt's states alone
        {"name": "attn_cross_37_4299", "kind": "attn", "batch": 2, "heads": 32, "prefix": 4299, "sq": 37, "own": 0,
         "padded": True},
        # 512x512 under guidance: both prompts in one batch, the shorter one padded
        {"name": "attn_512_cfg", "kind": "attn", "batch": 2, "heads": 32, "prefix": 150, "sq": 1024, "own": 1024,
         "padded": True},
        # a 1024x1024 edit step: image tokens over prompt, reference image and themselves
        {"name": "attn_1024_edit", "kind": "attn", "batch": 1, "heads": 32, "prefix": 4299, "sq": 4096, "own": 4096,
         "padded": False},
        # one token of one request through the attention's output projection
        {"name": "lora_token_q4k", "kind": "lora", "wt": "q4_k", "rows": 4096, "cols": 4096, "m": 1, "requests": 1,
         "adapters": 1, "rank": 16, "out": "bf16"},
        # single tokens of many requests, their adapters of different ranks, some without one
        {"name": "lora_tokens_48_q8", "kind": "lora", "wt": "q8_0", "rows": 12288, "cols": 4096, "m": 48,
         "requests": 48, "adapters": 12, "rank": 32, "out": "bf16"},
        # two 256x256 images of an odd number of rows through a bf16 projection, f32 sums kept
        {"name": "lora_257x2_bf16", "kind": "lora", "wt": "bf16", "rows": 4096, "cols": 4096, "m": 514,
         "requests": 2, "adapters": 2, "rank": 16, "out": "f32"},
        # the MLP's down projection at 1024x1024, one request, a wide adapter
        {"name": "lora_1024_down_q4k", "kind": "lora", "wt": "q4_k", "rows": 4096, "cols": 12288, "m": 4096,
         "requests": 1, "adapters": 1, "rank": 64, "out": "bf16"},
        # q/k/v of four 1024x1024 requests at once, three adapters and one request without
        {"name": "lora_1024x4_qkv_q4k", "kind": "lora", "wt": "q4_k", "rows": 12288, "cols": 4096, "m": 16384,
         "requests": 4, "adapters": 3, "rank": 32, "out": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    while True:
        kind = rng.choice(["store", "attn", "attn", "lora", "lora"])
        if kind == "store":
            c = {"kind": kind, "batch": rng.choice([1, 1, 2, 4]), "heads": rng.choice([24, 32]),
                 "prefix": _log(rng, 1, 8395)}
            if c["batch"] * c["heads"] * c["prefix"] <= 32 * 8395:
                return c
        elif kind == "attn":
            sq = _log(rng, 1, 4096)
            c = {"kind": kind, "batch": rng.choice([1, 1, 2, 4, 8]), "heads": rng.choice([24, 32]),
                 "prefix": _log(rng, 1, 16640), "sq": sq, "own": rng.choice([0, sq, sq, sq, _log(rng, 1, 512)]),
                 "padded": rng.random() < 0.4}
            if c["batch"] * c["heads"] * c["prefix"] <= 8 * 32 * 16640 and work(c)["flops"] <= 5.6e11:
                return c
        else:
            rows, cols = rng.choice([(4096, 4096), (12288, 4096), (4096, 12288), (24576, 4096)])
            wt = rng.choice(["q4_k", "q8_0", "bf16"])
            m = _log(rng, 1, 16384)
            c = {"kind": kind, "wt": wt, "rows": rows, "cols": cols, "m": m, "requests": min(m, rng.choice([1, 2, 4, 16, 64])),
                 "adapters": rng.choice([1, 2, 3, 8, 16]), "rank": rng.choice([4, 8, 12, 16, 32, 33, 64, 96]),
                 "out": rng.choice(["bf16", "f32"]) if wt == "bf16" else "bf16"}
            if work(c)["flops"] <= 1.66e12:
                return c


# ---------------- inputs, from a seed ----------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _valid(c):
    """[batch, prefix + own] bytes: of a padded batch, each prompt but the first is shorter by up to a third."""
    v = torch.ones(c["batch"], c["prefix"] + c["own"], dtype=torch.uint8)
    for b, n in enumerate(_lengths(c)):
        v[b, n:c["prefix"]] = 0
    return v.cuda()


def _lengths(c):
    p, b = c["prefix"], c["batch"]
    return [p - (p * i // (3 * max(b - 1, 1)) if c["padded"] else 0) for i in range(b)]


def _cache_inputs(c, seed):
    g = _gen(seed)
    shape = (c["batch"], c["heads"], c["prefix"], HD)
    # keys as the block leaves them: normed per head, each dimension with its weight; values of a projection
    w = 1 + 0.3 * torch.randn(HD, device="cuda", generator=g)
    k = torch.randn(shape, device="cuda", generator=g)
    k = (k / k.square().mean(-1, keepdim=True).sqrt() * w).to(torch.bfloat16)
    v = (torch.randn(shape, device="cuda", generator=g) * 0.7).to(torch.bfloat16)
    return g, k, v


def _attn_inputs(c, seed):
    g, k, v = _cache_inputs(c, seed)
    b, h = c["batch"], c["heads"]
    q = torch.randn(b, h, c["sq"], HD, device="cuda", generator=g)
    q = (q / q.square().mean(-1, keepdim=True).sqrt() * 1.5).to(torch.bfloat16)
    ko = torch.randn(b, h, c["own"], HD, device="cuda", generator=g).to(torch.bfloat16)
    vo = (torch.randn(b, h, HD, c["own"], device="cuda", generator=g) * 0.7).to(torch.bfloat16)
    return {"k": k, "v": v, "q": q, "ko": ko, "vto": vo, "valid": _valid(c) if c["padded"] else None}


def _weight(c, g):
    """A projection's stored bytes [rows, row bytes] as a GGUF file holds them, on the GPU."""
    n, k, wt = c["rows"], c["cols"], c["wt"]

    def codes(shape, mid, spread, lo, hi):
        return (mid + spread * torch.randn(shape, device="cuda", generator=g)).round_().clamp_(lo, hi).to(torch.int16)

    def half(x):
        return x.to(torch.float16).view(torch.uint8).reshape(-1, 2)

    if wt == "bf16":
        return (torch.randn(n, k, device="cuda", generator=g) * 0.02).to(torch.bfloat16).view(torch.uint8)
    nb = n * k // (32 if wt == "q8_0" else 256)
    wobble = 1 + 0.1 * torch.randn(nb, 1, device="cuda", generator=g)
    if wt == "q8_0":
        q = codes((nb, 32), 0, 35, -127, 127).to(torch.int8).view(torch.uint8)
        return torch.cat([half(0.02 / 35 * wobble), q], 1).reshape(n, -1)
    d = (0.02 / 2.9 / 50) * wobble
    sc = codes((nb, 8), 50, 6, 20, 63)
    mn = (sc + codes((nb, 8), 0, 1.5, -5, 5)).clamp_(0, 63)
    q = codes((nb, 4, 2, 32), 7.5, 2.9, 0, 15)
    pk = torch.cat([sc[:, :4] | (sc[:, 4:] >> 4 << 6), mn[:, :4] | (mn[:, 4:] >> 4 << 6),
                    (sc[:, 4:] & 15) | ((mn[:, 4:] & 15) << 4)], 1).to(torch.uint8)
    qs = (q[:, :, 0] | (q[:, :, 1] << 4)).to(torch.uint8).reshape(nb, 128)
    return torch.cat([half(d), half(7.5 * d), pk, qs], 1).reshape(n, -1)


def _lora_inputs(c, seed):
    g = _gen(seed)
    raw = _weight(c, g)
    x = torch.randn(c["m"], c["cols"], device="cuda", generator=g).to(torch.bfloat16)
    ranks = [max(1, c["rank"] - i * c["rank"] // (2 * c["adapters"])) for i in range(c["adapters"])]
    a = [(torch.randn(r, c["cols"], device="cuda", generator=g) / math.sqrt(c["cols"])).to(torch.bfloat16) for r in ranks]
    b = [(torch.randn(c["rows"], r, device="cuda", generator=g) * 0.3).to(torch.bfloat16) for r in ranks]
    scale = [float(2.0 / r ** 0.5) for r in ranks]
    # the adapter of each request: any of them; where there are more requests than adapters the last has none
    req = torch.randint(0, c["adapters"], (c["requests"],), device="cuda", generator=g)
    if c["requests"] > c["adapters"]:
        req[-1] = -1
    at = torch.arange(c["m"], device="cuda") * c["requests"] // c["m"]
    return {"raw": raw, "x": x, "a": a, "b": b, "scale": scale, "ids": req[at].to(torch.int32)}


# ---------------- the plain forms ----------------

_CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_MIDS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


def _encode(x):
    """Blocks of 32 along the last dimension (a multiple of 32): codes and exponents s."""
    x = x.float().unflatten(-1, (-1, 32))
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))  # max|x| = m 2^e, 0.5 <= m < 1
    s = torch.where(m <= 0.875, e - 3, e - 2).clamp(-120, 125)
    y = torch.ldexp(x, -s).abs()
    up = torch.tensor([i % 2 == 1 for i in range(7)], device=x.device)
    mids = torch.tensor(_MIDS, device=x.device)
    # a magnitude's code counts the midpoints below it, and those it meets whose upper neighbour is even
    code = ((y.unsqueeze(-1) > mids) | ((y.unsqueeze(-1) == mids) & up)).sum(-1)
    return (code + 8 * (x < 0)).to(torch.uint8), s.squeeze(-1).to(torch.int8)


def _decode(code, s):
    table = torch.tensor(_CODES + tuple(-c for c in _CODES), device=code.device)
    return torch.ldexp(table[code.long()], s.int().unsqueeze(-1)).flatten(-2)


def _encode_kv(k, v):
    p = k.shape[2]
    vt = torch.nn.functional.pad(v.transpose(2, 3), (0, -p % 32))
    return _encode(k), _encode(vt.contiguous())


def _plain_store(s):
    k, v = _encode_kv(s["k"], s["v"])
    p = s["k"].shape[2]
    return {"k": _decode(*k).to(torch.bfloat16), "v": _decode(*v)[..., :p].transpose(2, 3).contiguous().to(torch.bfloat16)}


def _plain_attn(s):
    c = s["case"]
    k = torch.cat([_decode(*s["k4"]), s["ko"].float()], 2)
    vt = torch.cat([_decode(*s["v4"])[..., :c["prefix"]], s["vto"].float()], 3)
    t = torch.matmul(s["q"].float() * HD ** -0.5, k.transpose(2, 3).contiguous())
    if s["valid"] is not None:
        t = t.masked_fill((s["valid"] == 0)[:, None, None, :], -math.inf)
    t = (t - t.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(t / t.sum(-1, keepdim=True), vt.transpose(2, 3).contiguous())
    return o.transpose(1, 2).reshape(c["batch"], c["sq"], -1).to(torch.bfloat16)


def _dequant(c, raw):
    """The stored projection's values, f32."""
    n, k, wt = c["rows"], c["cols"], c["wt"]
    if wt == "bf16":
        return raw.view(torch.bfloat16).reshape(n, k).float()
    if wt == "q8_0":
        b = raw.reshape(-1, 34)
        return (b[:, :2].contiguous().view(torch.float16).float() * b[:, 2:].contiguous().view(torch.int8)).reshape(n, k)
    b = raw.reshape(-1, 144)
    d, m = b[:, :2].contiguous().view(torch.float16).float(), b[:, 2:4].contiguous().view(torch.float16).float()
    p = b[:, 4:16].short()
    sc = torch.cat([p[:, :4] & 63, (p[:, 8:] & 15) | (p[:, :4] >> 6 << 4)], 1)
    mn = torch.cat([p[:, 4:8] & 63, (p[:, 8:] >> 4) | (p[:, 4:8] >> 6 << 4)], 1)
    q = b[:, 16:].reshape(-1, 4, 32)
    q = torch.stack([q & 15, q >> 4], 2).reshape(-1, 8, 32)
    return ((d * sc).unsqueeze(2) * q - (m * mn).unsqueeze(2)).reshape(n, k)


def _plain_lora(s):
    x = s["x"].float()
    # every row against every adapter's A, those of other requests taken out, then all the B
    t = (x @ s["acat"].float().t()) * (s["ids"][:, None] == s["owner"]) * s["scales"]
    y = x @ s["w"].t() + t @ s["bcat"].float().t()
    return y if s["case"]["out"] == "f32" else y.to(torch.bfloat16)


# ---------------- the framework's calls ----------------

_ctx = None


def _qimm():
    global _ctx
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3-image21_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import qimm
    if _ctx is None:
        _ctx = qimm.Context(0)
    return qimm, _ctx


class _State(dict):
    """A case's buffers and handles; the handles are given back when it goes."""

    def __init__(self, **kw):
        super().__init__(**kw)
        self.held = []
        weakref.finalize(self, _State.give_back, self.held)

    __hash__ = object.__hash__

    @staticmethod
    def give_back(held):
        for h in reversed(held):
            h.free()

    def hold(self, h):
        self.held.append(h)
        return h


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ptr(t):
    return t.data_ptr() if t is not None and t.numel() else None


def prepare(case, seed):
    c, kind = case, case["kind"]
    if kind == "store":
        _, k, v = _cache_inputs(c, seed)
        s = _State(case=c, k=k, v=v)
        if own:
            _, ctx = _qimm()
            s["kv"] = s.hold(ctx.kv_create_q4(1, c["batch"], c["heads"], c["prefix"]))
            s["out"] = {"k": torch.empty_like(k), "v": torch.empty_like(v)}
        return s
    if kind == "attn":
        s = _State(case=c, **_attn_inputs(c, seed))
        if own:
            _, ctx = _qimm()
            s["kv"] = s.hold(ctx.kv_create_q4(1, c["batch"], c["heads"], c["prefix"]))
            s["kv"].store(0, s["k"].data_ptr(), s["v"].data_ptr(), _stream())
            s["out"] = torch.empty(c["batch"], c["sq"], c["heads"] * HD, dtype=torch.bfloat16, device="cuda")
        else:
            s["k4"], s["v4"] = _encode_kv(s["k"], s["v"])
        return s
    s = _State(case=c, **_lora_inputs(c, seed))
    if own:
        qimm, ctx = _qimm()
        wt = {"q4_k": qimm.Q4_K, "q8_0": qimm.Q8_0, "bf16": qimm.BF16}[c["wt"]]
        s["w"] = s.hold(ctx.upload(wt, c["rows"], c["cols"], s["raw"].cpu().numpy().tobytes()))
        s["ad"] = s.hold(ctx.adapters_create(c["rows"], c["cols"], [
            (f, qimm.BF16, a.cpu().view(torch.uint8).numpy().tobytes(), b.cpu().view(torch.uint8).numpy().tobytes())
            for f, a, b in zip(s["scale"], s["a"], s["b"])]))
        s["out"] = torch.empty(c["m"], c["rows"], dtype=torch.float32 if c["out"] == "f32" else torch.bfloat16, device="cuda")
    else:
        s["w"] = _dequant(c, s["raw"])
        s["acat"], s["bcat"] = torch.cat(s["a"]), torch.cat(s["b"], 1)
        s["owner"] = torch.cat([torch.full((len(a),), i, device="cuda") for i, a in enumerate(s["a"])])
        s["scales"] = torch.cat([torch.full((len(a),), f, device="cuda") for f, a in zip(s["scale"], s["a"])])
    return s


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"store": _plain_store, "attn": _plain_attn, "lora": _plain_lora}[c["kind"]](s)
    qimm, ctx = _qimm()
    if c["kind"] == "store":
        s["kv"].store(0, s["k"].data_ptr(), s["v"].data_ptr(), _stream())
        s["kv"].load(0, s["out"]["k"].data_ptr(), s["out"]["v"].data_ptr(), _stream())
    elif c["kind"] == "attn":
        args = (s["q"].data_ptr(), c["batch"], c["heads"], c["sq"], s["kv"], 0, _ptr(s["ko"]), _ptr(s["vto"]), c["own"],
                HD ** -0.5, s["out"].data_ptr())
        if s["valid"] is not None:
            ctx.attention_masked(*args, key_valid=s["valid"].data_ptr(), stream=_stream())
        else:
            ctx.attention(*args, stream=_stream())
    else:
        ctx.qmatmul_adapters(s["w"], s["ad"], s["ids"].data_ptr(), s["x"].data_ptr(), c["m"], c["cols"],
                             s["out"].data_ptr(), qimm.F32 if c["out"] == "f32" else qimm.BF16, _stream())
    return s["out"]


def work(case):
    c = case
    if c["kind"] == "store":  # read and written in bf16, written and read again in 4.25 bits, K and V
        n = 2 * c["batch"] * c["heads"] * c["prefix"] * HD
        return {"bytes": n * (2 + 2 + 2 * 4.25 / 8), "flops": 0}
    if c["kind"] == "attn":
        h, keys = c["heads"], sum(_lengths(c))
        cache, mine = 2 * h * keys * HD, 2 * h * c["batch"] * c["own"] * HD
        return {"bytes": cache * 4.25 / 8 + 2 * mine + 4 * c["batch"] * h * c["sq"] * HD,
                "flops": 4.0 * h * HD * c["sq"] * (keys + c["batch"] * c["own"])}
    n, k, m = c["rows"], c["cols"], c["m"]
    ranks = [max(1, c["rank"] - i * c["rank"] // (2 * c["adapters"])) for i in range(c["adapters"])]
    value = {"q4_k": 144 / 256, "q8_0": 34 / 32, "bf16": 2.0}[c["wt"]]
    used = min(c["adapters"], c["requests"])
    return {"bytes": n * k * value + 2 * m * k + (4 if c["out"] == "f32" else 2) * m * n + 2 * sum(ranks[:used]) * (n + k),
            "flops": 2.0 * m * n * k + 2.0 * m * (n + k) * sum(ranks) / len(ranks)}


# ---------------- 64 bits ----------------

def _near(x):
    """The values that blocks of 32 along the last dimension stand for, f64."""
    x = x.double().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1, keepdim=True)
    s = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 7.0))
    # log2 may round across a power of two: step to the smallest s that holds
    s = torch.where(top > 7 * torch.exp2(s), s + 1, s)
    s = torch.where(top <= 7 * torch.exp2(s - 1), s - 1, s).clamp(-120, 125)
    one = torch.exp2(s)
    y = x.abs() / one
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))  # the spacing of the values around y
    return (((y / step).round() * step).clamp(max=6.0) * one * torch.sign(x)).flatten(-2)


def _near_kv(k, v):
    p = k.shape[2]
    vt = torch.cat([v.transpose(2, 3), v.new_zeros(v.shape[0], v.shape[1], HD, -p % 32)], 3)
    return _near(k), _near(vt)[..., :p].transpose(2, 3)


def exact(case, seed):
    c = case
    if c["kind"] == "store":
        _, k, v = _cache_inputs(c, seed)
        k, v = _near_kv(k, v)
        return {"k": k, "v": v.contiguous()}
    if c["kind"] == "attn":
        i = _attn_inputs(c, seed)
        pk, pv = _near_kv(i["k"], i["v"])
        out = torch.empty(c["batch"], c["sq"], c["heads"], HD, dtype=torch.float64, device="cuda")
        for b in range(c["batch"]):
            seen = i["valid"][b].bool() if i["valid"] is not None else torch.ones(c["prefix"] + c["own"], dtype=torch.bool, device="cuda")
            for h in range(c["heads"]):
                k = torch.cat([pk[b, h], i["ko"][b, h].double()])[seen]
                v = torch.cat([pv[b, h], i["vto"][b, h].double().t()])[seen]
                out[b, :, h] = torch.softmax(i["q"][b, h].double() @ k.t() / math.sqrt(HD), -1) @ v
        return out.flatten(2)
    i = _lora_inputs(c, seed)
    x, raw, n, k = i["x"].double(), i["raw"], c["rows"], c["cols"]
    if c["wt"] == "bf16":
        w = raw.view(torch.bfloat16).double()
    elif c["wt"] == "q8_0":
        blocks = raw.view(n, k // 32, 34)
        w = (blocks[..., 2:].contiguous().view(torch.int8).double() * blocks[..., :2].contiguous().view(torch.float16).double()).view(n, k)
    else:
        blocks = raw.view(n, k // 256, 144)
        two = blocks[..., :4].contiguous().view(torch.float16).double()
        lo, hi, mix = (blocks[..., a:a + 4].int() for a in (4, 8, 12))
        w = torch.empty(n, k // 256, 256, dtype=torch.float64, device="cuda")
        for j in range(8):  # sub-block j: 32 values, low nibbles for even j
            s = (lo[..., j] & 63) if j < 4 else (mix[..., j - 4] & 15) + 16 * (lo[..., j - 4] >> 6)
            m = (hi[..., j] & 63) if j < 4 else (mix[..., j - 4] >> 4) + 16 * (hi[..., j - 4] >> 6)
            q = blocks[..., 16 + 32 * (j // 2):48 + 32 * (j // 2)].int()
            q = q >> 4 if j % 2 else q & 15
            w[..., 32 * j:32 * j + 32] = (two[..., 0] * s)[..., None] * q - (two[..., 1] * m)[..., None]
        w = w.view(n, k)
    y = x @ w.t()
    for j, (a, b, f) in enumerate(zip(i["a"], i["b"], i["scale"])):
        rows = i["ids"] == j
        y[rows] += f * (x[rows] @ a.double().t()) @ b.double().t()
    return y
