"""The operators of a paged K/V cache for many requests of unequal lengths: block tables and slot
maps from request lengths, the store of new tokens into pages, and the attention that reads them.
Each in its plain form (elementary torch operations in 32 bits), through the public binding, and in
64 bits.

A case is a dict of plain values; its "kind" names the call:

- "plan": one step of the page tables (Context.page_plan): every request adds tokens, none, or is given
  back; new pages come from the queue of free ones, in request order, and each new token gets its
  row, its position and its slot (page * page size + place in the page);
- "store": keys and values of the rows of a step into their slots and back (Pages.store, load);
- "attn": attention of a step's rows over the pages of their requests (Pages.attention): requests
  with one new token, with chunks of them or with both mixed; every row over all keys of its
  request, or causal, or causal in a window with a few first keys that stay visible.

Sizes: 32 heads of 128 are the model's block; fewer key heads than heads, and heads of 64, are the
generic layouts of the text and vision models beside it. Prompts have any number of tokens, a
reference image adds its own; an image of H x W pixels is H/16 x W/16 tokens.
"""
import math
import os
import sys
import weakref

import numpy as np
import torch

own = False


def listed():
    return [
        # the smallest step: 48 requests, one new token each
        {"name": "plan_tokens_48", "kind": "plan", "requests": 48, "page": 64, "low": 20, "high": 4299, "chunks": 0,
         "new": 0, "gone": 0},
        # a step of a large server: chunks of new prompts, single tokens, a few requests given back
        {"name": "plan_churn_2048", "kind": "plan", "requests": 2048, "page": 16, "low": 20, "high": 16640,
         "chunks": 128, "new": 509, "gone": 40},
        # the new tokens of 48 requests, in bf16
        {"name": "store_tokens_48", "kind": "store", "requests": 48, "rows": 48, "kv_heads": 8, "dim": 128, "page": 64,
         "type": "bf16", "padding": 0},
        # the f32 projections of an edit with two 1024x1024 reference images, the rows padded to 8448
        {"name": "store_edit_8395", "kind": "store", "requests": 1, "rows": 8395, "kv_heads": 32, "dim": 128,
         "page": 64, "type": "f32", "padding": 53},
        # the smallest attention: one token over an ordinary prompt
        {"name": "token_333", "kind": "attn", "requests": 1, "low": 333, "high": 333, "heads": 32, "kv_heads": 32,
         "dim": 128, "page": 16, "chunks": 0, "new": 1, "causal": True, "window": 0, "sinks": 0},
        # one token of each of 48 requests with prompts of every length, grouped heads
        {"name": "tokens_48_ragged", "kind": "attn", "requests": 48, "low": 100, "high": 16640, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "chunks": 0, "new": 1, "causal": True, "window": 0, "sinks": 0},
        # one long request
        {"name": "token_131001", "kind": "attn", "requests": 1, "low": 131001, "high": 131001, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 128, "chunks": 0, "new": 1, "causal": True, "window": 0, "sinks": 0},
        # tokens of long requests in a window, the first keys visible
        {"name": "tokens_16_window", "kind": "attn", "requests": 16, "low": 1500, "high": 33000, "heads": 32,
         "kv_heads": 8, "dim": 64, "page": 16, "chunks": 0, "new": 1, "causal": True, "window": 1024, "sinks": 4},
        # a mixed step: two chunks of prompts among single tokens
        {"name": "mixed_32", "kind": "attn", "requests": 32, "low": 700, "high": 8395, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "chunks": 2, "new": 517, "causal": True, "window": 0, "sinks": 0},
        # a whole prompt with reference images, causal
        {"name": "prompt_8395", "kind": "attn", "requests": 1, "low": 8395, "high": 8395, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "chunks": 1, "new": 8395, "causal": True, "window": 0, "sinks": 0},
        # two long prompts in a window with sinks
        {"name": "prompts_2_window", "kind": "attn", "requests": 2, "low": 9000, "high": 16640, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "chunks": 2, "new": 8395, "causal": True, "window": 1024, "sinks": 4},
        # image tokens of four 512x512 requests over prompts of their own lengths and themselves
        {"name": "images_4_512", "kind": "attn", "requests": 4, "low": 1100, "high": 5400, "heads": 32, "kv_heads": 32,
         "dim": 128, "page": 64, "chunks": 4, "new": 1024, "causal": False, "window": 0, "sinks": 0},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    while True:
        kind = rng.choice(["plan", "store", "attn", "attn", "attn"])
        if kind == "plan":
            n = _log(rng, 1, 2048)
            low = _log(rng, 1, 4299)
            c = {"kind": kind, "requests": n, "page": rng.choice([16, 32, 48, 64, 128]), "low": low,
                 "high": low + _log(rng, 1, 16640), "chunks": rng.choice([0, 0, min(n, _log(rng, 1, 128))]),
                 "new": _log(rng, 1, 509), "gone": rng.choice([0, n // 40])}
            return c
        if kind == "store":
            rows = _log(rng, 1, 8395)
            c = {"kind": kind, "requests": rng.choice([1, 2, 7, 48]), "rows": rows, "kv_heads": rng.choice([1, 2, 4, 5, 8, 32]),
                 "dim": rng.choice([64, 128, 128]), "page": rng.choice([16, 32, 48, 64, 128]),
                 "type": rng.choice(["bf16", "f16", "f32"]), "padding": rng.choice([0, 0, 3, 50])}
            c["requests"] = min(c["requests"], rows)
            return c
        kv = rng.choice([1, 2, 4, 5, 8, 32])
        n = rng.choice([1, 1, 2, 5, 16, 48])
        low = _log(rng, 1, 20000)
        c = {"kind": kind, "requests": n, "low": low, "high": low + _log(rng, 1, 20000), "heads": kv * rng.choice([1, 2, 3, 4, 7, 8]),
             "kv_heads": kv, "dim": rng.choice([64, 128, 128]), "page": rng.choice([16, 32, 48, 64, 128]),
             "chunks": rng.choice([0, 0, 1, n]), "new": _log(rng, 1, 8395), "causal": rng.random() < 0.8, "window": 0, "sinks": 0}
        c["chunks"] = min(c["chunks"], n)
        c["new"] = min(c["new"], low)
        if c["causal"] and rng.random() < 0.4:
            c["window"], c["sinks"] = _log(rng, 16, 4096), rng.choice([0, 1, 4, 17])
        if c["heads"] <= 64 and work(c)["flops"] <= 5.7e11 and sum(_lengths(c)) * kv * c["dim"] <= 2 ** 28:
            return c


# ---------------- sizes, from the case alone ----------------

def _lengths(c):
    """The requests' lengths: spread over the logarithm of low .. high."""
    return [int(c["low"] * (c["high"] / c["low"]) ** (i * 0.6180339887498949 % 1.0) + 0.5) for i in range(c["requests"])]


def _rows(c):
    """The rows of each request: chunks first among the requests, spread out, single tokens else."""
    n, k = c["requests"], c["chunks"]
    at = {i * n // k for i in range(k)} if k else ()
    return [c["new"] if i in at else 1 for i in range(n)]


def _added(c):
    """A plan's step: chunks, single tokens, and requests that are given back."""
    a = _rows(c)
    for i in range(c["gone"]):
        a[(i * 37 + 5) % c["requests"]] = -1
    return a


def _pages(n, page):
    return (n + page - 1) // page


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---------------- inputs, from a seed ----------------

def _plan_inputs(c, seed):
    g = _gen(seed)
    lengths, added, page = _lengths(c), _added(c), c["page"]
    have = [_pages(n, page) for n in lengths]
    after = [_pages(n + max(a, 0), page) for n, a in zip(lengths, added)]
    width = max(after) + 2
    total = sum(after) + 11
    perm = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    tables = torch.zeros(c["requests"], width, dtype=torch.int32, device="cuda")
    ends = torch.tensor([0] + have, device="cuda").cumsum(0)
    at = torch.arange(width, device="cuda")[None, :]
    held = at < torch.tensor(have, device="cuda")[:, None]
    tables[held] = perm[(ends[:-1, None] + at)[held]]
    free = total - sum(have)
    head = int(torch.randint(0, total, (1,), device="cuda", generator=g))
    queue = torch.full((total,), -7, dtype=torch.int32, device="cuda")
    queue[(head + torch.arange(free, device="cuda")) % total] = perm[sum(have):]
    rows = sum(max(a, 0) for a in added)
    return {"tables": tables, "lengths": _i32(lengths), "added": _i32(added), "queue": queue,
            "state": _i32([head, free, 0, 0]), "max_rows": rows + 5, "total": total}


def _slots(g, lengths, page):
    """Slots of the first lengths[i] tokens of each request, their pages dealt from a random order."""
    total = sum(_pages(n, page) for n in lengths) + 3
    perm = torch.randperm(total, device="cuda", generator=g)
    out, at = [], 0
    for n in lengths:
        k = _pages(n, page)
        out.append((perm[at:at + k, None] * page + torch.arange(page, device="cuda")).flatten()[:n])
        at += k
    return total, out


def _store_inputs(c, seed):
    g = _gen(seed)
    r, rows = c["requests"], c["rows"]
    n = [rows * (i + 1) // r - rows * i // r for i in range(r)]
    # every request's rows follow some tokens that it has
    before = [(i * 29 + 11) % 50 for i in range(r)]
    total, slots = _slots(g, [a + b for a, b in zip(before, n)], c["page"])
    slots = torch.cat([s[b:] for s, b in zip(slots, before)] + [torch.full((c["padding"],), -1, device="cuda")])
    t = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[c["type"]]
    shape = (rows + c["padding"], c["kv_heads"], c["dim"])
    return {"total": total, "slots": slots.to(torch.int32), "k": torch.randn(shape, device="cuda", generator=g).to(t),
            "v": (torch.randn(shape, device="cuda", generator=g) * 0.7).to(t)}


def _attn_inputs(c, seed):
    g = _gen(seed)
    lengths, rows, page, d = _lengths(c), _rows(c), c["page"], c["dim"]
    have = [_pages(n, page) for n in lengths]
    total = sum(have) + 3
    perm = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    tables = torch.zeros(c["requests"], max(have), dtype=torch.int32, device="cuda")
    at = 0
    for i, k in enumerate(have):
        tables[i, :k] = perm[at:at + k]
        at += k
    # keys as the block leaves them: normed per head, each dimension with its weight
    w = 1 + 0.3 * torch.randn(d, device="cuda", generator=g)
    k = torch.randn(total * page, c["kv_heads"], d, device="cuda", generator=g)
    k = (k / k.square().mean(-1, keepdim=True).sqrt() * w).to(torch.bfloat16)
    v = (torch.randn(total * page, c["kv_heads"], d, device="cuda", generator=g) * 0.7).to(torch.bfloat16)
    q = torch.randn(sum(rows), c["heads"], d, device="cuda", generator=g)
    q = (q / q.square().mean(-1, keepdim=True).sqrt() * 1.5).to(torch.bfloat16)
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    return {"tables": tables, "lengths": _i32(lengths), "starts": _i32(starts), "q": q, "k": k, "v": v, "total": total}


# ---------------- the plain forms ----------------

def _plain_plan(s):
    page, total, cap = s["case"]["page"], s["total"], s["max_rows"]
    old, added, tables, queue = s["lengths"].long(), s["added"].long(), s["tables"].long(), s["queue"].long()
    head, free = s["state"][0].long(), s["state"][1].long()
    width = tables.shape[1]
    rows = added.clamp(min=0)
    ends = rows.cumsum(0)
    fits = (added > 0) & (old >= 0) & (old + added <= width * page) & (ends <= cap)
    have = (old + page - 1) // page
    need = torch.where(fits, (old + added + page - 1) // page - have, 0)
    cum = need.cumsum(0)
    served = fits & ((need == 0) | (cum <= free))
    taken = torch.where(served, need, 0).sum()
    gone = added < 0
    freed = torch.where(gone, have.clamp(0, width), 0)
    starts = torch.cat([ends.new_zeros(1), ends]).clamp(max=cap)
    # the pages that requests take, and those that they give back
    at = torch.arange(width, device=old.device)[None, :]
    new = served[:, None] & (at >= have[:, None]) & (at < (have + need)[:, None])
    tables = torch.where(new, queue[(head + (cum - need)[:, None] + at - have[:, None]) % total], tables)
    back = gone[:, None] & (at < freed[:, None])
    to = (head + free + (freed.cumsum(0) - freed)[:, None] + at) % total
    queue = torch.cat([queue, queue[:1]]).scatter(0, torch.where(back, to, total).flatten(), tables.flatten())[:total]
    t = torch.arange(cap, device=old.device)
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=len(old) - 1)
    pos = old[r] + t - starts[r]
    ok = served[r] & (t < starts[-1])
    slot = tables[r, torch.where(ok, pos // page, 0)] * page + pos % page
    state = torch.stack([(head + taken) % total, free - taken + freed.sum(), starts[-1], ((added > 0) & ~served).sum()])
    return {"tables": tables.int(), "queue": queue.int(), "state": state.int(), "starts": starts.int(),
            "lengths": torch.where(gone, 0, torch.where(served, old + added, old)).int(),
            "slots": torch.where(ok, slot, -1).int(), "positions": torch.where(ok, pos, 0).int()}


def _plain_store(s):
    ok, at = s["slots"] >= 0, s["slots"].long()
    out = {}
    for name in ("k", "v"):
        # rows without a slot go behind the last page
        cache = s["cache_" + name]
        cache[torch.where(ok, at, len(cache) - 1)] = s[name].to(torch.bfloat16)
        out[name] = torch.where(ok[:, None, None], cache[at.clamp(min=0)], 0)
    return out


def _plain_attn(s):
    c, lengths, rows = s["case"], s["host_lengths"], s["host_rows"]
    page, kv, d, g = c["page"], c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    k, v = s["k"].view(-1, page, kv, d), s["v"].view(-1, page, kv, d)
    out, at = [], 0
    for i, (n, m) in enumerate(zip(lengths, rows)):
        pages = s["tables"][i, :_pages(n, page)].long()
        kt = k[pages].flatten(0, 1)[:n].float().permute(1, 2, 0).contiguous()
        vt = v[pages].flatten(0, 1)[:n].float().transpose(0, 1).contiguous()
        q = s["q"][at:at + m].float() * d ** -0.5
        t = torch.matmul(q.view(m, kv, g, d).transpose(0, 1).reshape(kv, m * g, d), kt).view(kv, m, g, n)
        if c["causal"] and (m > 1 or c["window"]):
            pos, key = torch.arange(n - m, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None, :]
            hide = key > pos
            if c["window"]:
                hide |= (key <= pos - c["window"]) & (key >= c["sinks"])
            t.masked_fill_(hide[None, :, None, :], -math.inf)
        t = t.sub_(t.amax(-1, keepdim=True)).exp_()
        t = t.div_(t.sum(-1, keepdim=True)).view(kv, m * g, n)
        out.append(torch.matmul(t, vt).view(kv, m, g, d).transpose(0, 1).reshape(m, kv * g * d).to(torch.bfloat16))
        at += m
    return torch.cat(out)


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


def prepare(case, seed):
    c, kind = case, case["kind"]
    if kind == "plan":
        s = _State(case=c, **_plan_inputs(c, seed))
        if own:
            qimm, ctx = _qimm()
            n, cap = c["requests"], s["max_rows"]
            out = {k: torch.empty(m, dtype=torch.int32, device="cuda")
                   for k, m in (("lengths", n), ("state", 4), ("starts", n + 1), ("slots", cap), ("positions", cap))}
            # tables and queue are the program's own, written in place
            out["tables"], out["queue"] = s["tables"], s["queue"]
            s["work"] = torch.empty(qimm.page_plan_work(n), dtype=torch.int32, device="cuda")
            s["out"] = out
            s["call"] = qimm.PagePlan(page_size=c["page"], pages=s["total"], requests=n, max_pages=s["tables"].shape[1],
                                      max_rows=cap, tables=s["tables"].data_ptr(), lengths=s["lengths"].data_ptr(),
                                      added=s["added"].data_ptr(), queue=s["queue"].data_ptr(), state=s["state"].data_ptr(),
                                      lengths_out=out["lengths"].data_ptr(), state_out=out["state"].data_ptr(),
                                      starts=out["starts"].data_ptr(), slots=out["slots"].data_ptr(),
                                      positions=out["positions"].data_ptr(), work=s["work"].data_ptr())
        return s
    if kind == "store":
        s = _State(case=c, **_store_inputs(c, seed))
        if own:
            qimm, ctx = _qimm()
            s["pages"] = s.hold(ctx.pages_create(1, s["total"], c["page"], c["kv_heads"], c["dim"]))
            s["type"] = {"bf16": qimm.BF16, "f16": qimm.F16, "f32": qimm.F32}[c["type"]]
            s["out"] = {n: torch.empty(s[n].shape, dtype=torch.bfloat16, device="cuda") for n in ("k", "v")}
        else:
            for n in ("k", "v"):
                s["cache_" + n] = torch.zeros(s["total"] * c["page"] + 1, c["kv_heads"], c["dim"], dtype=torch.bfloat16, device="cuda")
        return s
    s = _State(case=c, **_attn_inputs(c, seed))
    s["host_lengths"], s["host_rows"] = _lengths(c), _rows(c)
    if own:
        qimm, ctx = _qimm()
        s["pages"] = s.hold(ctx.pages_create(1, s["total"], c["page"], c["kv_heads"], c["dim"]))
        every = torch.arange(s["total"] * c["page"], dtype=torch.int32, device="cuda")
        s["pages"].store(0, s["k"].data_ptr(), s["v"].data_ptr(), qimm.BF16, len(every), every.data_ptr(), stream=_stream())
        rows = sum(s["host_rows"])
        s["out"] = torch.empty(rows, c["heads"] * c["dim"], dtype=torch.bfloat16, device="cuda")
        s["call"] = qimm.PagedAttention(q=s["q"].data_ptr(), q_row=c["heads"] * c["dim"], q_head=c["dim"], rows=rows,
                                        heads=c["heads"], requests=c["requests"], max_pages=s["tables"].shape[1],
                                        tables=s["tables"].data_ptr(), lengths=s["lengths"].data_ptr(),
                                        starts=s["starts"].data_ptr() if c["chunks"] else None, causal=int(c["causal"]),
                                        window=c["window"], sinks=c["sinks"], scale=c["dim"] ** -0.5,
                                        out=s["out"].data_ptr())
    return s


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"plan": _plain_plan, "store": _plain_store, "attn": _plain_attn}[c["kind"]](s)
    if c["kind"] == "plan":
        _qimm()[1].page_plan(s["call"], _stream())
    elif c["kind"] == "store":
        n = len(s["slots"])
        s["pages"].store(0, s["k"].data_ptr(), s["v"].data_ptr(), s["type"], n, s["slots"].data_ptr(), stream=_stream())
        s["pages"].load(0, s["out"]["k"].data_ptr(), s["out"]["v"].data_ptr(), n, s["slots"].data_ptr(), stream=_stream())
    else:
        s["pages"].attention(0, s["call"], _stream())
    return s["out"]


def _seen(c, n, m):
    """Keys that the m last rows of n tokens see, over the rows, and how many keys any of them sees."""
    if not c["causal"]:
        return m * n, n
    w, f = c["window"] or n, c["sinks"] if c["window"] else 0
    # row at p: the last min(w, p + 1) keys and those of the first f that lie before them
    pairs = sum(min(w, p + 1) + min(f, max(0, p + 1 - w)) for p in range(n - m, n))
    low = max(0, n - m + 1 - w)
    return pairs, n - low + min(f, low)


def work(case):
    c = case
    if c["kind"] == "plan":
        rows = [max(a, 0) for a in _added(c)]
        new = sum(_pages(n + a, c["page"]) - _pages(n, c["page"]) for n, a in zip(_lengths(c), rows))
        back = sum(_pages(n, c["page"]) for n, a in zip(_lengths(c), _added(c)) if a < 0)
        return {"bytes": 16 * c["requests"] + 8 * (new + back) + 8 * sum(rows), "flops": 0}
    if c["kind"] == "store":  # read in its type, written in bf16, read and written again in bf16
        n = 2 * c["rows"] * c["kv_heads"] * c["dim"]
        return {"bytes": n * ((4 if c["type"] == "f32" else 2) + 6) + 8 * c["rows"], "flops": 0}
    d, pairs, keys = c["dim"], 0, 0
    for n, m in zip(_lengths(c), _rows(c)):
        a, b = _seen(c, n, m)
        pairs, keys = pairs + a, keys + b
    return {"bytes": 4 * keys * c["kv_heads"] * d + 4 * sum(_rows(c)) * c["heads"] * d, "flops": 4.0 * c["heads"] * d * pairs}


# ---------------- in 64 bits ----------------

def _exact_plan(c, seed):
    i = _plan_inputs(c, seed)
    tables, lengths, added, queue, state = (i[n].cpu().numpy().astype(np.int64) for n in ("tables", "lengths", "added", "queue", "state"))
    page, total, cap, (head, free) = c["page"], i["total"], i["max_rows"], state[:2]
    starts, slots, positions = [0], np.full(cap, -1), np.zeros(cap, dtype=np.int64)
    asked = taken = freed = refused = row = 0
    after = lengths.copy()
    for r, (n, a) in enumerate(zip(lengths, added)):
        have = -(-int(n) // page)
        if a < 0:
            for k in range(have):
                queue[(head + free + freed) % total] = tables[r, k]
                freed += 1
            after[r] = 0
        elif a > 0:
            row += a
            fits = n + a <= tables.shape[1] * page and row <= cap
            need = -(-int(n + a) // page) - have if fits else 0
            asked += need
            if fits and (need == 0 or asked <= free):
                for k in range(need):
                    tables[r, have + k] = queue[(head + asked - need + k) % total]
                taken += need
                p = np.arange(n, n + a)
                slots[row - a:row], positions[row - a:row] = tables[r, p // page] * page + p % page, p
                after[r] = n + a
            else:
                refused += 1
        starts.append(min(row, cap))
    out = {"tables": tables, "queue": queue, "state": np.array([(head + taken) % total, free - taken + freed, starts[-1], refused]),
           "starts": np.array(starts), "lengths": after, "slots": slots, "positions": positions}
    return {n: torch.from_numpy(x).to(torch.int32) for n, x in out.items()}


def exact(case, seed):
    c = case
    if c["kind"] == "plan":
        return _exact_plan(c, seed)
    if c["kind"] == "store":
        i = _store_inputs(c, seed)
        there = (i["slots"] >= 0).double()[:, None, None]
        return {n: i[n].double() * there for n in ("k", "v")}
    i = _attn_inputs(c, seed)
    d, g, page = c["dim"], c["heads"] // c["kv_heads"], c["page"]
    out = torch.empty(len(i["q"]), c["heads"], d, dtype=torch.float64, device="cuda")
    tables, row = i["tables"].long(), 0
    for r, (n, m) in enumerate(zip(_lengths(c), _rows(c))):
        token = torch.arange(n, device="cuda")
        slot = tables[r, token // page] * page + token % page
        for h in range(c["kv_heads"]):
            k, v = i["k"][slot, h].double(), i["v"][slot, h].double()
            step = max(1, 2 ** 27 // (n * g))
            for a in range(0, m, step):
                b = min(m, a + step)
                x = torch.einsum("igd,jd->igj", i["q"][row + a:row + b, h * g:(h + 1) * g].double(), k) / math.sqrt(d)
                if c["causal"]:
                    p = (n - m + torch.arange(a, b, device="cuda"))[:, None]
                    sees = token <= p
                    if c["window"]:
                        sees &= (p - token < c["window"]) | (token < c["sinks"])
                    x = torch.where(sees[:, None, :], x, -math.inf)
                out[row + a:row + b, h * g:(h + 1) * g] = torch.softmax(x, -1) @ v
        row += m
    return out.flatten(1)
