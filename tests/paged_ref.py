"""Plain forms of the paged cache's operators for the tests: a step of the page tables in Python
integers, the attention of a step's rows in 64 bits."""
import numpy as np


def pages_of(n, page):
    return -(-n // page)


def plan(page, pages, tables, lengths, added, queue, state, max_rows):
    """The arrays that one step leaves: tables, lengths, queue, state, starts, slots, positions."""
    tables, queue, after = tables.copy(), queue.copy(), lengths.copy()
    width, head, free = tables.shape[1], int(state[0]) % pages, min(max(int(state[1]), 0), pages)
    starts, slots, positions = [0], np.full(max_rows, -1, np.int32), np.zeros(max_rows, np.int32)
    rows = asked = taken = freed = refused = 0
    for r, (n, a) in enumerate(zip(lengths.tolist(), added.tolist())):
        have = min(pages_of(max(n, 0), page), width)
        if a < 0:
            for k in range(have):
                queue[(head + free + freed) % pages] = tables[r, k]
                freed += 1
            after[r] = 0
        elif a > 0:
            rows += a
            fits = n >= 0 and n + a <= width * page and rows <= max_rows
            need = pages_of(n + a, page) - have if fits else 0
            asked += need
            if fits and (need == 0 or asked <= free):
                for k in range(need):
                    tables[r, have + k] = queue[(head + asked - need + k) % pages]
                taken += need
                after[r] = n + a
                for i in range(a):
                    p = n + i
                    slots[rows - a + i], positions[rows - a + i] = tables[r, p // page] * page + p % page, p
            else:
                refused += 1
        starts.append(min(rows, max_rows))
    state = np.array([(head + taken) % pages, free - taken + freed, starts[-1], refused], np.int32)
    return dict(tables=tables, lengths=after, queue=queue, state=state, starts=np.array(starts, np.int32), slots=slots,
                positions=positions)


def attention(torch, q, k, v, tables, lengths, starts, page, causal, window=0, sinks=0, scale=None):
    """q [T,H,D], k and v [pages * page, Hkv, D] as they are stored; 64 bits. The outputs [T,H,D], zeros
    where a row sees nothing and NaN for rows of no request, and the means of |v| under the same weights."""
    t, h, d = q.shape
    kv = k.shape[1]
    g, pages = h // kv, k.shape[0] // page
    scale = d ** -0.5 if scale is None else scale
    out = torch.full((t, h, d), float("nan"), dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for r in range(len(lengths)):
        a, b, n = int(starts[r]), int(starts[r + 1]), int(lengths[r])
        if a == b:
            continue
        m = b - a
        token = torch.arange(n, device=q.device)
        page_of = tables[r].long()[token // page]
        there = (page_of >= 0) & (page_of < pages)
        slot = torch.where(there, page_of * page + token % page, 0)
        pos = n - m + torch.arange(m, device=q.device)[:, None]
        sees = (token <= pos) if causal else torch.ones(m, n, dtype=torch.bool, device=q.device)
        if window:
            sees = sees & ((token > pos - window) | (token < sinks))
        sees = sees & there
        for x in range(kv):
            kk, vv = k[slot, x].double(), v[slot, x].double()
            qq = q[a:b, x * g:(x + 1) * g].double()
            s = (qq.reshape(m * g, d) @ kk.t().contiguous()).reshape(m, g, n) * scale
            s = torch.where(sees[:, None, :], s, -float("inf"))
            s = s - (s.amax(-1, keepdim=True) if n else 0.0)
            p = torch.where(sees[:, None, :], s.exp(), 0.0)
            w = p / p.sum(-1, keepdim=True)
            w = torch.where(sees.any(-1)[:, None, None], w, 0.0)
            # a hidden key's value does not count, whatever it is; a NaN or an infinity that is seen does
            fine = torch.where(torch.isfinite(vv), vv, 0.0)
            o = (w.reshape(m * g, n) @ fine).reshape(m, g, d)
            av = (w.reshape(m * g, n) @ fine.abs()).reshape(m, g, d)
            for j in torch.nonzero(~torch.isfinite(vv).all(-1)).flatten().tolist():
                hit = sees[:, j][:, None, None] & ~torch.isfinite(vv[j])[None, None, :]
                o = torch.where(hit, o + vv[j], o)
            out[a:b, x * g:(x + 1) * g], mag[a:b, x * g:(x + 1) * g] = o, av
    return out, mag


# |error| <= TOL * (mean of |v| under the weights): the probabilities and the output are rounded to bf16,
# half a step of 2^-8 each; the f32 scores, sums of up to 128 products of |q k| scale <= 16 in all, are
# off by 128 2^-24 16 = 2^-13, in the numerator and the sum: 2^-12, doubled for the f32 sums over the keys
TOL = 2.0 ** -7 + 2.0 ** -11


def assert_near(torch, got, want, mag):
    """NaN where the reference has one, the same infinities, and else within TOL."""
    got = got.double().reshape(want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    ok = torch.isfinite(want)
    off = (got - want).abs()[ok] - TOL * mag[ok] - 1e-30
    assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())
