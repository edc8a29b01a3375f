"""Attention over the paged cache against 64 bits: lengths around every tile's and page's end, grouped
heads, chunks and single tokens mixed, windows with sinks, what hidden keys hold, tables and lengths out
of range, strides, streams and graphs."""
import numpy as np
import pytest

import paged_ref
import qimm
from gpu_util import dev, host, stream
from paged_ref import assert_near

pytestmark = pytest.mark.gpu


class Case:
    """A cache with random pages, its tables and a step's rows. rows: the rows of each request."""

    def __init__(self, torch, ctx, lengths, rows, heads, kv, d, page, seed=0, layers=1, spare=2):
        self.torch, self.ctx, self.page, self.heads, self.d, self.layers = torch, ctx, page, heads, d, layers
        rng = np.random.default_rng(seed)
        have = [paged_ref.pages_of(n, page) for n in lengths]
        self.pages = sum(have) + spare
        perm, at = rng.permutation(self.pages), 0
        # entries past a request's pages are anything
        tables = rng.integers(-2 ** 31, 2 ** 31 - 1, (len(lengths), max(max(have), 1) + 1)).astype(np.int32)
        for r, k in enumerate(have):
            tables[r, :k] = perm[at:at + k]
            at += k
        self.tables, self.lengths = dev(torch, tables), list(lengths)
        self.starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.t = int(self.starts[-1])
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.q = (torch.randn(self.t, heads, d, device="cuda", generator=gen) * 1.5).to(torch.bfloat16)
        # no value of the cache is left to chance: slots of no token hold NaN
        self.k = torch.randn(self.pages * page, kv, d, device="cuda", generator=gen).to(torch.bfloat16)
        self.v = torch.randn(self.pages * page, kv, d, device="cuda", generator=gen).to(torch.bfloat16)
        used = torch.zeros(self.pages * page, dtype=torch.bool, device="cuda")
        for r, n in enumerate(lengths):
            used[self.slots(r, n)] = True
        self.k[~used] = float("nan")
        self.v[~used] = float("nan")
        self.pg = ctx.pages_create(layers, self.pages, page, kv, d)
        self.put()

    def slots(self, r, n):
        token = self.torch.arange(n, device="cuda")
        return self.tables[r].long()[token // self.page] * self.page + token % self.page

    def put(self, layer=0):
        every = self.torch.arange(self.pages * self.page, dtype=self.torch.int32, device="cuda")
        self.pg.store(layer, self.k.data_ptr(), self.v.data_ptr(), qimm.BF16, len(every), every.data_ptr(), stream=stream(self.torch))
        self.torch.cuda.synchronize()

    def call(self, causal=True, window=0, sinks=0, scale=None, single=False, rows=None, q=None, q_row=0, q_head=0, out=None):
        torch = self.torch
        self.lengths_d, self.starts_d = dev(torch, np.array(self.lengths, np.int32)), dev(torch, self.starts)
        rows = self.t if rows is None else rows
        self.out = torch.full((max(rows, 1), self.heads * self.d), 7.0, dtype=torch.bfloat16, device="cuda") if out is None else out
        q = self.q if q is None else q
        return qimm.PagedAttention(q=q.data_ptr(), q_row=q_row, q_head=q_head, rows=rows, heads=self.heads, requests=len(self.lengths),
                                   max_pages=self.tables.shape[1], tables=self.tables.data_ptr(), lengths=self.lengths_d.data_ptr(),
                                   starts=None if single else self.starts_d.data_ptr(), causal=int(causal), window=window, sinks=sinks,
                                   scale=self.d ** -0.5 if scale is None else scale, out=self.out.data_ptr())

    def want(self, causal=True, window=0, sinks=0, scale=None):
        return paged_ref.attention(self.torch, self.q, self.k, self.v, self.tables, self.lengths, self.starts, self.page, causal,
                                   window, sinks, scale)

    def check(self, **kw):
        single = kw.pop("single", False)
        self.pg.attention(0, self.call(single=single, **kw), stream(self.torch))
        assert_near(self.torch, self.out, *self.want(**kw))

    def free(self):
        self.pg.free()


ENDS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 130, 255, 257, 300, 511, 513, 1000]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 48, 64, 512])
@pytest.mark.parametrize("heads,kv", [(1, 1), (8, 2), (6, 2), (5, 1), (32, 1), (33, 1), (80, 2)])
def test_single_tokens(torch_cuda, qctx, heads, kv, page, d):
    c = Case(torch_cuda, qctx, ENDS, [1] * len(ENDS), heads, kv, d, page, seed=heads)
    c.check(single=True)
    c.check(causal=False)
    c.check(single=True, window=33, sinks=5)
    c.free()


@pytest.mark.parametrize("d,page,heads,kv", [(128, 16, 4, 4), (64, 32, 4, 1), (128, 48, 14, 2), (64, 512, 3, 3), (128, 64, 8, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (7, 3), (64, 4), (100, 200), (10 ** 9, 2 ** 40)])
def test_chunks_and_tokens_mixed(torch_cuda, qctx, d, page, heads, kv, window, sinks):
    lengths = [1, 40, 129, 300, 77, 500, 33, 64, 1030, 600]
    rows = [1, 40, 3, 1, 0, 131, 2, 1, 257, 9]
    c = Case(torch_cuda, qctx, lengths, rows, heads, kv, d, page, seed=window % 97)
    c.check(window=window, sinks=sinks)
    if not window:
        c.check(causal=False)
    c.free()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv", [(4, 4), (16, 2)])
def test_long_requests(torch_cuda, qctx, heads, kv, d):
    """Lengths that are split over many workgroups, next to short ones."""
    lengths = [20011, 3, 8193, 1, 700, 16384]
    c = Case(torch_cuda, qctx, lengths, [1] * 6, heads, kv, d, 64)
    c.check(single=True)
    c.check(single=True, window=5000, sinks=100)
    c.free()
    c = Case(torch_cuda, qctx, lengths, [5, 2, 40, 1, 300, 0], heads, kv, d, 16)
    c.check()
    c.check(causal=False)
    c.check(window=3000, sinks=4)
    c.free()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv,rows", [(4, 1, 1), (1, 1, 1), (32, 1, 1), (16, 2, 12), (1, 1, 33), (5, 1, 129)])
def test_one_request_in_as_many_shares_as_there_may_be(torch_cuda, qctx, heads, kv, rows, d):
    """Shares joined in teams and the teams' sums after them, call after call."""
    c = Case(torch_cuda, qctx, [70001], [rows], heads, kv, d, 128)
    for _ in range(3):
        c.check()
    first = c.out.clone()
    c.check()
    assert torch_cuda.equal(first, c.out)  # the order of the sums does not depend on that of the arrivals
    c.check(causal=False)
    c.free()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("keys", [512, 513, 700, 1030, 1280, 1285, 2100, 4097, 4200, 16000])
def test_rows_in_few_and_many_shares(torch_cuda, qctx, keys, d):
    """Two to 64 shares of a tile of rows: teams of them that are whole, of one share, and one alone; the same
    outputs each time."""
    c = Case(torch_cuda, qctx, [keys], [40], 2, 1, d, 64, seed=keys)
    c.check()
    before = c.out.clone()
    for _ in range(3):
        c.check()
        assert torch_cuda.equal(before, c.out)
    c.check(window=keys // 2 + 3, sinks=2)
    c.free()


def test_many_requests(torch_cuda, qctx):
    rng = np.random.default_rng(5)
    lengths = rng.integers(1, 90, 3000)
    lengths[[0, 1500]] = 2500
    c = Case(torch_cuda, qctx, lengths.tolist(), [1] * 3000, 4, 2, 64, 16)
    c.check(single=True)
    c.free()
    rows = np.minimum(rng.integers(0, 4, 700), lengths[:700])
    c = Case(torch_cuda, qctx, lengths[:700].tolist(), rows.tolist(), 2, 1, 128, 32)
    c.check()
    c.check(window=20, sinks=2)
    c.free()


def test_a_prompt_from_nothing(torch_cuda, qctx):
    for n in (1, 31, 33, 129, 700, 2049):
        for heads, kv, d in ((2, 2, 128), (8, 1, 64)):
            c = Case(torch_cuda, qctx, [n], [n], heads, kv, d, 16, seed=n)
            c.check()
            c.check(causal=False)
            c.check(window=50, sinks=3)
            c.free()


def test_rows_that_see_nothing(torch_cuda, qctx):
    """More rows than tokens: those before the first token, and requests without any, give zeros; rows
    of no request stay as they were."""
    torch = torch_cuda
    c = Case(torch, qctx, [0, 5, 0, 40], [1, 9, 3, 2], 4, 2, 128, 16)
    d = Case(torch, qctx, [30], [300], 4, 2, 64, 32)
    for kw in (dict(), dict(window=5), dict(window=2 ** 31 - 1)):
        d.check(**kw)
    d.free()
    for kw in (dict(), dict(window=3, sinks=1), dict(window=10 ** 10), dict(window=2 ** 31 - 1, sinks=2), dict(causal=False)):
        c.pg.attention(0, c.call(rows=c.t + 3, out=torch.full((c.t + 3, 4 * 128), 7.0, dtype=torch.bfloat16, device="cuda"), **kw),
                       stream(torch))
        assert_near(torch, c.out[:c.t], *c.want(**kw))
        assert bool((c.out[c.t:] == 7.0).all()) and not c.out[0].any() and not c.out[10:13].any()
    c.free()


@pytest.mark.parametrize("bad", ["nan", "inf", "-inf", "mixed"])
@pytest.mark.parametrize("d", [64, 128])
def test_what_hidden_keys_hold(torch_cuda, qctx, bad, d):
    """Values and keys that are no numbers where a row does not see them: later tokens of the step,
    tokens before the window. Rows that see them get them."""
    torch = torch_cuda
    for rows in (1, 6, 90):
        c = Case(torch, qctx, [200, 333], [rows, min(rows, 7)], 4, 2, d, 32, seed=rows)
        values = {"nan": [float("nan")] * 3, "inf": [float("inf")] * 3, "-inf": [-float("inf")] * 3,
                  "mixed": [float("inf"), -float("inf"), float("nan")]}[bad]
        tok = [c.slots(0, 200), c.slots(1, 333)]
        for i, x in enumerate(values):  # values: one dim of an early token, one of the last, one in between
            c.v[tok[0][[20, 199, 200 - rows // 2 - 1][i]], 0, 5 + i] = x
            c.v[tok[1][[3, 332, 329][i]], 1, d - 1 - i] = x
        c.put()
        for kw in (dict(), dict(window=11, sinks=2), dict(window=150, sinks=30), dict(causal=False)):
            c.check(**kw)
        # a key that is no number: rows that see it are not compared, the others as ever
        c.v.nan_to_num_(1.0, 1.0, 1.0)
        c.k[tok[0][199], 0, 3] = c.k[tok[0][20], 1, 3] = float("nan")
        c.put()
        for kw in (dict(window=11, sinks=2), dict()):
            c.pg.attention(0, c.call(**kw), stream(torch))
            out = c.out.view(c.t, 4, d)
            want, mag = c.want(**kw)
            free = torch.ones(c.t, 4, dtype=torch.bool, device="cuda")
            free[rows - 1, :2] = False  # key head 0: the request's last row
            if not kw:
                free[:rows, 2:] = False
            assert_near(torch, out[free], want[free], mag[free])
            assert torch.isnan(out[~free]).all()
        c.free()


def test_tables_and_lengths_out_of_range(torch_cuda, qctx):
    """Entries outside the pages hide their keys; lengths past the table are cut to it; starts outside
    the rows are cut to them."""
    torch = torch_cuda
    for d in (64, 128):
        for rows in (1, 40):
            c = Case(torch, qctx, [300, 100], [rows, 1], 4, 1, d, 16)
            for i, x in ((2, -1), (3, c.pages), (7, 2 ** 31 - 1), (18, -2 ** 31)):
                c.tables[0, i] = x
            c.tables[1, :7] = -1
            c.check()
            c.check(causal=False)
            assert not c.out[rows].any()
            c.free()
    c = Case(torch, qctx, [160], [3], 2, 2, 64, 16)
    c.tables = c.tables[:, :10].contiguous()
    a = c.call()
    c.lengths_d.fill_(2 ** 31 - 1)
    c.pg.attention(0, a, stream(torch))
    assert_near(torch, c.out, *c.want())
    c.lengths_d.fill_(-4)
    c.pg.attention(0, a, stream(torch))
    assert not c.out.any()
    a = c.call(rows=2)
    c.starts_d.copy_(dev(torch, np.array([-3, 9], np.int32)))
    c.pg.attention(0, a, stream(torch))
    c.starts = np.array([0, 2], np.int32)
    c.q = c.q[:2]
    assert_near(torch, c.out[:2], *c.want())
    c.free()


def test_starts_that_overlap_leave_the_next_call_alone(torch_cuda, qctx):
    """Rows that several requests claim: more pieces than the rows can have; whatever is computed for them, a
    later call finds its counters as they should be."""
    torch = torch_cuda
    c = Case(torch, qctx, [9000, 70, 9000, 8000], [60, 50, 3, 40], 8, 2, 64, 16)
    c.check()
    for starts in ([0, 153, 0, 153, 153], [153, 0, 153, 0, 153], [-5, 400, -7, 2 ** 31 - 1, 3], [0, 153, 153, 0, 153]):
        a = c.call()
        c.starts_d.copy_(dev(torch, np.array(starts, np.int32)))
        for _ in range(2):
            c.pg.attention(0, a, stream(torch))
        torch.cuda.synchronize()
        c.check()
    c.free()


def test_strided_queries_and_scales(torch_cuda, qctx):
    """Queries inside a fused projection, and head-major as qk_norm_rope leaves them."""
    torch = torch_cuda
    c = Case(torch, qctx, [70, 300], [3, 40], 6, 3, 64, 16)
    fused = torch.full((c.t, 12 * 64 + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    fused[:, 8:8 + 6 * 64] = c.q.flatten(1)
    major = torch.full((6, c.t + 2, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    major[:, :c.t] = c.q.transpose(0, 1)
    for scale in (0.01, 0.25):
        want = c.want(scale=scale)
        for q, row, head in ((fused[:, 8:], fused.shape[1], 64), (major, 64, (c.t + 2) * 64)):
            c.pg.attention(0, c.call(scale=scale, q=q, q_row=row, q_head=head), stream(torch))
            assert_near(torch, c.out, *want)
    c.free()


def test_large_and_equal_scores(torch_cuda, qctx):
    """One key that takes nearly all, late and early; scores that are all equal."""
    torch = torch_cuda
    for at in (0, 700, 1499):
        c = Case(torch, qctx, [1500], [2], 4, 2, 128, 16)
        c.k[c.slots(0, 1500)[at]] = (c.q[1].view(2, 2, 128)[:, 0] * 3).to(torch.bfloat16)
        c.put()
        # |q k| scale reaches 1.5^2 3 128 / sqrt(128) = 76: the scores' error is 5 times the tolerance's share
        c.pg.attention(0, c.call(), stream(torch))
        want, mag = c.want()
        assert_near(torch, c.out, want, mag * (1 + 4 * 2.0 ** -5))
        c.free()
    c = Case(torch, qctx, [999], [3], 2, 1, 64, 32)
    c.q.zero_()
    c.check()
    c.free()


def test_a_layer_behind_32_bits(torch_cuda, qctx):
    """Pages, layers and rows of tables whose bytes and values lie past 2^32."""
    torch, kv, d, page = torch_cuda, 4, 128, 64
    pages = 36000  # a layer of 4.7e9 bytes
    pg = qctx.pages_create(2, pages, page, kv, d)
    gen = torch.Generator(device="cuda").manual_seed(0)
    n = 900
    table = torch.arange(pages - 15, pages, dtype=torch.int32, device="cuda").flip(0).contiguous()
    token = torch.arange(n, device="cuda")
    slots = (table.long()[token // page] * page + token % page).to(torch.int32)
    k, v = (torch.randn(n, kv, d, device="cuda", generator=gen).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(3, 8, d, device="cuda", generator=gen).to(torch.bfloat16)
    pg.store(1, k.data_ptr(), v.data_ptr(), qimm.BF16, n, slots.data_ptr(), stream=stream(torch))
    got = [torch.empty_like(k) for _ in range(2)]
    pg.load(1, got[0].data_ptr(), got[1].data_ptr(), n, slots.data_ptr(), stream(torch))
    assert torch.equal(got[0], k) and torch.equal(got[1], v)
    # the reference has the same tokens in pages of their own
    want = paged_ref.attention(torch, q, torch.cat([k, k[:60]]), torch.cat([v, v[:60]]), torch.arange(15, device="cuda")[None], [n], [0, 3], page, True)
    out = torch.empty(3, 8 * d, dtype=torch.bfloat16, device="cuda")
    lengths, starts = dev(torch, np.array([n], np.int32)), dev(torch, np.array([0, 3], np.int32))
    pg.attention(1, qimm.PagedAttention(q=q.data_ptr(), rows=3, heads=8, requests=1, max_pages=15, tables=table.data_ptr(),
                                        lengths=lengths.data_ptr(), starts=starts.data_ptr(), causal=1, scale=d ** -0.5,
                                        out=out.data_ptr()), stream(torch))
    assert_near(torch, out, *want)
    pg.free()


def test_attention_refuses(torch_cuda, qctx):
    torch = torch_cuda
    c = Case(torch, qctx, [20, 30], [2, 1], 4, 2, 64, 16)
    lib = qctx.lib
    for layer in (-1, 1):
        assert lib.qimm_attention_paged(c.pg.h, layer, qimm.C.byref(c.call()), None) == 2
    for field, value, status in [("rows", -1, 2), ("requests", -1, 2), ("requests", 65537, 2), ("max_pages", -1, 2), ("heads", 0, 2), ("heads", 3, 2),
                                 ("rows", 2 ** 30, 2), ("rows", 2 ** 29 - 64, 2), ("starts", None, 2), ("window", -1, 1), ("sinks", -1, 1), ("sinks", 2, 1), ("scale", 0.0, 1),
                                 ("scale", -1.0, 1), ("scale", float("nan"), 1), ("scale", float("inf"), 1), ("q", None, 1), ("out", None, 1),
                                 ("tables", None, 1), ("lengths", None, 1), ("q", c.q.data_ptr() + 2, 1), ("q_row", 260, 1), ("q_head", -64, 1)]:
        a = c.call()
        setattr(a, field, value)
        assert lib.qimm_attention_paged(c.pg.h, 0, qimm.C.byref(a), None) == status, (field, value)
        assert qctx.lib.qimm_last_error(qctx.h)
    a = c.call(causal=False)
    a.window = 4
    assert lib.qimm_attention_paged(c.pg.h, 0, qimm.C.byref(a), None) == 1
    a = c.call()
    a.rows = a.requests = 0
    a.starts = a.q = a.out = None
    assert lib.qimm_attention_paged(c.pg.h, 0, qimm.C.byref(a), None) == 0
    c.free()
