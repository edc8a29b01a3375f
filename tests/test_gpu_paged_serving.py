"""The paged cache as a server of requests uses it: steps in which requests come, go on and are given back,
by themselves, replayed from a graph, on streams of their own and two at once; the attention's keys
as the norm and RoPE kernel leaves them, and image tokens over prompts of their own lengths."""
import numpy as np
import pytest

import oracle as O
import paged_ref
import qimm
from gpu_util import bf16_dev, dev, host, stream
from paged_ref import assert_near

pytestmark = pytest.mark.gpu


class Server:
    """Page tables, queue and a cache for up to n requests; every array is the program's own."""

    def __init__(self, torch, ctx, n, pages, page, heads, kv, d, max_rows, max_pages):
        def zeros(*shape):
            return torch.zeros(*shape, dtype=torch.int32, device="cuda")

        self.torch, self.ctx, self.n, self.page, self.heads, self.kv, self.d, self.max_rows = torch, ctx, n, page, heads, kv, d, max_rows
        self.pg = ctx.pages_create(1, pages, page, kv, d)
        self.tables, self.lengths, self.added = zeros(n, max_pages), zeros(n), zeros(n)
        self.queue, self.state = torch.randperm(pages, device="cuda").to(torch.int32), zeros(4)
        self.state[1] = pages
        self.starts, self.slots, self.positions = zeros(n + 1), zeros(max_rows), zeros(max_rows)
        self.work = zeros(qimm.page_plan_work(n))
        self.q = torch.zeros(max_rows, heads, d, dtype=torch.bfloat16, device="cuda")
        self.k, self.v = (torch.zeros(max_rows, kv, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.out = torch.full((max_rows, heads, d), 7.0, dtype=torch.bfloat16, device="cuda")

    def step(self, s, window=0, sinks=0):
        at = {f: getattr(self, f).data_ptr() for f in ("tables", "lengths", "added", "queue", "state", "starts", "slots", "positions", "work")}
        self.ctx.page_plan(qimm.PagePlan(page_size=self.page, pages=len(self.queue), requests=self.n, max_pages=self.tables.shape[1],
                                         max_rows=self.max_rows, lengths_out=at["lengths"], state_out=at["state"], **at), s)
        self.pg.store(0, self.k.data_ptr(), self.v.data_ptr(), qimm.BF16, self.max_rows, at["slots"], stream=s)
        self.pg.attention(0, qimm.PagedAttention(q=self.q.data_ptr(), rows=self.max_rows, heads=self.heads, requests=self.n,
                                                 max_pages=self.tables.shape[1], tables=at["tables"], lengths=at["lengths"],
                                                 starts=at["starts"], causal=1, window=window, sinks=sinks, scale=self.d ** -0.5,
                                                 out=self.out.data_ptr()), s)


class Requests:
    """What the host knows of the requests: their keys and values so far."""

    def __init__(self, torch, srv, seed):
        self.torch, self.srv, self.rng = torch, srv, np.random.default_rng(seed)
        self.kv = [[] for _ in range(srv.n)]
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def next(self, longest, chunk):
        """A step's `added`; the rows' queries, keys and values into the server's arrays."""
        srv, rows = self.srv, 0
        added = []
        for r in range(srv.n):
            n = sum(len(k) for k, _ in self.kv[r])
            if n == 0:
                a = int(self.rng.integers(1, chunk + 1)) if self.rng.random() < 0.4 else 0
            else:
                a = -1 if n > longest or self.rng.random() < 0.04 else int(self.rng.choice([1, 1, 1, 0, 3, chunk // 2]))
            if a > 0 and rows + a > srv.max_rows:
                a = 0
            rows += max(a, 0)
            added.append(a)
        for x in (srv.q, srv.k, srv.v):
            x.copy_(self.torch.randn(x.shape, device="cuda", generator=self.gen))
        srv.added.copy_(self.torch.tensor(added, dtype=self.torch.int32))
        return added

    def check(self, added, window=0, sinks=0):
        """The step's outputs against 64 bits over the dense history, its arrays against each other."""
        torch, srv = self.torch, self.srv
        lengths, starts = host(srv.lengths).tolist(), host(srv.starts).tolist()
        for r, a in enumerate(added):
            before = sum(len(k) for k, _ in self.kv[r])
            if a < 0:
                self.kv[r] = []
            served = a > 0 and lengths[r] == before + a
            if a > 0 and not served:
                assert lengths[r] == before and (srv.slots[starts[r]:starts[r + 1]] == -1).all()
            if served:
                lo, hi = starts[r], starts[r + 1]
                assert hi - lo == a and host(srv.positions[lo:hi]).tolist() == list(range(before, before + a))
                self.kv[r].append((srv.k[lo:hi].clone(), srv.v[lo:hi].clone()))
                k, v = (torch.cat([x[i] for x in self.kv[r]]) for i in range(2))
                n = len(k)
                table = torch.arange(paged_ref.pages_of(n, 16), device="cuda")[None]
                pad = (0, 0, 0, 0, 0, -n % 16)
                want = paged_ref.attention(torch, srv.q[lo:hi], torch.nn.functional.pad(k, pad), torch.nn.functional.pad(v, pad), table, [n],
                                           [0, a], 16, True, window, sinks)
                assert_near(torch, srv.out[lo:hi], *want)
            assert lengths[r] == sum(len(k) for k, _ in self.kv[r])
        # every page is held once or free
        tables, queue, state = host(srv.tables), host(srv.queue), host(srv.state)
        held = [tables[r, :paged_ref.pages_of(n, srv.page)] for r, n in enumerate(lengths)]
        free = queue[(state[0] + np.arange(state[1])) % len(queue)]
        assert sorted(np.concatenate(held + [free]).tolist()) == list(range(len(queue)))
        assert (srv.slots[starts[-1]:] == -1).all() and state[2] == starts[-1]


@pytest.mark.parametrize("page,heads,kv,d,window,sinks", [(16, 8, 2, 128, 0, 0), (48, 4, 4, 64, 0, 0), (32, 6, 1, 128, 40, 3)])
def test_requests_come_and_go(torch_cuda, qctx, page, heads, kv, d, window, sinks):
    """Some steps find too few pages: requests are refused and come again."""
    torch = torch_cuda
    srv = Server(torch, qctx, 9, 2400 // page, page, heads, kv, d, 300, 700 // page + 1)
    req, refused = Requests(torch, srv, page), 0
    for i in range(40):
        added = req.next(600, 140)
        srv.step(stream(torch), window, sinks)
        req.check(added, window, sinks)
        refused += int(srv.state[3])
    assert refused > 0
    srv.pg.free()


@pytest.mark.parametrize("heads,kv,d", [(8, 2, 128), (2, 2, 64)])
def test_a_captured_step(torch_cuda, qctx, heads, kv, d):
    """One graph for all steps, its arrays updated in place; eager work of the program between the replays.
    A second server makes the same steps eagerly: bit for bit the same."""
    torch = torch_cuda
    a, b = (Server(torch, qctx, 7, 150, 16, heads, kv, d, 200, 60) for _ in range(2))
    b.queue.copy_(a.queue)
    req = Requests(torch, a, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # the step once before, on arrays that are put back
        keep = [x.clone() for x in (a.tables, a.lengths, a.queue, a.state)]
        a.step(side.cuda_stream)
        for x, y in zip((a.tables, a.lengths, a.queue, a.state), keep):
            x.copy_(y)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(stream(torch))
    a.out.fill_(7.0)
    for i in range(25):
        added = req.next(500, 90)
        for x, y in zip((b.added, b.q, b.k, b.v), (a.added, a.q, a.k, a.v)):
            x.copy_(y)
        if i % 3 == 0:
            torch.cuda.synchronize()
        graph.replay()
        junk = torch.randn(512, 512, device="cuda") @ torch.randn(512, 512, device="cuda")
        b.step(stream(torch))
        assert torch.isfinite(junk).all()
        for f in ("tables", "lengths", "queue", "state", "starts", "slots", "positions", "out"):
            assert torch.equal(getattr(a, f), getattr(b, f)), f
        req.check(added)
    a.pg.free()
    b.pg.free()


def test_long_requests_replayed(torch_cuda, qctx):
    """Requests that are split into shares, of single tokens and of rows, from a graph: every replay finds
    the counters as it needs them, whatever lengths the one before had."""
    torch, heads, kv, d, page = torch_cuda, 8, 2, 128, 64
    pages = 700
    pg = qctx.pages_create(1, pages, page, kv, d)
    gen = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(pages * page, kv, d, device="cuda", generator=gen).to(torch.bfloat16) for _ in range(2))
    every = torch.arange(pages * page, dtype=torch.int32, device="cuda")
    pg.store(0, k.data_ptr(), v.data_ptr(), qimm.BF16, len(every), every.data_ptr(), stream=stream(torch))
    tables = torch.randperm(pages, device="cuda", generator=gen)[:690].to(torch.int32).reshape(3, 230).contiguous()
    lengths, starts = dev(torch, np.array([14000, 9000, 100], np.int32)), dev(torch, np.array([0, 1, 31, 32], np.int32))
    q = torch.randn(32, heads, d, device="cuda", generator=gen).to(torch.bfloat16)
    out = torch.empty(32, heads * d, dtype=torch.bfloat16, device="cuda")
    call = qimm.PagedAttention(q=q.data_ptr(), rows=32, heads=heads, requests=3, max_pages=230, tables=tables.data_ptr(),
                               lengths=lengths.data_ptr(), starts=starts.data_ptr(), causal=1, scale=d ** -0.5, out=out.data_ptr())
    pg.attention(0, call, stream(torch))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pg.attention(0, call, stream(torch))
    for n in ([14000, 9000, 100], [1, 14720, 14000], [600, 700, 14001], [14720, 14720, 14720], [14000, 9000, 100]):
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        first = out.clone()
        assert_near(torch, out, *paged_ref.attention(torch, q, k, v, tables, n, [0, 1, 31, 32], page, True))
        out.fill_(3.0)
        pg.attention(0, call, stream(torch))
        assert torch.equal(out, first)
    pg.free()


def test_two_servers_at_once(torch_cuda):
    """Two contexts, two caches, two streams, no order between them."""
    torch = torch_cuda
    ctxs = [qimm.Context(0), qimm.Context(0)]
    servers = [Server(torch, c, 5, 300, 16, 8, 2, 128, 260, 80) for c in ctxs]
    reqs = [Requests(torch, s, i) for i, s in enumerate(servers)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(15):
        added = [r.next(900, 200) for r in reqs]
        torch.cuda.synchronize()
        for s, st in zip(servers, streams):
            s.step(st.cuda_stream)
        torch.cuda.synchronize()
        for r, a in zip(reqs, added):
            r.check(a)
    for s in servers:
        s.pg.free()
    torch.cuda.synchronize()
    for c in ctxs:
        c.close()


def test_keys_of_the_norm_and_rope_kernel(torch_cuda, qctx):
    """A step's rows at their requests' positions: the plan's positions pick the RoPE rows, the kernel's
    head-major keys and queries go into the pages and the attention by their strides."""
    torch, heads, kv, d = torch_cuda, 4, 4, 128
    srv = Server(torch, qctx, 3, 60, 16, heads, kv, d, 90, 20)
    srv.lengths.copy_(torch.tensor([0, 33, 100], dtype=torch.int32))
    srv.tables[1, :3] = srv.queue[:3]
    srv.tables[2, :7] = srv.queue[3:10]
    srv.state[0], srv.state[1] = 10, 50
    rng = np.random.default_rng(0)
    pe = O.rope_table([(1, 1, 1)], [0] * 200 + [1])[:200]
    pe_d = dev(torch, np.ascontiguousarray(pe))
    w = dev(torch, (1 + 0.1 * rng.standard_normal(d)).astype(np.float32))
    gen = torch.Generator(device="cuda").manual_seed(1)
    # what the requests hold so far
    old = torch.randn(2, 200, kv, d, device="cuda", generator=gen).to(torch.bfloat16)
    for r, n in ((1, 33), (2, 100)):
        tok = torch.arange(n, device="cuda")
        s = (srv.tables[r].long()[tok // 16] * 16 + tok % 16).to(torch.int32)
        srv.pg.store(0, old[0].data_ptr(), old[1].data_ptr(), qimm.BF16, n, s.data_ptr(), stream=stream(torch))
    srv.added.copy_(torch.tensor([40, 1, 7], dtype=torch.int32))
    at = {f: getattr(srv, f).data_ptr() for f in ("tables", "lengths", "added", "queue", "state", "starts", "slots", "positions", "work")}
    qctx.page_plan(qimm.PagePlan(page_size=16, pages=60, requests=3, max_pages=20, max_rows=90, lengths_out=at["lengths"], state_out=at["state"], **at),
                   stream(torch))
    rows = 48
    x = torch.randn(3, rows, heads, d, device="cuda", generator=gen)
    rows_pe = pe_d[srv.positions[:rows].long()].contiguous()
    q, k = (torch.empty(heads, rows, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for src, dst in ((x[0], q), (x[1], k)):
        qctx.qk_norm_rope(src.contiguous().data_ptr(), 1, rows, heads, w.data_ptr(), rows_pe.data_ptr(), dst.data_ptr(), stream(torch))
    # keys head-major in bf16, values token-major in f32: two calls of one store each
    v16 = x[2].to(torch.bfloat16)
    srv.pg.store(0, k.data_ptr(), v16.contiguous().data_ptr(), qimm.BF16, rows, at["slots"], k_row=d, k_head=rows * d, stream=stream(torch))
    out = torch.empty(rows, heads * d, dtype=torch.bfloat16, device="cuda")
    srv.pg.attention(0, qimm.PagedAttention(q=q.data_ptr(), q_row=d, q_head=rows * d, rows=rows, heads=heads, requests=3, max_pages=20,
                                            tables=at["tables"], lengths=at["lengths"], starts=at["starts"], causal=1, scale=d ** -0.5,
                                            out=out.data_ptr()), stream(torch))
    starts = host(srv.starts).tolist()
    assert starts == [0, 40, 41, 48]
    for r, n in enumerate((0, 33, 100)):
        lo, hi = starts[r], starts[r + 1]
        kk = torch.cat([old[0, :n], k[:, lo:hi].transpose(0, 1)])
        vv = torch.cat([old[1, :n], v16[lo:hi]])
        pad = (0, 0, 0, 0, 0, -len(kk) % 16)
        table = torch.arange(paged_ref.pages_of(len(kk), 16), device="cuda")[None]
        # the queries' norms are sqrt(128) times the weights: |q k| scale up to 128 * 1.3^2 / sqrt(128) = 19
        want, mag = paged_ref.attention(torch, q[:, lo:hi].transpose(0, 1), torch.nn.functional.pad(kk, pad), torch.nn.functional.pad(vv, pad),
                                        table, [len(kk)], [0, hi - lo], 16, True)
        assert_near(torch, out[lo:hi], want, mag * 1.05)
    srv.pg.free()


def test_image_tokens_over_their_own_prompts(torch_cuda, qctx):
    """Every image's tokens over its prompt's pages and themselves, no mask: what the dense attention gives
    for each request alone, which a batch of it would pad to the longest prompt."""
    torch, heads, d, page, s = torch_cuda, 4, 128, 32, 256
    prompts = [7, 200, 77]
    srv = Server(torch, qctx, 3, 60, page, heads, heads, d, 3 * s, 20)
    gen = torch.Generator(device="cuda").manual_seed(4)

    def draw(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(torch.bfloat16)

    total = [n + s for n in prompts]
    srv.added.copy_(torch.tensor(total, dtype=torch.int32))
    srv.max_rows = sum(total)
    srv.slots, srv.positions = (torch.zeros(sum(total), dtype=torch.int32, device="cuda") for _ in range(2))
    at = {f: getattr(srv, f).data_ptr() for f in ("tables", "lengths", "added", "queue", "state", "starts", "slots", "positions", "work")}
    qctx.page_plan(qimm.PagePlan(page_size=page, pages=60, requests=3, max_pages=20, max_rows=sum(total), lengths_out=at["lengths"],
                                 state_out=at["state"], **at), stream(torch))
    k, v, q = draw(sum(total), heads, d), draw(sum(total), heads, d), draw(3, heads, s, d)
    srv.pg.store(0, k.data_ptr(), v.data_ptr(), qimm.BF16, sum(total), at["slots"], stream=stream(torch))
    out = torch.empty(3 * s, heads * d, dtype=torch.bfloat16, device="cuda")
    starts = dev(torch, np.array([0, s, 2 * s, 3 * s], np.int32))
    rows = q.transpose(1, 2).contiguous()
    srv.pg.attention(0, qimm.PagedAttention(q=rows.data_ptr(), rows=3 * s, heads=heads, requests=3, max_pages=20, tables=at["tables"],
                                            lengths=at["lengths"], starts=starts.data_ptr(), causal=0, scale=d ** -0.5,
                                            out=out.data_ptr()), stream(torch))
    first = 0
    for r, n in enumerate(total):
        kk, vv = k[first:first + n], v[first:first + n]
        pad = (0, 0, 0, 0, 0, -n % 16)
        table = torch.arange(paged_ref.pages_of(n, 16), device="cuda")[None]
        want, mag = paged_ref.attention(torch, rows[r], torch.nn.functional.pad(kk, pad), torch.nn.functional.pad(vv, pad), table, [n], [0, s], 16, False)
        assert_near(torch, out[r * s:(r + 1) * s], want, mag)
        dense = torch.empty(1, s, heads * d, dtype=torch.bfloat16, device="cuda")
        ko, vto = kk.transpose(0, 1).contiguous(), vv.permute(1, 2, 0).contiguous()
        qctx.attention(q[r].data_ptr(), 1, heads, s, None, 0, ko.data_ptr(), vto.data_ptr(), n, d ** -0.5, dense.data_ptr(), stream(torch))
        # both within the tolerance of the same values
        assert ((dense.double().view(s, heads, d) - out[r * s:(r + 1) * s].double().view(s, heads, d)).abs() <= 2 * paged_ref.TOL * mag + 1e-30).all()
        first += n
    srv.pg.free()


def test_steps_without_rows(torch_cuda, qctx):
    """A step in which no request has a row: nothing is written."""
    torch = torch_cuda
    srv = Server(torch, qctx, 4, 10, 16, 4, 2, 64, 12, 3)
    srv.step(stream(torch))
    assert (srv.slots == -1).all() and not srv.starts.any() and (srv.out == 7.0).all() and srv.state.tolist() == [0, 10, 0, 0]
    srv.added.fill_(-1)
    srv.step(stream(torch))
    assert not srv.lengths.any() and srv.state.tolist() == [0, 10, 0, 0]
    srv.pg.free()
