"""The page tables of a step and the store of rows into pages, against Python integers and the
rows themselves: all outputs are whole numbers or roundings, so they are equal."""
import numpy as np
import pytest

import paged_ref
import qimm
from gpu_util import dev, host, stream

pytestmark = pytest.mark.gpu


class Plan:
    """A step's device arrays; `same` writes lengths and state in place."""

    def __init__(self, torch, page, tables, lengths, added, queue, state, max_rows, same=False):
        n = len(lengths)
        self.tables, self.lengths, self.added = dev(torch, tables), dev(torch, lengths), dev(torch, added)
        self.queue, self.state = dev(torch, queue), dev(torch, state)
        self.lengths_out = self.lengths if same else torch.full_like(self.lengths, -99)
        self.state_out = self.state if same else torch.full((4,), -99, dtype=torch.int32, device="cuda")
        self.starts = torch.full((n + 1,), -99, dtype=torch.int32, device="cuda")
        self.slots, self.positions = (torch.full((max(max_rows, 1),), -99, dtype=torch.int32, device="cuda") for _ in range(2))
        self.work = torch.empty(qimm.page_plan_work(n), dtype=torch.int32, device="cuda")
        p = {f: getattr(self, f).data_ptr() for f in ("tables", "lengths", "added", "queue", "state", "lengths_out", "state_out",
                                                      "starts", "slots", "positions", "work")}
        self.call = qimm.PagePlan(page_size=page, pages=len(queue), requests=n, max_pages=tables.shape[1], max_rows=max_rows, **p)
        self.max_rows = max_rows

    def check(self, want):
        for f, g in (("tables", self.tables), ("lengths", self.lengths_out), ("queue", self.queue), ("state", self.state_out),
                     ("starts", self.starts), ("slots", self.slots[:self.max_rows]), ("positions", self.positions[:self.max_rows])):
            assert np.array_equal(host(g), want[f]), f


def a_case(rng, n, page, longest, most_new, short=0, rows_short=0):
    """Requests of random lengths with random steps, `short` pages too few, `rows_short` rows too few."""
    lengths = rng.integers(0, longest + 1, n)
    added = rng.choice([0, 1, 1, 1, -1, most_new], n) if most_new else np.ones(n, int)
    added = np.where((added > 1), rng.integers(1, max(most_new, 1) + 1, n), added)
    lengths, added = lengths.astype(np.int32), added.astype(np.int32)
    have = [paged_ref.pages_of(int(x), page) for x in lengths]
    after = [paged_ref.pages_of(int(x + max(a, 0)), page) for x, a in zip(lengths, added)]
    width = max(max(after), 1) + int(rng.integers(0, 3))
    pages = max(sum(after) + 3 - short, sum(have) + 1)
    perm = rng.permutation(pages).astype(np.int32)
    tables = rng.integers(-2 ** 31, 2 ** 31 - 1, (n, width)).astype(np.int32)
    at = 0
    for r, k in enumerate(have):
        tables[r, :k] = perm[at:at + k]
        at += k
    head, free = int(rng.integers(0, pages)), pages - at
    queue = rng.integers(-2 ** 31, 2 ** 31 - 1, pages).astype(np.int32)
    queue[(head + np.arange(free)) % pages] = perm[at:]
    rows = max(int(np.maximum(added, 0).sum()) + int(rng.integers(0, 70)) - rows_short, 0)
    return tables, lengths, added, queue, np.array([head, free, 0, 0], np.int32), rows


@pytest.mark.parametrize("same", [False, True])
@pytest.mark.parametrize("n,page,longest,most_new,short,rows_short", [
    (1, 16, 0, 1, 0, 0), (1, 48, 0, 700, 0, 0), (2, 16, 33, 0, 0, 0), (7, 16, 100, 40, 0, 0), (48, 64, 4299, 0, 0, 0),
    (48, 32, 500, 300, 9, 0), (65, 16, 200, 64, 0, 500), (300, 512, 5000, 2000, 3, 0), (1023, 16, 50, 5, 40, 0), (1024, 16, 50, 5, 0, 0),
    (1025, 32, 70, 40, 0, 99), (5000, 16, 40, 30, 100, 0), (20000, 128, 3, 1, 0, 0)])
def test_plan(torch_cuda, qctx, n, page, longest, most_new, short, rows_short, same):
    torch = torch_cuda
    case = a_case(np.random.default_rng(n + page), n, page, longest, most_new, short, rows_short)
    want = paged_ref.plan(page, len(case[3]), case[0], case[1], case[2], case[3], case[4], case[5])
    p = Plan(torch, page, *case, same=same)
    qctx.page_plan(p.call, stream(torch))
    p.check(want)
    if not same:  # a step that writes elsewhere can be made again
        qctx.page_plan(p.call, stream(torch))
        p.check(want)


@pytest.mark.parametrize("n,every", [(4096, 1), (4096, 300), (4097, 1), (4097, 300), (20000, 150)])
def test_plan_of_many_that_add_nothing(torch_cuda, qctx, n, every):
    """One request in `every` has a step: few rows lie thousands of requests apart."""
    torch = torch_cuda
    case = list(a_case(np.random.default_rng(n + every), n, 16, 40, 7))
    case[2][np.arange(n) % every != every - 1] = 0
    p = Plan(torch, 16, *case)
    qctx.page_plan(p.call, stream(torch))
    p.check(paged_ref.plan(16, len(case[3]), *case))


@pytest.mark.parametrize("n,rows", [(200, 0), (1000, 0), (1500, 7), (9000, 700), (65536, 0), (65536, 40)])
def test_plan_of_many_given_back(torch_cuda, qctx, n, rows):
    """Most requests give their pages back, up to a few that add a token."""
    torch = torch_cuda
    case = list(a_case(np.random.default_rng(n + rows), n, 16, 60, 0))
    case[2][:] = np.where(np.arange(n) % 11 == 3, 0, -1)
    case[2][np.random.default_rng(n).permutation(n)[:rows]] = 1
    case[5] = rows + 3 if rows else 0
    p = Plan(torch, 16, *case)
    qctx.page_plan(p.call, stream(torch))
    p.check(paged_ref.plan(16, len(case[3]), *case))


def test_plan_of_the_largest_chunk(torch_cuda, qctx):
    torch = torch_cuda
    page, new = 16, 300001
    pages = paged_ref.pages_of(new + 5, page) + 2
    case = (np.zeros((3, pages), np.int32), np.array([0, 5, 7], np.int32), np.array([0, new, 1], np.int32),
            np.random.default_rng(1).permutation(pages).astype(np.int32), np.array([pages - 1, pages, 0, 0], np.int32), new + 9)
    p = Plan(torch, page, *case)
    qctx.page_plan(p.call, stream(torch))
    p.check(paged_ref.plan(page, pages, *case))


@pytest.mark.parametrize("n", [3, 3000])
def test_plan_without_positions(torch_cuda, qctx, n):
    torch = torch_cuda
    case = a_case(np.random.default_rng(n), n, 16, 60, 9)
    p = Plan(torch, 16, *case)
    p.call.positions = None
    qctx.page_plan(p.call, stream(torch))
    want = paged_ref.plan(16, len(case[3]), *case)
    assert np.array_equal(host(p.slots), want["slots"]) and (p.positions == -99).all()


def test_plan_of_lengths_that_make_no_sense(torch_cuda, qctx):
    """Negative lengths, lengths past the table, sums past 32 bits, a state outside the queue: refused
    or cut, and nothing outside the arrays is touched."""
    torch = torch_cuda
    big = 2 ** 31 - 1
    tables = np.zeros((6, 2), np.int32)
    lengths = np.array([-5, 1000, big, 3, -1, 40], np.int32)
    added = np.array([1, 1, 1, big, -1, -7], np.int32)
    queue = np.arange(5, dtype=np.int32)
    for state in ([0, 5, 0, 0], [3, 0, 0, 0]):
        case = (tables, lengths, added, queue, np.array(state, np.int32), 8)
        p = Plan(torch, 16, *case)
        qctx.page_plan(p.call, stream(torch))
        want = paged_ref.plan(16, 5, *case)
        # pages given back that do not fit into the queue are not counted
        want["state"][1] = min(want["state"][1], 5)
        for f in ("lengths", "starts", "slots", "positions", "state"):
            assert np.array_equal(host({"lengths": p.lengths_out, "state": p.state_out}.get(f, getattr(p, f))), want[f]), f
    for state in ([-3, 2, 0, 0], [12, 3, 0, 0], [0, 99, 0, 0], [1, -4, 0, 0]):
        case = (tables, np.zeros(6, np.int32), np.ones(6, np.int32), queue, np.array(state, np.int32), 8)
        p = Plan(torch, 16, *case)
        qctx.page_plan(p.call, stream(torch))
        p.check(paged_ref.plan(16, 5, *case))


def test_plan_without_rows_or_pages(torch_cuda, qctx):
    """No row and no table entry to write; every request is left or refused."""
    torch = torch_cuda
    case = (np.zeros((3, 1), np.int32), np.array([3, 0, 2], np.int32), np.array([0, 1, -1], np.int32), np.arange(4, dtype=np.int32),
            np.array([1, 2, 0, 0], np.int32), 0)
    p = Plan(torch, 16, *case)
    p.call.slots = p.call.positions = None
    qctx.page_plan(p.call, stream(torch))
    want = paged_ref.plan(16, 4, *case)
    assert np.array_equal(host(p.lengths_out), want["lengths"]) and np.array_equal(host(p.state_out), want["state"])
    assert np.array_equal(host(p.queue), want["queue"]) and not host(p.starts).any()


def test_plan_refuses(torch_cuda, qctx):
    torch = torch_cuda
    case = a_case(np.random.default_rng(3), 4, 16, 30, 3)
    for field, value, status in [("page_size", 0, 2), ("page_size", 24, 2), ("page_size", 528, 2), ("pages", 0, 2), ("pages", 2 ** 27, 2),
                                 ("requests", 0, 2), ("requests", 65537, 2), ("max_pages", -1, 2), ("max_rows", -1, 2),
                                 ("max_rows", 2 ** 31, 2), ("tables", None, 1), ("lengths", None, 1), ("added", None, 1), ("queue", None, 1),
                                 ("state", None, 1), ("lengths_out", None, 1), ("state_out", None, 1), ("starts", None, 1),
                                 ("slots", None, 1), ("work", None, 1)]:
        p = Plan(torch, 16, *case)
        setattr(p.call, field, value)
        with pytest.raises(qimm.QimmError):
            qctx.page_plan(p.call, stream(torch))
        assert qctx.lib.qimm_page_plan(qctx.h, qimm.C.byref(p.call), None) == status, field


# ---------------- rows into pages and back ----------------

TYPES = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


def rounded(torch, x):
    return x.float().to(torch.bfloat16)


def slots_of(rng, page, pages, runs, t):
    """Runs of consecutive tokens of requests, starting anywhere, over pages in any order, then slots alone."""
    perm, out, at = rng.permutation(pages), [], 0
    for begin, n in runs:
        k = paged_ref.pages_of(begin + n, page)
        tok = np.arange(begin, begin + n)
        out += (perm[at + tok // page] * page + tok % page).tolist()
        at += k
    assert at <= pages and len(out) <= t
    return np.array(out + [-1] * (t - len(out)), np.int32)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("kv,d,page,runs,t", [
    (1, 64, 16, [(0, 1)], 1), (1, 128, 16, [(15, 2)], 2), (3, 128, 48, [(7, 61), (0, 1), (2, 1), (47, 3)], 70), (8, 128, 64, [(i * 3 % 64, 1) for i in range(48)], 48),
    (5, 64, 32, [(1, 130), (2, 131), (3, 133)], 401), (2, 64, 512, [(509, 520)], 520), (32, 128, 128, [(5, 700)], 703)])
def test_store_and_load(torch_cuda, qctx, kind, kv, d, page, runs, t):
    torch = torch_cuda
    rng = np.random.default_rng(t + d)
    pages = sum(paged_ref.pages_of(b + n, page) for b, n in runs) + 2
    pg = qctx.pages_create(2, pages, page, kv, d)
    assert 0 <= pg.device_bytes() - 2 * pages * page * kv * d * 4 < 1 << 27  # and the attention's scratch
    code = {"f32": qimm.F32, "f16": qimm.F16, "bf16": qimm.BF16}[kind]
    every = dev(torch, np.arange(pages * page, dtype=np.int32))
    gen = torch.Generator(device="cuda").manual_seed(t)
    back, new = [], []
    for n in (pages * page, t):
        back.append([torch.randn(n, kv, d, device="cuda", generator=gen).to(getattr(torch, TYPES[kind])) for _ in range(2)])
    # every slot of both layers first, then the rows into layer 1
    for layer in (0, 1):
        pg.store(layer, back[0][0].data_ptr(), back[0][1].data_ptr(), code, len(every), every.data_ptr(), stream=stream(torch))
    slots = slots_of(rng, page, pages, runs, t)
    slots_d = dev(torch, slots)
    pg.store(1, back[1][0].data_ptr(), back[1][1].data_ptr(), code, t, slots_d.data_ptr(), stream=stream(torch))
    for layer in (0, 1):
        got = [torch.full((pages * page, kv, d), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        pg.load(layer, got[0].data_ptr(), got[1].data_ptr(), len(every), every.data_ptr(), stream(torch))
        for i in range(2):
            want = rounded(torch, back[0][i])
            if layer:
                want[slots_d[slots_d >= 0].long()] = rounded(torch, back[1][i])[slots_d >= 0]
            assert torch.equal(got[i], want)
    got = [torch.full((t, kv, d), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    pg.load(1, got[0].data_ptr(), got[1].data_ptr(), t, slots_d.data_ptr(), stream(torch))
    for i in range(2):
        assert torch.equal(got[i], rounded(torch, back[1][i]) * (slots_d >= 0)[:, None, None])
    pg.free()


def test_store_of_slots_in_any_order(torch_cuda, qctx):
    """Reversed, shuffled, in steps, quads that lack a row, outside the pages on both sides."""
    torch, kv, d, page, pages = torch_cuda, 2, 128, 16, 40
    rng = np.random.default_rng(0)
    most = page * pages
    orders = [np.arange(most)[::-1], rng.permutation(most), np.arange(0, most, 4), np.arange(most)[np.arange(most) % 7 != 3],
              np.concatenate([[most, -1, 2 ** 31 - 1, -2 ** 31], np.arange(8), [most + 8], np.arange(9, 13)]), np.arange(3, 18)]
    for n, slots in enumerate(orders):
        pg = qctx.pages_create(1, pages, page, kv, d)
        s = dev(torch, slots.astype(np.int32))
        gen = torch.Generator(device="cuda").manual_seed(n)
        k, v = (torch.randn(len(s), kv, d, device="cuda", generator=gen).to(torch.bfloat16) for _ in range(2))
        pg.store(0, k.data_ptr(), v.data_ptr(), qimm.BF16, len(s), s.data_ptr(), stream=stream(torch))
        got = [torch.full((len(s), kv, d), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        pg.load(0, got[0].data_ptr(), got[1].data_ptr(), len(s), s.data_ptr(), stream(torch))
        ok = dev(torch, (slots >= 0) & (slots < most))[:, None, None]
        for x, y in zip(got, (k, v)):
            assert torch.equal(x, torch.where(ok, y, torch.zeros_like(y)))
        pg.free()


@pytest.mark.parametrize("kind", list(TYPES))
def test_store_of_strided_rows(torch_cuda, qctx, kind):
    """Rows inside a fused projection, and head-major rows as qk_norm_rope leaves them; special values."""
    torch, kv, d, page, t = torch_cuda, 3, 64, 16, 37
    code, dt = {"f32": qimm.F32, "f16": qimm.F16, "bf16": qimm.BF16}[kind], getattr(torch, TYPES[kind])
    gen = torch.Generator(device="cuda").manual_seed(1)
    fused = torch.randn(t, 9 * d + 8, device="cuda", generator=gen).to(dt)
    fused[0, :6] = torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 65504.0], device="cuda").to(dt)
    heads = torch.randn(kv, t + 5, d, device="cuda", generator=gen).to(dt)
    s = dev(torch, np.arange(1, t + 1, dtype=np.int32))
    pg = qctx.pages_create(1, 4, page, kv, d)
    size = fused.element_size()
    pg.store(0, heads.data_ptr(), fused.data_ptr() + 16 * 0 + 0 * size, code, t, s.data_ptr(), k_row=d, k_head=(t + 5) * d,
             v_row=9 * d + 8, v_head=2 * d, stream=stream(torch))
    k, v = (torch.empty(t, kv, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pg.load(0, k.data_ptr(), v.data_ptr(), t, s.data_ptr(), stream(torch))
    want_v = torch.stack([fused[:, 2 * d * i:2 * d * i + d] for i in range(kv)], 1)
    assert torch.equal(k, rounded(torch, heads[:, :t].transpose(0, 1)))
    w = rounded(torch, want_v)
    assert torch.equal(torch.isnan(v), torch.isnan(w)) and torch.equal(v.nan_to_num(3.0), w.nan_to_num(3.0))
    assert torch.equal(v.view(torch.int16)[0, 0, 3:5], w.view(torch.int16)[0, 0, 3:5])
    pg.free()


def test_pages_refuse(torch_cuda, qctx):
    torch = torch_cuda
    for args in [(0, 4, 16, 1, 128), (1, 0, 16, 1, 128), (1, 4, 24, 1, 128), (1, 4, 0, 1, 128), (1, 4, 1024, 1, 128), (1, 4, 16, 0, 128),
                 (1, 4, 16, 65536, 128), (1, 4, 16, 1, 96), (1, 4, 16, 1, 256), (1, 2 ** 27, 16, 1, 64), (1, 2 ** 22, 512, 32, 64)]:
        with pytest.raises(qimm.QimmError) as e:
            qctx.pages_create(*args)
        assert "QIMM_ERR_SHAPE" in str(e.value)
    with pytest.raises(qimm.QimmError) as e:
        qctx.pages_create(2 ** 55, 4, 16, 1, 128)
    assert "QIMM_ERR_OOM" in str(e.value)
    pg = qctx.pages_create(2, 4, 16, 2, 64)
    x = torch.zeros(4096, device="cuda")
    s = torch.zeros(8, dtype=torch.int32, device="cuda")
    lib, a, b = qctx.lib, x.data_ptr(), s.data_ptr()
    ok = dict(layer=0, k=a, v=a, type=qimm.F32, rows=1, k_row=0, k_head=0, v_row=0, v_head=0, slots=b)
    for change, status in [(dict(layer=-1), 2), (dict(layer=2), 2), (dict(type=qimm.Q8_0), 3), (dict(type=7), 3), (dict(k=None), 1),
                           (dict(v=None), 1), (dict(slots=None), 1), (dict(rows=-1), 1), (dict(k=a + 4), 1), (dict(v=a + 8), 1),
                           (dict(k_row=66), 1), (dict(v_head=-64), 1), (dict(type=qimm.BF16, k_head=68), 1), (dict(rows=2 ** 31), 2)]:
        c = {**ok, **change}
        assert lib.qimm_pages_store(pg.h, *[c[f] for f in ok], None) == status, change
    for args, status in [((-1, a, a, 1, b), 2), ((2, a, a, 1, b), 2), ((0, None, a, 1, b), 1), ((0, a, a + 2, 1, b), 1), ((0, a, a, 1, None), 1),
                         ((0, a, a, -1, b), 1)]:
        assert lib.qimm_pages_load(pg.h, *args, None) == status, args
    assert lib.qimm_pages_store(pg.h, 0, None, None, qimm.F32, 0, 0, 0, 0, 0, None, None) == 0
    assert lib.qimm_pages_load(pg.h, 0, None, None, 0, None, None) == 0
    pg.free()
