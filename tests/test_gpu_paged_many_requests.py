"""Attention over the paged cache for batches of more than 64 requests, where the pieces are counted by the
workgroup: chunks and single tokens mixed, both forms divided over their keys."""
import numpy as np
import pytest

from gpu_util import stream
from test_gpu_paged_attention import Case

pytestmark = pytest.mark.gpu


def batch(n, seed, long):
    """n requests: one in eight with a chunk, a few without rows, `long` of them over thousands of keys."""
    rng = np.random.default_rng(seed)
    rows = np.where(rng.integers(0, 8, n) == 3, rng.integers(2, 90, n), 1)
    rows[rng.integers(0, n, n // 20)] = 0
    lengths = rows + rng.integers(0, 200, n)
    for i in range(long):
        at = (i * 29 + 7) % n
        lengths[at], rows[at] = rng.integers(2000, 9000), (140, 1, 33)[i % 3]
    lengths[n - 1], rows[n - 1] = 3001, 150
    return lengths.tolist(), rows.tolist()


@pytest.mark.parametrize("n", [65, 257, 700])
@pytest.mark.parametrize("heads,kv,d,page", [(4, 1, 128, 32), (6, 2, 64, 16), (2, 2, 128, 64)])
def test_chunks_and_tokens(torch_cuda, qctx, n, heads, kv, d, page):
    lengths, rows = batch(n, n + heads, 6)
    c = Case(torch_cuda, qctx, lengths, rows, heads, kv, d, page, seed=n)
    for kw in (dict(), dict(window=700, sinks=5), dict(causal=False)):
        c.check(**kw)
        before = c.out.clone()
        c.pg.attention(0, c.call(**kw), stream(torch_cuda))
        assert torch_cuda.equal(before, c.out)
    c.free()


@pytest.mark.parametrize("heads,kv,d", [(4, 1, 128), (8, 4, 64)])
@pytest.mark.parametrize("long", [0, 2, 12])
def test_64_and_65_requests(torch_cuda, qctx, heads, kv, d, long):
    """The same 64 requests counted by the waves, and with one more of no rows by the workgroup."""
    torch = torch_cuda
    lengths, rows = batch(64, 3 + long, long)
    c = Case(torch, qctx, lengths + [5], rows + [0], heads, kv, d, 16)
    for kw in (dict(), dict(window=900, sinks=3), dict(causal=False)):
        c.check(**kw)
        before = c.out.clone()
        a = c.call(**kw)
        a.requests = 64
        c.pg.attention(0, a, stream(torch))
        assert torch.equal(before, c.out)
    c.free()


def test_long_tokens_among_many(torch_cuda, qctx):
    """Single tokens alone, without starts; a few over tens of thousands of keys."""
    rng = np.random.default_rng(1)
    lengths = rng.integers(0, 60, 300)
    lengths[[3, 150, 299]] = [30000, 9001, 16384]
    for d, heads, kv in ((64, 4, 4), (128, 8, 1)):
        c = Case(torch_cuda, qctx, lengths.tolist(), [1] * 300, heads, kv, d, 64)
        c.check(single=True)
        c.check(single=True, window=8000, sinks=2)
        c.free()


def test_prompts_of_a_large_batch(torch_cuda, qctx):
    """More tiles than workgroups run at once: nothing is divided; some prompts are whole, some continued."""
    rng = np.random.default_rng(2)
    rows = rng.integers(100, 200, 90)
    lengths = rows + np.where(np.arange(90) % 2, 0, rng.integers(0, 900, 90))
    c = Case(torch_cuda, qctx, lengths.tolist(), rows.tolist(), 16, 4, 128, 48)
    c.check()
    c.check(window=64)
    c.free()
