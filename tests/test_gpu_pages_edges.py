"""GPU: reserve and compact around the numbers of columns, pages and sequences at which they take another way, against the
oracle, bit for bit."""
import pytest
import torch

from oracle import paged_oracle as oracle
from prefixlm import PagedKVCache, paged_kvcache_compact, paged_kvcache_reserve

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _to(cache):
    return PagedKVCache(*(x.to(DEV) for x in cache))


def _same(got, want):
    for name, a, b in zip(PagedKVCache._fields, got, want):
        assert torch.equal(a.cpu(), b), (name, (a.cpu() != b).nonzero()[:5].tolist())


@pytest.mark.parametrize("P", [3000, 16384, 16385])
@pytest.mark.parametrize("W", [1, 1023, 1024, 1025, 2048])
def test_reserve_by_columns(W, P):
    """W columns ask: of pages that two to five sequences share, some of them all among these, and of none."""
    g = torch.Generator().manual_seed(W + P)
    ps, M = 16, 2
    lens = torch.randint(1, 16, (W,), generator=g, dtype=torch.int32)
    cache = oracle.dealt(1, P, 1, ps, 64, W, M, [0] * W, g)
    table, refs = cache[3], cache[2]
    table[:, 0] = torch.randperm(P, generator=g)[:max(1, W // 3)].int()[torch.randint(0, max(1, W // 3), (W,), generator=g)]
    table[torch.rand(W, generator=g) < 0.2, 0] = -1
    refs[:] = torch.bincount(table[:, 0][table[:, 0] >= 0].long(), minlength=P)
    refs[table[: W // 5, 0].clamp_min(0).long()] += (table[: W // 5, 0] >= 0).int()     # held outside the table too
    refs[torch.rand(P, generator=g) < 0.3] += 1
    dev = _to(cache)
    short = paged_kvcache_reserve(dev, lens.to(DEV), 1)
    want, left = oracle.reserve(cache, lens, 1)
    _same(dev, want)
    assert torch.equal(short.cpu(), left)


def test_reserve_of_the_most_sequences():
    N, ps, P = 8192, 16, 20000
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 40, (N,), generator=g, dtype=torch.int32)
    new = torch.where(torch.rand(N, generator=g) < 0.9, 0, torch.randint(1, 40, (N,), generator=g)).int()
    cache = oracle.dealt(1, P, 1, ps, 64, N, 5, lens.tolist(), g)
    for new in (new, torch.where(torch.arange(N) == N - 1, 5, 0).int(), torch.zeros(N, dtype=torch.int32)):
        dev = _to(cache)
        short = paged_kvcache_reserve(dev, lens.to(DEV), new.to(DEV))
        want, left = oracle.reserve(cache, lens, new)
        _same(dev, want)
        assert torch.equal(short.cpu(), left)


@pytest.mark.parametrize("share", [0.01, 0.5, 0.99])
@pytest.mark.parametrize("P", [16383, 16384, 16385, 32768])
def test_compact_by_pages(P, share):
    """As many pages as stay in registers, and one more; half in use is the most that can move."""
    g = torch.Generator().manual_seed(P)
    N, M = 64, 256
    cache = oracle.dealt(1, P, 1, 16, 64, N, M, [0] * N, g)
    used = torch.randperm(P, generator=g)[:int(P * share)] if share != 0.5 else torch.arange(P // 2, P)
    table = used[torch.randint(0, used.numel(), (N, M), generator=g)]
    cache[3][:] = table
    cache[2][used] = 1
    cache[2] += torch.bincount(table.view(-1), minlength=P).int()
    dev = _to(cache)
    n = paged_kvcache_compact(dev)
    want, u = oracle.compact(cache)
    _same(dev, want)
    assert n.tolist() == [u]
