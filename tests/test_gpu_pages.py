"""GPU: handing out, sharing, freeing, moving and copying pages against the oracle, all bit for bit."""
import pytest
import torch

from oracle import paged_oracle as oracle
from prefixlm import (PagedKVCache, paged_kvcache, paged_kvcache_compact, paged_kvcache_copy, paged_kvcache_fork,
                      paged_kvcache_free, paged_kvcache_reserve)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _to(cache):
    return PagedKVCache(*(x.to(DEV) for x in cache))


def _same(got, want, tag=""):
    for name, a, b in zip(PagedKVCache._fields, got, want):
        assert torch.equal(a.cpu(), b), (tag, name, (a.cpu() != b).nonzero()[:5].tolist())


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _int(g, lo, hi, n):
    return torch.randint(lo, hi, (n,), generator=g, dtype=torch.int32)


SHAPES = [(1, 1, 16, 64), (2, 3, 16, 128), (1, 2, 64, 128), (3, 1, 256, 64)]


@pytest.mark.parametrize("L,H,ps,D", SHAPES)
@pytest.mark.parametrize("N", [1, 7, 33])
def test_reserve(N, L, H, ps, D):
    """Sequences that share pages in every way, at lengths inside and at the ends of pages."""
    M = 6
    for seed in range(4):
        g = _gen(seed)
        lens = _int(g, 0, M * ps + 1, N)
        lens[::3] = lens[::3] // ps * ps
        cache = oracle.dealt(L, N * M + 5, H, ps, D, N, M, lens.tolist(), g)
        parents = _int(g, -1, N, N)
        cache = oracle.fork(cache, parents)
        lens = torch.where(parents >= 0, lens[parents.clamp_min(0).long()], lens)
        new = torch.where(torch.rand(N, generator=g) < 0.3, 0, _int(g, 1, 2 * ps, N)).int()
        dev = _to(cache)
        short = paged_kvcache_reserve(dev, lens.to(DEV), new.to(DEV))
        want, left = oracle.reserve(cache, lens, new)
        _same(dev, want, seed)
        assert torch.equal(short.cpu(), left) and not left.any()


def test_reserve_when_pages_run_out():
    """Those before the end of the supply get theirs; what is left is counted, shared pages that stay
    shared among it."""
    L, H, ps, D, N, M = 1, 1, 16, 64, 12, 8
    some = 0
    for seed in range(8):
        g = _gen(50 + seed)
        lens = _int(g, 0, 100, N)
        cache = oracle.dealt(L, N * M, H, ps, D, N, M, lens.tolist(), g)
        cache = oracle.fork(cache, _int(g, -1, N, N))
        cache[2][(cache[2] == 0).nonzero()[seed + 1:, 0]] = 1       # others hold all but a few
        new = _int(g, 0, 30, N)
        dev = _to(cache)
        short = paged_kvcache_reserve(dev, lens.to(DEV), new.to(DEV))
        want, left = oracle.reserve(cache, lens, new)
        _same(dev, want, seed)
        assert torch.equal(short.cpu(), left)
        some += int(left.sum())
    assert some


def test_reserve_odd_lengths_and_entries():
    """Lengths and rows outside the table, negative and past 32 bits; entries that are no page; ints."""
    ps, N, M, P = 16, 9, 3, 40
    g = _gen(1)
    cache = oracle.dealt(2, P, 1, ps, 64, N, M, [48] * N, g)
    cache[3][2] = torch.tensor([P, -7, 2**31 - 1])
    cache[2][:] = torch.bincount(cache[3][(cache[3] >= 0) & (cache[3] < P)].long(), minlength=P)
    lens = torch.tensor([0, 5, 10, 48, 47, -3, 2**31 - 1, 16, 40], dtype=torch.int32)
    new = torch.tensor([2**31 - 1, -1, 100, 4, 1, 20, 5, -2**31, 0], dtype=torch.int32)
    for a, m in ((lens, new), (lens.long() * 2**20, new), (7, 11), (0, 2**31 - 1), (lens, 3), (20, new), (0, 0)):
        dev = _to(cache)
        short = paged_kvcache_reserve(dev, *(x.to(DEV) if isinstance(x, torch.Tensor) else x for x in (a, m)))
        want, left = oracle.reserve(cache, a.clamp(-2**31, 2**31 - 1) if isinstance(a, torch.Tensor) else a, m)
        _same(dev, want)
        assert torch.equal(short.cpu(), left)


def test_reserve_many_sequences_and_pages():
    """More sequences than the kernel has threads, more items than one round of them, more pages than one
    look at the counts; the lowest pages in order."""
    ps, N, M, P = 16, 2500, 9, 70000
    g = _gen(4)
    lens = _int(g, 0, 60, N)
    cache = oracle.dealt(1, P, 1, ps, 64, N, M, lens.tolist(), g)
    cache = oracle.fork(cache, torch.where(torch.rand(N, generator=g) < 0.2, _int(g, 0, N, N), -1))
    cache[2][(torch.rand(P, generator=g) < 0.9) & (cache[2] == 0)] = 1
    new = torch.where(torch.rand(N, generator=g) < 0.5, 1, _int(g, 0, 85, N)).int()
    dev = _to(cache)
    short = paged_kvcache_reserve(dev, lens.to(DEV), new.to(DEV))
    want, left = oracle.reserve(cache, lens, new)
    _same(dev, want)
    assert torch.equal(short.cpu(), left)


@pytest.mark.parametrize("N,M", [(1, 1), (5, 3), (64, 40), (300, 17), (1500, 5), (2049, 3), (5000, 9), (8192, 2)])
def test_fork(N, M):
    g = _gen(N)
    P = 3 * N + 7
    cache = oracle.dealt(1, P, 1, 16, 64, N, M, [0] * N, g)
    cache[3][:] = torch.randint(-3, P + 3, (N, M), generator=g)
    cache[2][:] = torch.bincount(cache[3][(cache[3] >= 0) & (cache[3] < P)].long(), minlength=P)
    for parents in (_int(g, -2, N + 2, N), torch.zeros(N, dtype=torch.int32), torch.arange(N, dtype=torch.int32),
                    torch.arange(N, dtype=torch.int32).flip(0), torch.full((N,), 2**31 - 1, dtype=torch.int32)):
        dev = _to(cache)
        assert paged_kvcache_fork(dev, parents.to(DEV)) is None
        _same(dev, oracle.fork(cache, parents))
        dev = _to(cache)
        paged_kvcache_fork(dev, parents.to(DEV).long() + (2**33 if int(parents[0]) == 2**31 - 1 else 0))
        _same(dev, oracle.fork(cache, parents))


@pytest.mark.parametrize("N,M,ps", [(1, 1, 16), (5, 3, 32), (64, 40, 1024), (300, 17, 64)])
def test_free(N, M, ps):
    g = _gen(N)
    P = 2 * N + 7
    cache = oracle.dealt(1, P, 1, ps, 64, N, M, [0] * N, g)
    cache[3][:] = torch.randint(-3, P + 3, (N, M), generator=g)
    cache[2][:] = torch.bincount(cache[3][(cache[3] >= 0) & (cache[3] < P)].long(), minlength=P)
    keep = _int(g, -5, M * ps + 5, N)
    keep[::2] = keep[::2] // ps * ps
    for x in (keep, 0, ps, ps + 1, -9, 2**31 - 1, 2**40, keep.long() * 2**40):
        dev = _to(cache)
        assert paged_kvcache_free(dev, x.to(DEV) if isinstance(x, torch.Tensor) else x) is None
        _same(dev, oracle.free(cache, x))
    dev = _to(cache)
    paged_kvcache_free(dev)
    assert (dev.page_table == -1).all() and not dev.refs.any()


@pytest.mark.parametrize("L,H,ps,D", SHAPES)
@pytest.mark.parametrize("share", [0.0, 0.1, 0.5, 0.97, 1.0])
def test_compact(share, L, H, ps, D):
    """None in use, few, nearly all, all; shared pages move once, entries that are no page stay."""
    for P in (1, 2, 50, 301):
        g = _gen(P)
        N, M = 9, 7
        cache = oracle.dealt(L, P, H, ps, D, N, M, [0] * N, g)
        table = torch.randint(0, P, (N, M), generator=g)
        table[torch.rand(N, M, generator=g) >= share] = -1
        table[3, 3] = P + 5
        if share == 1.0:
            cache[2][:] = 1
        cache[3][:] = table
        cache[2] += torch.bincount(table[(table >= 0) & (table < P)], minlength=P).int()
        dev = _to(cache)
        used = paged_kvcache_compact(dev)
        want, n = oracle.compact(cache)
        _same(dev, want, P)
        assert used.tolist() == [n]
        again = paged_kvcache_compact(dev)      # nothing left to move
        _same(dev, want, P)
        assert again.tolist() == [n]


def test_compact_many_pages():
    g = _gen(0)
    P, N, M = 40000, 100, 30
    cache = oracle.dealt(1, P, 1, 16, 64, N, M, [0] * N, g)
    cache[3][:] = torch.randint(0, P, (N, M), generator=g)
    cache[2][:] = torch.bincount(cache[3].view(-1).long(), minlength=P)
    dev = _to(cache)
    used = paged_kvcache_compact(dev)
    want, n = oracle.compact(cache)
    _same(dev, want)
    assert used.tolist() == [n]


@pytest.mark.parametrize("L,H,ps,D", SHAPES)
def test_copy(L, H, ps, D):
    g = _gen(ps)
    P, Q = 23, 40
    a, b = oracle.dealt(L, P, H, ps, D, 1, 1, [0], g), oracle.dealt(L, Q, H, ps, D, 2, 3, [0, 0], g)
    for n in (0, 1, 5, 23):
        src, dst = torch.randint(0, P, (n,), generator=g), torch.randperm(Q, generator=g)[:n]
        if n > 4:
            src[1], dst[2], src[3] = P, -1, -2**31
        for kind in (torch.int32, torch.int64):
            dev = _to(b)
            assert paged_kvcache_copy(dev, src.to(DEV, kind), dst.to(DEV, kind), source=_to(a)) is None
            _same(dev, oracle.copy(b, src, dst, a), n)
    src, dst = torch.randperm(Q, generator=g)[:20].int().chunk(2)
    dev = _to(b)
    paged_kvcache_copy(dev, src.to(DEV), dst.to(DEV))
    _same(dev, oracle.copy(b, src, dst))


def test_offsets_past_32_bits():
    """Pages on both sides of 2^31 elements, moved, copied and left behind."""
    H, ps, D = 4, 1024, 128
    P = (5 << 29) // (H * ps * D)
    c = paged_kvcache(P, ps, 2, 3 * ps, H)
    g = _gen(3)
    rows = torch.randn(H, ps, D, generator=g).bfloat16().to(DEV)
    c.k_pages[0, P - 2], c.v_pages[0, P - 2] = rows, -rows
    c.page_table[0, 0], c.refs[P - 2] = P - 2, 1
    paged_kvcache_copy(c, torch.tensor([P - 2], dtype=torch.int32, device=DEV), torch.tensor([P - 1], dtype=torch.int32, device=DEV))
    assert torch.equal(c.k_pages[0, P - 1], rows) and torch.equal(c.v_pages[0, P - 1], -rows)
    c.refs[:P - 3] = 1      # others hold all but the last ones
    paged_kvcache_fork(c, torch.tensor([0, 0], dtype=torch.int32, device=DEV))
    assert not paged_kvcache_reserve(c, 1000, 1).any() and c.page_table[:, 0].tolist() == [P - 2, P - 3]
    assert torch.equal(c.v_pages[0, P - 3, :, :1000], -rows[:, :1000]) and not c.v_pages[0, P - 3, :, 1000:].any()
    c.refs[:P - 3] = 0
    assert paged_kvcache_compact(c).tolist() == [2] and c.page_table[:, 0].tolist() == [1, 0]
    assert torch.equal(c.k_pages[0, 1], rows) and torch.equal(c.k_pages[0, 0, :, :1000], rows[:, :1000])


def test_refusals():
    g = _gen(1)
    c = _to(oracle.dealt(2, 10, 2, 16, 128, 2, 4, [64, 64], g))
    two = torch.zeros(2, dtype=torch.int32, device=DEV)
    many = torch.full((8193, 1), -1, dtype=torch.int32, device=DEV)
    bad = [(c._replace(refs=c.refs[:9]), "refs"), (c._replace(page_table=c.page_table.long()), "page_table"),
           (c._replace(page_table=c.page_table[:1].expand(2, 4)), "page_table"),
           (c._replace(page_table=c.refs[:8].view(2, 4)), "overlap")]
    pooled = [(c._replace(k_pages=c.k_pages.float()), "k_pages"), (c._replace(v_pages=c.k_pages), "overlap"),
              (c._replace(v_pages=c.v_pages[:1]), "differ")]
    for call, caches in ((lambda x: paged_kvcache_reserve(x, 0, 1), bad + pooled + [(c._replace(page_table=many), "8193")]),
                         (lambda x: paged_kvcache_fork(x, two), bad[1:] + [(c._replace(refs=c.refs.long()), "refs")]),
                         (lambda x: paged_kvcache_free(x, two), bad[1:] + [(c._replace(refs=c.refs[::2]), "refs")]),
                         (lambda x: paged_kvcache_compact(x), bad + pooled),
                         (lambda x: paged_kvcache_copy(x, two, two), pooled)):
        for x, needle in caches:
            with pytest.raises(ValueError, match=needle):
                call(x)
    three, cpu = torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32)
    for x in (three, cpu, two.float()):
        for call in (lambda: paged_kvcache_reserve(c, x, 1), lambda: paged_kvcache_reserve(c, 0, x), lambda: paged_kvcache_fork(c, x),
                     lambda: paged_kvcache_free(c, x), lambda: paged_kvcache_copy(c, x, two)):
            with pytest.raises(ValueError):
                call()
    with pytest.raises(ValueError, match="8193"):
        paged_kvcache_fork(c._replace(page_table=many), torch.zeros(8193, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="parents"):
        paged_kvcache_fork(c, 0)
    for other in (paged_kvcache(10, 16, 1, 16, 2), paged_kvcache(10, 32, 1, 16, 2, layers=2), paged_kvcache(10, 16, 1, 16, 1, layers=2),
                  paged_kvcache(10, 16, 1, 16, 2, 64, layers=2)):
        with pytest.raises(ValueError, match="differ"):
            paged_kvcache_copy(c, two, two, source=other)
    with pytest.raises(ValueError, match="overlap"):
        paged_kvcache_copy(c, two, two, source=c)
    with pytest.raises(ValueError, match="lists"):
        paged_kvcache_copy(c, two[None], two[None])
