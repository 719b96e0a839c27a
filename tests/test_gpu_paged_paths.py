"""GPU: sizes that choose each way through the attention over pages, many sequences and very unequal ones, calls that are
captured and replayed, and a run of the page operators and the attention together, as an engine uses them.

Tolerances: those of tests/test_gpu_paged.py.
"""
import math

import pytest
import torch

from oracle import paged_oracle as oracle
from prefixlm import (PagedKVCache, _capi, flash_attn_with_paged_kvcache, paged_kvcache, paged_kvcache_compact, paged_kvcache_copy,
                      paged_kvcache_fork, paged_kvcache_free, paged_kvcache_reserve)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24


def _rows(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).bfloat16()


def _to(cache):
    return PagedKVCache(*(x.to(DEV) for x in cache))


def _tol(q, top, rows, mag, want):
    """top: the largest magnitude of a key; rows: the most that a query sees."""
    A = q.double().abs().sum(-1, keepdim=True) * top / math.sqrt(q.shape[-1])
    return 2.0 ** -8 * want.abs() + (2 * 140 * U * A + (rows + 100 + 256) * U) * mag + 1e-30


def _check(q, cache, k, v, lens, causal, only=None):
    dev = _to(cache)
    out = flash_attn_with_paged_kvcache(q.to(DEV), dev, k.to(DEV) if k is not None else None, v.to(DEV) if v is not None else None,
                                        lens.to(DEV), causal=causal)
    at = list(range(q.shape[0])) if only is None else only
    sub = [*cache[:3], cache[3][at]]
    args = [x[at] if x is not None else None for x in (k, v)]
    want, mag, new = oracle.attend(q[at], sub, *args, lens[at], causal)
    top = max(float(cache[0].abs().max().float()), float(k.abs().max().float()) if k is not None else 0.0)
    over = (out[at].double().cpu() - want).abs() - _tol(q[at], top, cache[3].shape[1] * cache[0].shape[3], mag, want)
    assert over.max().item() <= 0, over.max().item()
    # the pages of the others are compared where all are checked
    if only is None:
        for a, b in zip(dev[:2], new[:2]):
            assert torch.equal(a.cpu(), b)
    return out


def _shares(B, S, Hq, Hkv, D, ps, M):
    return _capi.load().prefixlm_paged_workspace_size(B, S, Hq, Hkv, D, ps, M) > 0


# rows that share keys, key-value heads, sequences, capacity, whether the units are cut into pieces
SIZES = [(1, 1, 2, 2, 784, False), (1, 1, 2, 2, 800, True), (1, 1, 16, 8, 512, False), (1, 1, 20, 13, 4096, True),
         (1, 1, 96, 4, 640, False), (1, 1, 100, 4, 640, False), (2, 1, 2, 2, 256, False), (2, 1, 2, 2, 272, True),
         (1, 16, 16, 8, 512, False), (1, 7, 32, 8, 640, True), (3, 5, 65, 4, 640, False), (5, 4, 3, 2, 256, False),
         (17, 1, 2, 2, 640, True), (32, 2, 33, 8, 384, False), (64, 1, 2, 1, 1280, True), (65, 1, 2, 2, 256, False),
         (65, 1, 2, 2, 640, True), (130, 1, 16, 16, 512, False), (200, 1, 65, 4, 512, False), (129, 2, 1, 1, 2048, True)]


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("S,G,B,H,cap,shared", SIZES)
def test_by_their_sizes(S, G, B, H, cap, shared, D):
    print(f"[case] {S} {G} {B} {H} {cap} {D}", flush=True)
    ps = 16
    assert _shares(B, S, G * H, H, D, ps, cap // ps) == shared
    g = torch.Generator().manual_seed(B + S)
    lens = torch.randint(0, cap - S + 1, (B,), generator=g, dtype=torch.int32)
    lens[0], lens[-1] = cap - S, 0
    cache = oracle.dealt(1, sum(-(-(int(n) + S) // ps) for n in lens) + 9, H, ps, D, B, cap // ps, (lens + S).tolist(), g)
    q, k, v = _rows(g, B, S, H * G, D), _rows(g, B, S, H, D), _rows(g, B, S, H, D)
    few = sorted({0, B // 3, B // 2, B - 1})
    _check(q, cache, k, v, lens, True, only=None if B * S * G * H < 200 else few)
    _check(q, cache, None, None, lens, False, only=few)


@pytest.mark.parametrize("S,G", [(1, 1), (1, 4), (20, 1), (70, 1)])
@pytest.mark.parametrize("B", [63, 64, 65, 128, 129, 200, 256, 257])
def test_many_sequences(B, S, G):
    """Lengths past the first 64 sequences, whose tiles lie in further registers; empty ones among them."""
    print(f"[case] {B} {S} {G}", flush=True)
    H, D, ps, cap = 1, 64, 64, 2112
    g = torch.Generator().manual_seed(B + S)
    lens = (torch.rand(B, generator=g) ** 4 * (cap - S)).int()
    lens[::7], lens[B // 2], lens[-1] = 0, cap - S, cap - S - 1
    cache = oracle.dealt(1, sum(-(-(int(n) + S) // ps) for n in lens) + 1, H, ps, D, B, cap // ps, (lens + S).tolist(), g)
    q, k, v = _rows(g, B, S, H * G, D), _rows(g, B, S, H, D), _rows(g, B, S, H, D)
    out = _check(q, cache, k, v, lens, True, only=sorted({0, 1, 61, 62, B // 2, B - 2, B - 1}))
    dev = _to(cache)
    again = flash_attn_with_paged_kvcache(q.to(DEV), dev, k.to(DEV), v.to(DEV), lens.to(DEV), causal=True)
    assert torch.equal(out, again)


@pytest.mark.parametrize("S,G", [(1, 1), (1, 3), (2, 8), (33, 1), (150, 1)])
def test_one_long_sequence_among_short_ones(S, G):
    B, H, D, ps, cap = 8, 2, 128, 32, 8192
    assert _shares(B, S, G * H, H, D, ps, cap // ps)
    lens = torch.tensor([0, 1, 63, 64, 65, 5, 5, cap - S], dtype=torch.int32)
    g = torch.Generator().manual_seed(S)
    cache = oracle.dealt(1, sum(-(-(int(n) + S) // ps) for n in lens) + 1, H, ps, D, B, cap // ps, (lens + S).tolist(), g)
    q, k, v = _rows(g, B, S, H * G, D), _rows(g, B, S, H, D), _rows(g, B, S, H, D)
    _check(q, cache, k, v, lens, True)
    for n in (torch.zeros_like(lens), torch.full_like(lens, 64), torch.full_like(lens, 1)):
        _check(q, [*cache[:3], cache[3]], None, None, torch.minimum(n, lens), False)


class Engine:
    """A cache and its lengths on the device beside the oracle's on the host, step by step."""

    def __init__(self, L, P, ps, N, cap, H, G, D, seed):
        self.cache = paged_kvcache(P, ps, N, cap, H, D, layers=L)
        self.want = [x.cpu() for x in self.cache]
        self.lens = torch.zeros(N, dtype=torch.int32, device=DEV)
        self.g = torch.Generator().manual_seed(seed)
        self.shape = (L, H, G, D)

    def same(self, tag=""):
        for name, a, b in zip(PagedKVCache._fields, self.cache, self.want):
            assert torch.equal(a.cpu(), b), (tag, name)

    def step(self, S, new, tag=""):
        """S queries and rows for every slot, of which `new` count."""
        L, H, G, D = self.shape
        N = self.lens.numel()
        short = paged_kvcache_reserve(self.cache, self.lens, new.to(DEV))
        lens = self.lens.cpu()
        self.want, left = oracle.reserve(self.want, lens, new)
        assert torch.equal(short.cpu(), left) and not left.any(), tag
        for layer in range(L):
            q, k, v = _rows(self.g, N, S, H * G, D), _rows(self.g, N, S, H, D), _rows(self.g, N, S, H, D)
            out = flash_attn_with_paged_kvcache(q.to(DEV), self.cache, k.to(DEV), v.to(DEV), self.lens, causal=True, layer=layer)
            ref, mag, self.want = oracle.attend(q, self.want, k, v, lens, True, layer=layer)
            top = max(float(x.abs().max().float()) for x in (self.want[0], k))
            tol = _tol(q, top, self.want[3].shape[1] * self.want[0].shape[3], mag, ref)
            assert ((out.double().cpu() - ref).abs() <= tol).all(), (tag, layer)
        self.lens += new.to(DEV)
        self.same(tag)


def test_prompts_samples_tokens_and_what_follows():
    """Prompts come in, one is sampled three times, tokens and drafts with a part taken back, beams that go on
    from others, a sequence that ends, pages that move, a smaller pool, and on."""
    N, L, ps = 6, 2, 16
    e = Engine(L, 64, ps, N, 160, 2, 2, 64, 5)
    e.step(37, torch.tensor([37, 20, 0, 0, 0, 0], dtype=torch.int32), "prompts")     # slots past the prompts' ends hold no rows
    e.lens.copy_(torch.tensor([37, 20, 0, 0, 0, 0]))
    parents = torch.tensor([0, 1, 0, 0, -1, 9], dtype=torch.int32)
    paged_kvcache_fork(e.cache, parents.to(DEV))
    e.want = oracle.fork(e.want, parents)
    e.lens.copy_(torch.tensor([37, 20, 37, 37, 0, 0]))
    e.same("fork")
    assert int((e.want[2] == 3).sum()) == 3 and int(e.want[2].max()) == 3          # three pages shared by three
    on = torch.tensor([1, 1, 1, 1, 0, 0], dtype=torch.int32)
    for i in range(14):
        e.step(1, on, ("token", i))
    e.step(5, 5 * on, "draft")
    e.lens -= torch.tensor([3, 0, 5, 1, 0, 0], dtype=torch.int32, device=DEV)        # rejected
    paged_kvcache_free(e.cache, e.lens)
    e.want = oracle.free(e.want, e.lens.cpu())
    e.same("taken back")
    parents = torch.tensor([2, 1, 2, 0, 4, 5], dtype=torch.int32)
    paged_kvcache_fork(e.cache, parents.to(DEV))
    e.want = oracle.fork(e.want, parents)
    e.lens.copy_(e.lens[parents.long().to(DEV)])
    for i in range(4):
        e.step(1, on, ("beam", i))
    keep = torch.tensor([2**31 - 1, 0, 2**31 - 1, 2**31 - 1, 0, 0], dtype=torch.int32)
    paged_kvcache_free(e.cache, keep.to(DEV))
    e.want = oracle.free(e.want, keep)
    e.lens[1] = 0
    used = paged_kvcache_compact(e.cache)
    e.want, n = oracle.compact(e.want)
    e.same("compact")
    assert used.tolist() == [n]
    small = paged_kvcache(n + 12, ps, N, 160, 2, 64, layers=L)
    pages = torch.arange(n, dtype=torch.int32, device=DEV)
    paged_kvcache_copy(small, pages, pages, source=e.cache)
    small.page_table.copy_(e.cache.page_table)
    small.refs[:n] = e.cache.refs[:n]
    e.cache, e.want = small, [x.cpu() for x in small]
    for i in range(3):
        e.step(1, torch.tensor([1, 0, 1, 1, 0, 0], dtype=torch.int32), ("after", i))
    e.step(20, torch.tensor([20, 11, 20, 20, 0, 0], dtype=torch.int32), "next turns")


@pytest.mark.parametrize("S,G,cap", [(1, 1, 256), (1, 4, 1024), (4, 2, 512), (33, 1, 512), (70, 2, 1024)])
def test_a_captured_step(S, G, cap):
    """Reserve, attention in two layers, fork and free in one graph: replayed with lengths that move on the device, with
    eager work between, against eager calls on another cache."""
    print(f"[case] {S} {G} {cap}", flush=True)
    N, L, H, D, ps = 3, 2, 2, 64, 16
    P = 5 * cap // ps
    g = torch.Generator().manual_seed(S)
    a, b = (paged_kvcache(P, ps, N, cap, H, D, layers=L) for _ in range(2))
    lens = torch.tensor([9, 0, 16], dtype=torch.int32, device=DEV)
    new = torch.full((N,), S, dtype=torch.int32, device=DEV)
    parents = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    keep = torch.full((N,), 2**31 - 1, dtype=torch.int32, device=DEV)
    q, k, v = _rows(g, N, S, H * G, D).to(DEV), _rows(g, N, S, H, D).to(DEV), _rows(g, N, S, H, D).to(DEV)

    def step(cache, lens):
        paged_kvcache_free(cache, keep)
        paged_kvcache_fork(cache, parents)
        short = paged_kvcache_reserve(cache, lens, new)
        return short, *(flash_attn_with_paged_kvcache(q, cache, k, v, lens, causal=True, layer=i) for i in range(L)), \
            paged_kvcache_compact(cache)

    def clear(c):
        for x, y in zip(c, paged_kvcache(P, ps, N, cap, H, D, layers=L)):
            x.copy_(y)
        paged_kvcache_reserve(c, 0, lens)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(a, lens)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a, lens)
    clear(a), clear(b)
    for i in range(7):
        for x in (q, k, v):
            x.copy_(_rows(g, *x.shape))
        parents.copy_(torch.tensor([[0, 1, 2], [0, 0, 2], [1, 0, -1]][i % 3]))
        keep.copy_(torch.tensor([[2**31 - 1] * 3, [2**31 - 1, 5, 2**31 - 1]][i % 2]))
        if i % 2:
            lens[1] = 5
        lens.copy_(lens[torch.where(parents >= 0, parents, torch.arange(3, device=DEV)).long()])
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, step(b, lens.clone())):
            assert torch.equal(x, y), i
        for name, x, y in zip(PagedKVCache._fields, a, b):
            assert torch.equal(x, y), (i, name)
        lens.add_(S)


def test_two_streams_at_once():
    """The same operators on two streams, whose workspaces must be their own."""
    N, H, D, ps, cap = 4, 4, 128, 32, 4096
    g = torch.Generator().manual_seed(1)
    first = []
    for i in range(2):
        lens = torch.randint(100, cap - 100, (N,), generator=g, dtype=torch.int32)
        c = oracle.dealt(1, N * cap // ps, H, ps, D, N, cap // ps, lens.tolist(), g)
        first.append((c, lens.to(DEV), *(_rows(g, N, S, H * G, D).to(DEV) for S, G in ((1, 1), (1, 4), (20, 1)))))
    caches, kept = ([_to(f[0]) for f in first] for _ in range(2))
    parents = torch.tensor([1, 1, 0, 3], dtype=torch.int32, device=DEV)

    def work(i):
        c, lens = caches[i], first[i][1]
        # the pages too: sequence 2 gives its own up, and the copies of the reserve go there
        for x, y in zip(c, kept[i]):
            x.copy_(y)
        out = [flash_attn_with_paged_kvcache(q, c, cache_seqlens=lens, causal=True) for q in first[i][2:]]
        paged_kvcache_fork(c, parents)
        out.append(paged_kvcache_reserve(c, lens[parents.long()], 3))
        return out + [x.clone() for x in c[2:]]

    want = [work(i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(work(i))
        torch.cuda.synchronize()
        for x, y in zip(want, got):
            for u, w in zip(x, y):
                assert torch.equal(u, w)
