"""GPU: attention over pages, batches of unequal sequences with every sequence against 64 bits, and the page calls with the
attention on two streams at once, the pages' contents compared.

Tolerances (u = 2^-24): a score sums up to 128 products in fp32, off by at most 140 u of the sum of their magnitudes, at
most A for a query's keys; the exponentials, their weighted sum and its normalisation are off by twice that of the sum of p |v|; n
keys add n u more, the joins 100 u. out is rounded to bf16, 2^-8 relative.
"""
import math

import pytest
import torch

from oracle import paged_oracle as oracle
from prefixlm import PagedKVCache, flash_attn_with_paged_kvcache, paged_kvcache_compact, paged_kvcache_fork, paged_kvcache_reserve

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24


def _rows(g, *shape):
    return torch.randn(*shape, generator=g).bfloat16()


def _to(cache):
    return PagedKVCache(*(x.to(DEV) for x in cache))


def _far(out, q, cache, k, v, n):
    """One sequence of n cached rows, causal, on the GPU in float64: the largest excess over the tolerance."""
    kp, vp, _, table = cache
    (H, ps, D), S = kp.shape[2:], q.shape[0]
    G = q.shape[1] // H
    pages = table[:-(-n // ps)].long()
    keys, values = (torch.cat((x[0, pages].transpose(0, 1).reshape(H, -1, D)[:, :n], y.transpose(0, 1)), 1).double()
                    for x, y in ((kp, k), (vp, v)))
    rows = q.double().view(S, H, G, D).permute(1, 0, 2, 3).reshape(H, S * G, D)
    hide = torch.ones(S, n + S, dtype=torch.bool, device=DEV).triu(n + 1).repeat_interleave(G, 0)
    worst = -math.inf
    for h in range(H):
        s = 1.0 / math.sqrt(D)
        A = (rows[h].abs() @ keys[h].abs().t().contiguous()).amax(-1, keepdim=True) * s
        p = torch.softmax((rows[h] @ keys[h].t().contiguous() * s).masked_fill(hide, -math.inf), -1)
        want, mag = p @ values[h], p @ values[h].abs()
        got = out.double().view(S, H, G, D)[:, h].reshape(S * G, D)
        tol = 2.0 ** -8 * want.abs() + (2 * 140 * U * A + (n + S + 100) * U) * mag + 1e-30
        worst = max(worst, ((got - want).abs() - tol).max().item())
    return worst


@pytest.mark.parametrize("D,ps", [(128, 64), (64, 16), (64, 128), (128, 32)])
@pytest.mark.parametrize("B,H,S,G,most", [(3, 9, 333, 4, 150), (16, 16, 40, 1, 600), (64, 8, 20, 1, 700), (65, 8, 20, 2, 400), (17, 4, 520, 1, 90),
                                          (70, 8, 1, 1, 3000), (40, 8, 1, 4, 2000), (33, 2, 3, 5, 2000)])
def test_every_sequence(B, H, S, G, most, D, ps):
    print(f"[case] {B} {H} {S} {G} {most} {D} {ps}", flush=True)
    g = torch.Generator().manual_seed(B + S)
    M = -(-(most + S) // ps)
    lens = (torch.rand(B, generator=g) ** 3 * most).int()
    lens[::5] = lens[0]
    lens[B // 2], lens[-1], lens[1] = 0, 1, most
    cache = _to(oracle.dealt(1, B * M, H, ps, D, B, M, (lens + S).tolist(), g))
    q, k, v = (_rows(g, B, S, n, D).to(DEV) for n in (H * G, H, H))
    out = flash_attn_with_paged_kvcache(q, cache, k, v, lens.to(DEV), causal=True)
    for b in range(B):
        one = (*cache[:3], cache.page_table[b])
        assert _far(out[b], q[b], one, k[b], v[b], int(lens[b])) <= 0, b


def test_two_streams_hold_their_own_pages():
    """Beams that share pages get their own, take rows and are compacted on two streams; every tensor of both caches, and the
    attention before and after, as one stream alone gives them."""
    N, H, D, ps, cap, L = 6, 4, 128, 32, 2048, 2
    g = torch.Generator().manual_seed(3)
    first = []
    for i in range(2):
        lens = torch.randint(100, cap - 100, (N,), generator=g, dtype=torch.int32)
        c = _to(oracle.dealt(L, N * cap // ps + 20, H, ps, D, N, cap // ps, lens.tolist(), g))
        first.append((c, lens.to(DEV), [_rows(g, N, 3, H, D).to(DEV) for _ in range(3)]))
    parents = torch.tensor([1, 1, 0, 3, 3, 3], dtype=torch.int32, device=DEV)

    def work(i):
        c, lens, (q, k, v) = PagedKVCache(*(x.clone() for x in first[i][0])), first[i][1], first[i][2]
        out = [flash_attn_with_paged_kvcache(q, c, cache_seqlens=lens, causal=True)]
        paged_kvcache_fork(c, parents)
        lens = lens[parents.long()]
        out.append(paged_kvcache_reserve(c, lens, 3))
        out += [flash_attn_with_paged_kvcache(q, c, k, v, lens, causal=True, layer=i) for i in range(L)]
        out.append(paged_kvcache_compact(c))
        out.append(flash_attn_with_paged_kvcache(q, c, cache_seqlens=lens + 3, causal=True))
        return [*out, *c]

    want = [work(i) for i in range(2)]
    assert int(want[0][1].sum()) == 0
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(work(i))
        torch.cuda.synchronize()
        for x, y in zip(want, got):
            for n, (u, w) in enumerate(zip(x, y)):
                assert torch.equal(u, w), n
