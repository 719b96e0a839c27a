"""GPU: attention over pages where rows have none, through each of its kernels: one row that shares the keys, up to 16, blocks
of 64 and of 128; pages that a tile of keys lies in and smaller ones; units whole and in pieces. Every sequence of a call
against 64 bits.

Tolerances (u = 2^-24): a score sums up to 128 products in fp32, off by at most 140 u of the sum of their magnitudes A,
the exponentials, their weighted sum and its normalisation by twice that of the sum of p |v|; n keys add n u more, the joins
100 u. out is rounded to bf16, 2^-8 relative. Pages are equal bit for bit.
"""
import math

import pytest
import torch

from oracle import paged_oracle as oracle
from prefixlm import PagedKVCache, _capi, flash_attn_with_paged_kvcache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24


def _rows(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).bfloat16()


def _to(cache):
    return PagedKVCache(*(x.to(DEV) for x in cache))


def _far(out, q, cache, k, v, lens, causal, heads=None):
    """The largest excess over the tolerance, of the key-value heads named."""
    H = cache[0].shape[2]
    G, D, n = q.shape[2] // H, q.shape[3], cache[3].shape[1] * cache[0].shape[3]
    worst = -math.inf
    for h in range(H) if heads is None else heads:
        mine = slice(h * G, h * G + G)
        sub = [x[:, :, h:h + 1].contiguous() for x in cache[:2]] + cache[2:]
        new = [x[:, :, h:h + 1] if x is not None else None for x in (k, v)]
        want, mag, _ = oracle.attend(q[:, :, mine], sub, *new, lens, causal)
        top = max(float(x.abs().max().float()) for x in (sub[0], new[0]) if x is not None)
        A = q[:, :, mine].double().abs().sum(-1, keepdim=True) * top / math.sqrt(D)
        tol = 2.0 ** -8 * want.abs() + (2 * 140 * U * A + (n + 100) * U) * mag + 1e-30
        worst = max(worst, ((out[:, :, mine].double().cpu() - want).abs() - tol).max().item())
    return worst


def _stored(cache, k, v, lens):
    """The pages with the rows that are stored."""
    kp, vp, refs, table = (x.clone() for x in cache)
    P, ps = kp.shape[1], kp.shape[3]
    for b, n in enumerate(lens.tolist()):
        for j in range(n, min(table.shape[1] * ps, n + k.shape[1])):
            p = int(table[b, j // ps])
            if 0 <= p < P and refs[p] == 1:
                kp[0, p, :, j % ps], vp[0, p, :, j % ps] = k[b, j - n], v[b, j - n]
    return kp, vp


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("ps", [16, 32, 64, 256])
@pytest.mark.parametrize("S,G,H", [(1, 1, 2), (1, 1, 37), (1, 3, 2), (2, 8, 2), (4, 4, 37), (20, 1, 2), (20, 1, 37), (10, 6, 2), (80, 1, 2),
                                   (80, 1, 20), (80, 1, 40), (33, 4, 1)])
def test_rows_without_a_page(S, G, H, ps, D):
    """Columns without a page at a sequence's start, in its middle and at its end, everywhere, and where the new rows go;
    entries that are no page; a page that others hold too. Pages that no sequence holds, and rows behind
    the last, hold values that would be seen in any sum."""
    print(f"[case] {S} {G} {H} {ps} {D}", flush=True)
    cap = 1024
    M, B = cap // ps, 7
    assert (_capi.load().prefixlm_paged_workspace_size(B, S, G * H, H, D, ps, M) > 0) == (H <= 2)
    lens = torch.tensor([0, 700, 530, 900, 600, 97, cap - S + 1], dtype=torch.int32)
    g = torch.Generator().manual_seed(S + ps)
    cache = oracle.dealt(1, B * M + 9, H, ps, D, B, M, (lens + S).tolist(), g)
    kp, vp, refs, table = cache
    P = refs.numel()
    bad = (-1, P, 2**31 - 1, -2**31)

    def drop(b, columns):
        for i, c in enumerate(columns):
            if 0 <= int(table[b, c]) < P:
                refs[table[b, c]] = 0
            table[b, c] = bad[i % 4]

    quarter = max(1, M // 4)
    drop(1, range(M))
    drop(2, range(quarter))
    drop(3, range(quarter, 2 * quarter))
    drop(4, range(max(0, 600 // ps - quarter // 2), 600 // ps + 1))     # and the first new rows' column
    drop(6, range(M - 1, M))
    refs[table[5, 97 // ps].long()] = 2
    full = torch.zeros(P, ps, dtype=torch.bool)
    for b, n in enumerate(lens.tolist()):
        for c in range(-(-n // ps)):
            if 0 <= int(table[b, c]) < P:
                full[table[b, c], :min(ps, n - c * ps)] = True
    kp.masked_fill_(~full[None, :, None, :, None], 0.0)
    vp.masked_fill_(~full[None, :, None, :, None], 1e4)
    q, k, v = _rows(g, B, S, H * G, D, scale=0.25), _rows(g, B, S, H, D), _rows(g, B, S, H, D)
    heads = sorted({0, H - 1})
    for causal in (False, True):
        dev = _to(cache)
        out = flash_attn_with_paged_kvcache(q.to(DEV), dev, k.to(DEV), v.to(DEV), lens.to(DEV), causal=causal)
        assert _far(out, q, cache, k, v, lens, causal, heads) <= 0, causal
        for a, b in zip(dev[:2], _stored(cache, k, v, lens)):
            assert torch.equal(a.cpu(), b)
        for a, b in zip(dev[2:], cache[2:]):
            assert torch.equal(a.cpu(), b)
        dev = _to(cache)
        out = flash_attn_with_paged_kvcache(q.to(DEV), dev, cache_seqlens=lens.to(DEV), causal=causal)
        assert _far(out, q, cache, None, None, lens, causal, heads) <= 0, causal
        assert not out[0].any() and not out[1].any()
        for a, b in zip(dev, cache):
            assert torch.equal(a.cpu(), b)
