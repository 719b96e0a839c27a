"""GPU: attention over a key-value cache in pages against the fp64 oracle; the pages it leaves bitwise.

Tolerances (u = 2^-24). A score sums up to 128 products in fp32, off by at most 140 u of the sum of their
magnitudes A, and exponentials of scores off by d change each weight by d relative, a sum of weighted
rows by 2 d of the sum of p |v|; n keys add n u more, and the splits' joins 100 u. The probabilities enter
P V as three bf16 terms, their 24 bits, or in blocks of 64 and 128 rows as two, each rounded to nearest: what the first leaves
is at most 2^-8 of p, what the second leaves of that 2^-8 again, 2^-16 p = 256 u of the sum of p |v|. out is rounded to
bf16, 2^-8 relative. Pages are equal bit for bit.
"""
import math

import pytest
import torch

from oracle import paged_oracle as oracle
from prefixlm import PagedKVCache, flash_attn_with_kvcache, flash_attn_with_paged_kvcache, paged_kvcache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24


def _rows(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).bfloat16()


def _to(cache):
    return PagedKVCache(*(x.to(DEV) for x in cache))


def _finite_max(x):
    x = x.float().abs()
    return x[torch.isfinite(x)].max()


def _tol(q, cache, k, mag, want, softmax_scale=None, top=None):
    """top: the largest magnitude of a key, of those whose weight is not 0."""
    D = q.shape[-1]
    finite = [x.float().abs() for x in ((cache[0], k) if k is not None else (cache[0],))]
    top = max(float(x[torch.isfinite(x)].max()) for x in finite) if top is None else top
    s = 1.0 / math.sqrt(D) if softmax_scale is None else abs(softmax_scale)
    A = q.double().abs().sum(-1, keepdim=True) * top * s
    n = cache[3].shape[1] * cache[0].shape[3]
    return 2.0 ** -8 * want.abs() + (2 * 140 * U * A + (n + 100 + 256) * U) * mag + 1e-30


def _same(got, want, tag=""):
    for name, a, b in zip(PagedKVCache._fields, got, want):
        assert torch.equal(a.cpu().view(torch.int16 if a.element_size() == 2 else torch.int32),
                           b.view(torch.int16 if b.element_size() == 2 else torch.int32)), (tag, name)


def _check(q, cache, k, v, lens, causal, tag="", softmax_scale=None, layer=0, top=None):
    dev = _to(cache)
    out = flash_attn_with_paged_kvcache(q.to(DEV), dev, k.to(DEV) if k is not None else None, v.to(DEV) if v is not None else None,
                                        lens.to(DEV) if isinstance(lens, torch.Tensor) else lens, softmax_scale, causal, layer)
    want, mag, new = oracle.attend(q, cache, k, v, lens, causal, softmax_scale, layer)
    got = out.double().cpu()
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), tag
    ok = torch.isfinite(want)
    over = ((got - want).abs() - _tol(q, cache, k, mag, want, softmax_scale, top))[ok]
    assert over.max().item() <= 0, (tag, (got - want).abs()[ok].max().item())
    _same(dev, new, tag)
    return out


def _poison(cache, lens):
    """NaN in every row that no sequence has filled."""
    kp, vp, refs, table = cache
    ps = kp.shape[3]
    full = torch.zeros(kp.shape[1], ps, dtype=torch.bool)
    for n, rows in enumerate(lens.tolist()):
        for c in range(table.shape[1]):
            if table[n, c] >= 0:
                full[table[n, c], :min(ps, max(0, rows - c * ps))] = True
    for x in (kp, vp):
        x.masked_fill_(~full[None, :, None, :, None], math.nan)
    return cache


# rows that share a key-value head's keys: 1 to 16 (one tile), to 32, and several blocks
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D,ps", [(128, 16), (64, 32), (128, 64), (64, 256)])
@pytest.mark.parametrize("S,G", [(1, 1), (1, 4), (1, 8), (1, 16), (1, 3), (2, 1), (5, 4), (17, 1), (3, 8), (31, 1), (33, 1), (70, 2),
                                 (130, 1), (1, 40)])
def test_matches_oracle(S, G, D, ps, causal):
    H, M = 2, max(1, 512 // ps)
    cap = M * ps
    lens = torch.tensor([0, 1, 15, 16, 31, 32, 33, 63, 64, 100, 127, 129, 300, cap - S], dtype=torch.int32)
    B, g = lens.numel(), torch.Generator().manual_seed(S * 100 + G)
    cache = oracle.dealt(2, 2 * B * M, H, ps, D, B, M, (lens + S).tolist(), g)
    q, k, v = _rows(g, B, S, H * G, D), _rows(g, B, S, H, D), _rows(g, B, S, H, D)
    _check(q, _poison(cache, lens), k, v, lens, causal, (S, G, D, ps), layer=1)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("S,G,D,ps", [(1, 1, 128, 64), (1, 2, 64, 16), (6, 4, 128, 32), (40, 1, 128, 16), (80, 1, 64, 64), (150, 1, 128, 32)])
def test_the_cache_alone_and_past_its_end(S, G, D, ps, causal):
    H, M = 3, 192 // ps
    lens = torch.tensor([0, 1, 2, 64, 100, 191, 192, -5, 193, 2**31 - 1, -2**31], dtype=torch.int32)
    B, g = lens.numel(), torch.Generator().manual_seed(20 + S)
    cache = oracle.dealt(1, B * M + 3, H, ps, D, B, M, [M * ps] * B, g)
    q, k, v = _rows(g, B, S, H * G, D), _rows(g, B, S, H, D), _rows(g, B, S, H, D)
    out = _check(q, cache, None, None, lens, causal, "alone")
    assert not out[0].any()
    _check(q, cache, k, v, lens, causal, "past the end")
    wide = torch.tensor([2**40, -2**40, 5, 64, 100, 191, 192, 0, 2**31, 2**32, -2**31 - 1])
    a = _check(q, cache, k, v, wide, causal, "int64")
    assert torch.equal(a[5], _check(q, cache, k, v, 191, causal, "int")[5])


@pytest.mark.parametrize("S", [1, 4, 40, 130])
@pytest.mark.parametrize("causal", [False, True])
def test_sequences_without_pages(S, causal):
    """An idle slot, pages missing in the middle, entries that are no page, pages that others hold: nothing is
    read or written there."""
    H, G, ps, D, M, P = 2, 2, 16, 128, 20, 120
    lens = torch.tensor([0, 60, 200, 130, 97], dtype=torch.int32)
    B, g = lens.numel(), torch.Generator().manual_seed(S)
    cache = oracle.dealt(1, P, H, ps, D, B, M, (lens + S).tolist(), g)
    refs, table = cache[2:]
    table[1] = -1
    table[2, 3:6], table[2, 12] = -1, P
    table[3, 0], table[3, 2] = 2**31 - 1, -2**31
    refs[table[4, 97 // ps].long()] = 2          # the new row's page is not sequence 4's alone
    q, k, v = _rows(g, B, S, H * G, D), _rows(g, B, S, H, D), _rows(g, B, S, H, D)
    _check(q, cache, k, v, lens, causal)
    out = _check(q, cache, None, None, lens, causal)
    assert not out[1].any()


@pytest.mark.parametrize("S,G", [(1, 1), (1, 8), (3, 4), (20, 1), (70, 1), (150, 1)])
def test_infinities_nan_and_the_lowest_values(S, G):
    """Values that are not finite in rows that a query must not see; scores that pass fp32's range before the
    scale; keys of the type's lowest value."""
    H, ps, D, M = 2, 32, 128, 8
    lens = torch.tensor([100, 33, 64, 5, 90, 40], dtype=torch.int32)
    B, g = lens.numel(), torch.Generator().manual_seed(S + G)
    cache = oracle.dealt(1, 60, H, ps, D, B, M, [M * ps] * B, g)
    q, k, v = _rows(g, B, S, H * G, D), _rows(g, B, S, H, D), _rows(g, B, S, H, D)
    table = cache[3]
    top = float(cache[0].abs().max().float())
    # what the last new row holds, only the last query of a causal call sees
    v[0, -1], k[1, -1], v[2, -1] = math.inf, math.nan, math.nan
    cache[1][0, table[3, 0], :, 2] = -math.inf
    # the lowest value in some keys: the sums before the scale end at -inf or its neighbour
    low = torch.finfo(torch.bfloat16).min
    cache[0][0, table[4, 1], :, 3:9] = low
    q[4] = q[4].abs()
    cache[0][0, table[5, 0]] = low / 64
    q[5] = q[5].abs()
    for causal in (True, False):
        _check(q, cache, k, v, lens, causal, causal, top=max(top, float(_finite_max(k))))


def test_scores_of_minus_infinity():
    """A row that sees keys whose scores are all -inf is NaN, as softmax gives it; beside others they weigh 0."""
    H, ps, D, M = 1, 16, 64, 4
    g = torch.Generator().manual_seed(5)
    cache = oracle.dealt(1, 20, H, ps, D, 2, M, [64, 64], g)
    q = _rows(g, 2, 1, 1, D).abs() + 0.1
    q = q.bfloat16()
    cache[0][0, cache[3][0, 0], :, :] = -math.inf
    cache[0][0, cache[3][1, 0], :, 3:] = -math.inf
    lens = torch.tensor([16, 16], dtype=torch.int32)
    out = _check(q, cache, None, None, lens, False)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 1e-3])
@pytest.mark.parametrize("S", [1, 9, 70, 140])
def test_scales(S, scale):
    H, G, ps, D, M = 2, 2, 16, 64, 12
    lens = torch.tensor([100, 33, 0], dtype=torch.int32)
    g = torch.Generator().manual_seed(S)
    cache = oracle.dealt(1, 60, H, ps, D, 3, M, (lens + S).tolist(), g)
    q, k, v = _rows(g, 3, S, H * G, D), _rows(g, 3, S, H, D), _rows(g, 3, S, H, D)
    _check(q, cache, k, v, lens, True, softmax_scale=scale)


@pytest.mark.parametrize("S", [1, 7, 50, 130])
def test_strides_of_the_operands(S):
    """q, k, v as parts of one projection; sequences before tokens and behind; a table that is part of a wider
    one; rows that start at any 2 bytes are refused or copied as the other caches do."""
    B, H, G, ps, D, M = 3, 2, 2, 16, 128, 12
    lens = torch.tensor([100, 33, 0], dtype=torch.int32)
    g = torch.Generator().manual_seed(S)
    cache = oracle.dealt(1, 70, H, ps, D, B, M, (lens + S).tolist(), g)
    one = _rows(g, S, B, H * G + 2 * H, D).to(DEV).transpose(0, 1)
    q, k, v = one.split((H * G, H, H), 2)
    assert not q.is_contiguous()
    dev = _to(cache)
    wide = torch.full((B, M + 5), -1, dtype=torch.int32, device=DEV)
    wide[:, 2:2 + M] = dev.page_table
    dev = dev._replace(page_table=wide[:, 2:2 + M])
    got = flash_attn_with_paged_kvcache(q, dev, k, v, lens.to(DEV), causal=True)
    want, mag, new = oracle.attend(q.cpu(), cache, k.cpu(), v.cpu(), lens, True)
    assert ((got.double().cpu() - want).abs() <= _tol(q.cpu(), cache, k.cpu(), mag, want)).all()
    _same(dev._replace(page_table=dev.page_table.contiguous()), new)
    off = torch.empty(v.numel() + 4, dtype=torch.bfloat16, device=DEV)[4:].view(v.shape).copy_(v)
    again = flash_attn_with_paged_kvcache(q, dev, k, off, lens.to(DEV), causal=True)
    assert torch.equal(again, got)


def test_the_contiguous_cache_gives_the_same():
    """Page 0 .. M - 1 of each sequence one after another hold the contiguous cache's rows."""
    B, H, ps, D, M = 4, 8, 64, 128, 16
    g = torch.Generator().manual_seed(9)
    kc, vc = (_rows(g, B, M * ps, H, D).to(DEV) for _ in range(2))
    q, k, v = (_rows(g, B, 1, H, D).to(DEV) for _ in range(3))
    lens = torch.tensor([1000, 77, 512, 0], dtype=torch.int32, device=DEV)
    cache = paged_kvcache(B * M, ps, B, M * ps, H)
    cache.page_table.copy_(torch.arange(B * M, device=DEV).view(B, M))
    cache.refs.fill_(1)
    for pages, x in zip(cache[:2], (kc, vc)):
        pages[0].copy_(x.view(B * M, ps, H, D).transpose(1, 2))
    want = flash_attn_with_kvcache(q, kc, vc, k, v, lens)
    got = flash_attn_with_paged_kvcache(q, cache, k, v, lens)
    # both are within the rounding of out and a little of the fp64 result
    assert ((got.float() - want.float()).abs() <= 2 * 2.0 ** -8 * want.float().abs() + 1e-4).all()
    for pages, x in zip(cache[:2], (kc, vc)):
        assert torch.equal(pages[0].transpose(1, 2).reshape(B, M * ps, H, D), x)


def test_offsets_past_32_bits():
    """Pages of the second half of a pool of 5 x 2^30 elements, of its last layer."""
    H, ps, D, L = 4, 1024, 128, 2
    P = (5 << 29) // (H * ps * D)
    pages = [torch.empty(L, P, H, ps, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    g = torch.Generator().manual_seed(2)
    table = torch.tensor([[P - 1, P - 5]], dtype=torch.int32)
    small = [_rows(g, 1, 2, H, ps, D), _rows(g, 1, 2, H, ps, D)]
    for x, y in zip(pages, small):
        x[1, table[0].long()] = y[0].to(DEV)
    refs = torch.ones(P, dtype=torch.int32, device=DEV)
    for S in (1, 40, 130):
        q, k, v = (_rows(g, 1, S, H, D) for _ in range(3))
        n = 2 * ps - 200
        out = flash_attn_with_paged_kvcache(q.to(DEV), PagedKVCache(*pages, refs, table.to(DEV)), k.to(DEV), v.to(DEV), n, causal=True,
                                            layer=1)
        ref = [*small, torch.ones(2, dtype=torch.int32), torch.tensor([[0, 1]], dtype=torch.int32)]
        want, mag, new = oracle.attend(q, ref, k, v, n, True)
        assert ((out.double().cpu() - want).abs() <= _tol(q, ref, k, mag, want)).all()
        for x, y in zip(pages, new):
            assert torch.equal(x[1, table[0].long()].cpu(), y[0])


def test_refusals():
    g = torch.Generator().manual_seed(1)
    B, H, ps, D, M = 2, 2, 16, 128, 4
    c = _to(oracle.dealt(2, 10, H, ps, D, B, M, [64, 64], g))
    q, k = _rows(g, B, 1, 4, D).to(DEV), _rows(g, B, 1, H, D).to(DEV)

    def call(q=q, c=c, k=k, v=k, lens=3, **kw):
        return flash_attn_with_paged_kvcache(q, c, k, v, lens, **kw)

    call()
    for kw, needle in (
            (dict(q=q.float()), "bf16"), (dict(q=q[:1]), "must be"), (dict(q=q[:, :, :3].contiguous()), "multiple"),
            (dict(q=q[..., :64].contiguous()), "must be"), (dict(q=q[:, :0]), "must be"), (dict(v=None), "together"),
            (dict(k=k[:, :, :1].contiguous()), "k must"), (dict(v=k.cpu()), "GPU tensor"), (dict(layer=2), "layer"), (dict(layer=-1), "layer"),
            (dict(lens=-1), "cache_seqlens"), (dict(lens=65), "cache_seqlens"),
            (dict(lens=torch.zeros(3, dtype=torch.int32, device=DEV)), "cache_seqlens"),
            (dict(lens=torch.zeros(2, device=DEV)), "cache_seqlens"), (dict(lens=torch.zeros(2, dtype=torch.int32)), "cache_seqlens"),
            (dict(c=c._replace(k_pages=c.k_pages.float())), "k_pages"), (dict(c=c._replace(v_pages=c.v_pages[:1])), "differ"),
            (dict(c=c._replace(k_pages=c.k_pages.transpose(2, 3))), "contiguous"),
            (dict(c=c._replace(refs=c.refs[:9])), "refs"), (dict(c=c._replace(refs=c.refs.long())), "refs"),
            (dict(c=c._replace(page_table=c.page_table.long())), "page_table"), (dict(c=c._replace(page_table=c.page_table[:1])), "must be"),
            (dict(c=c._replace(page_table=c.page_table[:1].expand(2, 4))), "page_table"),
            (dict(c=c._replace(page_table=c.page_table.t().contiguous().t())), "page_table"),
            (dict(c=c._replace(v_pages=c.k_pages)), "overlap"), (dict(k=c.k_pages[0, 0, :, :2].transpose(0, 1)[None].expand(2, -1, -1, -1)[:, :1]), "overlap"),
            (dict(c=c._replace(k_pages=c.k_pages.repeat(1, 1, 1, 1, 2)[..., :192].contiguous())), "differ")):
        with pytest.raises(ValueError, match=needle):
            call(**kw)
