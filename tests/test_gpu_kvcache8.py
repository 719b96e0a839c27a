"""GPU: attention over an 8-bit KV cache against the fp64 oracle; the cache it leaves bitwise.

Tolerances (u = 2^-24). A score sums 128 products in fp32, off by at most 140 u of the sum of their
magnitudes A, and exponentials of scores off by d change each weight by d relative, a sum of weighted
rows by 2 d of the sum of p |v|; n keys add n u more, and the splits' joins 100 u. out is rounded to
bf16, 2^-8 relative. A call on an empty cache runs the training forward, which rounds the
probabilities to bf16: 2^-8 of the sum of p |v| on top, and its exponentials' argument with it.
Several queries multiply p scale as two bf16 terms, each cut: of 2^e m, 1 <= m < 2, the first leaves
r < 2^(e-7), exactly, and the second less than 2^-7 of r's leading bit, at most 2^(e-8): 2^-15 of p.
Codes, scales and bf16 rows are equal bit for bit.
"""
import math

import pytest
import torch

from oracle import kvcache8_oracle as oracle
from prefixlm import KVCacheQ8, flash_attn_with_kvcache, flash_attn_with_kvcache_q8, kvcache_q8
from prefixlm.kvcache8 import kvcache_q8_attn

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
CODES = [torch.float8_e4m3fn, torch.int8]
U = 2.0 ** -24


def _rows(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).bfloat16()


def _filled(B, H, Smax, dtype, g):
    """A cache whose blocks and ring hold random rows (the two need not agree: calls read one or the
    other)."""
    cache = oracle.empty(B, H, Smax, dtype)
    for c in range(2):
        for b in range(B):
            for h in range(H):
                for blk in range(Smax // 64):
                    codes, scale = oracle.round_block(_rows(g, 64, 128, scale=1.0 + 3.0 * ((blk + h) % 3)), dtype)
                    cache[c][b, h, blk * 64:blk * 64 + 64], cache[2 + c][b, h, blk] = codes, scale
        cache[4 + c][:] = _rows(g, B, H, 128, 128)
    return cache


def _bits(x):
    return x.contiguous().view(torch.uint8) if x.element_size() == 1 else x


def _same_cache(got, want, tag=""):
    for name, a, b in zip(KVCacheQ8._fields, got, want):
        off = _bits(a.cpu()) != _bits(b)
        n = int((off & ~(torch.isnan(a.cpu().float()) & torch.isnan(b.float()))).sum())
        assert n == 0, (tag, name, n, off.nonzero()[:4].tolist())


def _to(cache):
    return KVCacheQ8(*(x.to(DEV) for x in cache))


def _tol(q, cache, k, mag, want, n, prefill=False, softmax_scale=None):
    top = max(float(cache[2].abs().max()) * oracle.code_max(cache[0].dtype), float(cache[4].float().abs().max()),
              float(k.float().abs().max()) if k is not None else 0.0)      # the largest magnitude of a key
    s = 1.0 / math.sqrt(128) if softmax_scale is None else abs(softmax_scale)
    A = q.double().abs().sum(-1, keepdim=True) * top * s
    rel = 2 * 140 * U * A + (n + 100) * U + (2.0 ** -7 if prefill else 2.0 ** -15 if q.shape[1] > 1 else 0.0)
    return 2.0 ** -8 * want.abs() + rel * mag + 1e-30


def _check(q, cache, k, v, lens, causal, tag="", prefill=False, softmax_scale=None):
    dev = _to(cache)
    out = flash_attn_with_kvcache_q8(q.to(DEV), dev, k.to(DEV) if k is not None else None, v.to(DEV) if v is not None else None,
                                     lens.to(DEV) if isinstance(lens, torch.Tensor) else lens, softmax_scale, causal)
    want, mag, new = oracle.attend(q, cache, k, v, lens, causal, softmax_scale)
    got = out.double().cpu()
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), tag
    ok = torch.isfinite(want)
    over = ((got - want).abs() - _tol(q, cache, k, mag, want, cache[0].shape[2], prefill, softmax_scale))[ok]
    assert over.max().item() <= 0, (tag, (got - want).abs()[ok].max().item())
    _same_cache(dev, new, tag)
    return out


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("S", [1, 2, 31, 45, 64, 65, 130])
def test_matches_oracle(S, causal, dtype):
    H, Smax = 2, 384
    lens = torch.tensor([0, 1, 62, 63, 64, 65, 127, 128, 190, Smax - S], dtype=torch.int32)
    g = torch.Generator().manual_seed(S)
    B = lens.numel()
    q, k, v = (_rows(g, B, S, H, 128) for _ in range(3))
    _check(q, _filled(B, H, Smax, dtype, g), k, v, lens, causal, (S, causal))


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("S", [1, 5, 70])
@pytest.mark.parametrize("causal", [False, True])
def test_without_new_rows_and_past_the_end(S, causal, dtype):
    """The cache alone, and rows that no longer fit; queries that see no key give 0."""
    H, Smax = 3, 192
    lens = torch.tensor([0, 1, 2, 64, 100, 191, 192], dtype=torch.int32)
    g = torch.Generator().manual_seed(20 + S)
    B = lens.numel()
    q, k, v = (_rows(g, B, S, H, 128) for _ in range(3))
    cache = _filled(B, H, Smax, dtype, g)
    out = _check(q, cache, None, None, lens, causal, "alone")
    assert not out[0].any()
    _check(q, cache, k, v, lens, causal, "past the end")
    odd = torch.tensor([-5, -1, 193, 1000, 2**31 - 1, -2**31, 64], dtype=torch.int32)
    _check(q, cache, k, v, odd, causal, "outside")
    _check(q, cache, None, None, odd, causal, "outside, alone")


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("B,S,causal", [(1, 1, False), (2, 63, True), (1, 64, False), (2, 129, True), (3, 200, False), (1, 256, True)])
def test_prefill(B, S, causal, dtype):
    g = torch.Generator().manual_seed(30 + S)
    q, k, v = (_rows(g, B, S, 2, 128) for _ in range(3))
    _check(q, _filled(B, 2, 256, dtype, g), k, v, 0, causal, "prefill", prefill=True)
    _check(q, _filled(B, 2, 256, dtype, g), k, v, torch.zeros(B, dtype=torch.int32), causal, "empty")


@pytest.mark.parametrize("dtype", CODES)
def test_int_lengths_scales_and_splits(dtype):
    g = torch.Generator().manual_seed(40)
    for S in (1, 3):
        q, k, v = (_rows(g, 1, S, 1, 128) for _ in range(3))
        cache = _filled(1, 1, 4096, dtype, g)
        for n, scale in ((4000, None), (4032, -0.2), (777, 0.0), (4095, 1.5)):
            _check(q, cache, k, v, n, True, (S, n), softmax_scale=scale)


def test_the_cache_does_not_depend_on_the_pieces():
    """One prompt in one call, in pieces, and row by row; and rows taken back and brought again."""
    B, H, n = 2, 2, 300
    g = torch.Generator().manual_seed(50)
    q, k, v = (_rows(g, B, n, H, 128).to(DEV) for _ in range(3))

    def bring(cache, at, stop, piece):
        while at < stop:
            m = min(piece, stop - at)
            flash_attn_with_kvcache_q8(q[:, at:at + m], cache, k[:, at:at + m], v[:, at:at + m],
                                       torch.full((B,), at, dtype=torch.int32, device=DEV), causal=True)
            at += m

    for dtype in CODES:
        want = kvcache_q8(B, n, H, dtype=dtype)
        flash_attn_with_kvcache_q8(q, want, k, v, 0, causal=True)
        for piece in (1, 7, 64, 100, 150):
            got = kvcache_q8(B, n, H, dtype=dtype)
            bring(got, 0, n, piece)
            slots = torch.arange(n // 64 * 64 - 64, n, device=DEV) % 128
            for name, a, b in zip(KVCacheQ8._fields, got, want):
                a, b = (a[:, :, slots], b[:, :, slots]) if "recent" in name else (_bits(a), _bits(b))
                assert torch.equal(a, b), (dtype, piece, name)
            # 64 rows back, into blocks that were complete, and on again with other rows, then these
            out = flash_attn_with_kvcache_q8(q[:, :1], got, cache_seqlens=n - 64)
            ref = flash_attn_with_kvcache_q8(q[:, :1], want, cache_seqlens=n - 64)
            assert torch.equal(out, ref)
            flash_attn_with_kvcache_q8(q[:, :40], got, q[:, :40], k[:, :40], n - 64)
            bring(got, n - 64, n, piece)
            for name, a, b in zip(KVCacheQ8._fields, got, want):
                a, b = (a[:, :, slots[-44:]], b[:, :, slots[-44:]]) if "recent" in name else (_bits(a), _bits(b))
                assert torch.equal(a, b), ("again", dtype, piece, name)


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("S", [1, 3, 70])
def test_rows_that_no_query_sees_do_not_matter(S, dtype):
    """NaN behind the lengths, in codes, scales and ring."""
    B, H, Smax = 4, 2, 320
    lens = torch.tensor([0, 10, 64, 200], dtype=torch.int32)
    g = torch.Generator().manual_seed(60 + S)
    q, k, v = (_rows(g, B, S, H, 128) for _ in range(3))
    cache = _filled(B, H, Smax, dtype, g)
    want = flash_attn_with_kvcache_q8(q.to(DEV), _to(cache), k.to(DEV), v.to(DEV), lens.to(DEV), causal=True)
    for b, n in enumerate(lens.tolist()):
        for c in range(2):
            cache[c][b, :, n // 64 * 64:].view(torch.uint8).fill_(0x7f)
            cache[2 + c][b, :, n // 64:] = math.nan
            free = sorted(set(range(128)) - {j % 128 for j in range(n // 64 * 64, n)})
            cache[4 + c][b, :, free] = math.nan
    got = flash_attn_with_kvcache_q8(q.to(DEV), _to(cache), k.to(DEV), v.to(DEV), lens.to(DEV), causal=True)
    assert torch.equal(got, want)
    # a later new row that is not finite stays out of the queries before it
    if S > 1:
        k2, v2 = k.clone(), v.clone()
        k2[:, -1], v2[:, -1] = math.inf, math.nan
        hid = flash_attn_with_kvcache_q8(q.to(DEV), _to(cache), k2.to(DEV), v2.to(DEV), lens.to(DEV), causal=True)
        ref, mag, _ = oracle.attend(q, cache, k, v, lens, True)
        assert ((hid.double().cpu() - ref).abs() <= _tol(q, [x.nan_to_num(0) if x.dtype == torch.float32 else x for x in cache[:4]]
                                                           + [x.nan_to_num(0) for x in cache[4:]], k, mag, ref, Smax))[:, :-1].all()


@pytest.mark.parametrize("dtype", CODES)
def test_cached_rows_past_a_causal_query(dtype):
    """Without new rows a causal query misses the last cached ones: their NaN must not reach it."""
    g = torch.Generator().manual_seed(70)
    S, n = 5, 128
    q = _rows(g, 1, S, 1, 128)
    cache = _filled(1, 1, 192, dtype, g)
    want, mag, _ = oracle.attend(q, cache, lens=n, causal=True)
    cache[3][0, 0, 1] = math.nan
    got = flash_attn_with_kvcache_q8(q.to(DEV), _to(cache), cache_seqlens=n, causal=True)
    assert torch.isnan(got).all()                     # rows 64 .. 127 are seen by every query here
    q = _rows(g, 1, 70, 1, 128)
    got = flash_attn_with_kvcache_q8(q.to(DEV), _to(cache), cache_seqlens=n, causal=True).double().cpu()
    want, mag, _ = oracle.attend(q, cache, lens=n, causal=True)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.isfinite(got[0, :6]).all()
    ok = torch.isfinite(want)
    cache[3].nan_to_num_(0)
    assert ((got - want).abs() <= _tol(q, cache, None, mag, want, 192))[ok].all()


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("S", [1, 2, 40])
def test_extreme_rows(S, dtype):
    """Blocks of zeros, of the smallest and of the largest values; keys of the type's lowest value."""
    B, H, Smax, n = 1, 4, 256, 150
    g = torch.Generator().manual_seed(80 + S)
    big = torch.finfo(torch.bfloat16).max
    k, v = (_rows(g, B, n + S, H, 128) for _ in range(2))
    k[:, :64, 0], v[:, :64, 0] = 0, 0
    k[:, :64, 1] *= 2.0 ** -120
    v[:, :64, 1] *= 2.0 ** -130
    v[:, :64, 2] *= 2.0 ** 100
    k[:, 64:n, 3] = torch.finfo(torch.bfloat16).min
    q = _rows(g, B, S, H, 128)
    q[:, :, 3] = q[:, :, 3].abs()
    _, _, cache = oracle.attend(k[:, :n], oracle.empty(B, H, Smax, dtype), k[:, :n], v[:, :n], 0)
    assert cache[2][0, 0, 0] == 2.0 ** -126
    out = flash_attn_with_kvcache_q8(q.to(DEV), _to(cache), k[:, n:].to(DEV), v[:, n:].to(DEV), n).double().cpu()
    want, mag, _ = oracle.attend(q, cache, k[:, n:], v[:, n:], n)
    assert torch.isfinite(out).all()
    rel = ((out - want).abs() / (mag + 1e-300))
    assert rel.max().item() <= 2.0 ** -8 + 2e-3       # scores here are below 2^6: 2 * 140 u * 2^6 * 10
    # a query that is not finite
    q[0, 0, 0, 0] = math.inf
    bad = flash_attn_with_kvcache_q8(q.to(DEV), _to(cache), k[:, n:].to(DEV), v[:, n:].to(DEV), n)
    assert torch.isfinite(bad[0, :, 1:]).all() and not torch.isfinite(bad[0, 0, 0]).any()
    # rows that are not finite: their block reads as NaN, the others as before
    k[0, 3, 2, 5], v[0, 70, 1, 9] = math.inf, math.nan
    dev = kvcache_q8(B, Smax, H, dtype=dtype)
    flash_attn_with_kvcache_q8(k[:, :n].to(DEV), dev, k[:, :n].to(DEV), v[:, :n].to(DEV), 0)
    _, _, new = oracle.attend(k[:, :n], oracle.empty(B, H, Smax, dtype), k[:, :n], v[:, :n], 0)
    for a, b in ((dev.k_scale, new[2]), (dev.v_scale, new[3])):
        fin = torch.isfinite(b)
        assert torch.equal(torch.isfinite(a.cpu()), fin) and torch.equal(a.cpu()[fin], b[fin])
    out = flash_attn_with_kvcache_q8(q[:, :, 3:].to(DEV), KVCacheQ8(*(x[:, 3:].contiguous() for x in dev)), cache_seqlens=n)
    assert torch.isfinite(out).all()
    assert torch.isnan(flash_attn_with_kvcache_q8(q.to(DEV), dev, cache_seqlens=n)[0, :, 1:3]).all()
    assert big > 1e38


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("exponent", [0, 127, 90, -50, -59, -60, -61, -80, -105, -126])
def test_every_mantissa_is_rounded_as_by_division(exponent, dtype):
    """Blocks with each of the 128 mantissas of their largest magnitude (and so of their scale) and rows
    of all mantissas, signs and 24 binades below it: codes equal those of the division."""
    m = torch.arange(128, dtype=torch.int32)
    sign = torch.tensor([0, 1], dtype=torch.int32)
    e = torch.arange(1, 25, dtype=torch.int32)
    biased = (exponent + 127 - e).clamp_min(0)
    bits = (sign[:, None, None] << 15) | (biased[None, :, None] << 7) | m[None, None, :]       # 2 * 24 * 128
    rows = torch.zeros(128, 64, 128, dtype=torch.int32)
    rows[:, :48] = bits.reshape(48, 128)
    rows[:, 63, 0] = (max(exponent + 127, 0) << 7) | m
    rows = rows.to(torch.int16).view(torch.bfloat16)                                            # [block, 64, 128]
    B = 8
    k = rows.reshape(B, 16 * 64, 1, 128)
    dev = kvcache_q8(B, 16 * 64, 1, dtype=dtype)
    flash_attn_with_kvcache_q8(k.to(DEV), dev, k.to(DEV), k.flip(0).to(DEV), 0)
    for codes, scale, x in ((dev.k_codes, dev.k_scale, k), (dev.v_codes, dev.v_scale, k.flip(0))):
        for b in range(B):
            for blk in range(16):
                c, s = oracle.round_block(x[b, blk * 64:blk * 64 + 64, 0], dtype)
                assert scale[b, 0, blk].item() == s.item()
                assert torch.equal(_bits(codes[b, 0, blk * 64:blk * 64 + 64].cpu()), _bits(c)), (b, blk)


def test_strided_rows():
    """q, k and v as the slices of one projection, and the keys of one token for every row."""
    B, S, H, n = 2, 3, 4, 100
    g = torch.Generator().manual_seed(90)
    qkv = _rows(g, B, S, 3 * H, 128).to(DEV)
    q, k, v = qkv.split(H, dim=2)
    for S2, take in ((3, slice(0, 3)), (1, slice(1, 2))):
        for dtype in CODES:
            cache = _filled(B, H, 192, dtype, torch.Generator().manual_seed(91))
            a, b = _to(cache), _to(cache)
            out = flash_attn_with_kvcache_q8(q[:, take], a, k[:, take], v[:, take], n)
            ref = flash_attn_with_kvcache_q8(q[:, take].contiguous(), b, k[:, take].contiguous(), v[:, take].contiguous(), n)
            assert torch.equal(out, ref)
            _same_cache(a, [x.cpu() for x in b])
            one = k[:, :1, :1].expand(B, S2, H, 128)
            a, b = _to(cache), _to(cache)
            assert torch.equal(flash_attn_with_kvcache_q8(q[:, take], a, one, one, n),
                               flash_attn_with_kvcache_q8(q[:, take], b, one.contiguous(), one.contiguous(), n))
            _same_cache(a, [x.cpu() for x in b])


@pytest.mark.parametrize("S", [1, 2])
def test_caches_past_32_bits(S):
    """Codes of more than 2^32 bytes a tensor; the last head of the last sequence."""
    B, H, Smax = 2, 16, 1100032
    n = 1100000 - 7
    cache = KVCacheQ8(*(torch.zeros(B, H, Smax, 128, dtype=torch.int8, device=DEV) for _ in range(2)),
                      *(torch.full((B, H, Smax // 64), 0.01, device=DEV) for _ in range(2)),
                      *(torch.zeros(B, H, 128, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)))
    cache.k_codes[-1, -1].random_(-100, 100)
    cache.v_codes[-1, -1].random_(-100, 100)
    q, k, v = (torch.randn(B, S, H, 128, device=DEV).bfloat16() for _ in range(3))
    out = flash_attn_with_kvcache_q8(q, cache, k, v, n)
    held = n // 64 * 64
    rows = [torch.cat((c[-1, -1, :held].double() * float(torch.tensor(0.01)), torch.zeros(n - held, 128, device=DEV).double(),
                       x[-1, :, -1].double())) for c, x in ((cache.k_codes, k), (cache.v_codes, v))]
    p = torch.softmax(q[-1, :, -1].double() @ rows[0].t() / math.sqrt(128), -1)
    want, mag = p @ rows[1], p @ rows[1].abs()
    # a split adds about 1.1e6 / 64 keys in 32 groups, one after another: (600 + 100) u, and 140 u of scores below 8
    tol = 2.0 ** -8 * want.abs() + (2 * 140 * U * 8 * 10 + 20000 * U) * mag
    assert ((out[-1, :, -1].double() - want).abs() <= tol).all()
    j = torch.arange(n, n + S, device=DEV) % 128
    assert torch.equal(cache.k_recent[:, :, j], k.transpose(1, 2))


def test_graph_replays():
    """A captured decode step, replayed over block borders with lengths that move on the device."""
    B, H = 3, 2
    g = torch.Generator().manual_seed(100)
    for dtype in CODES:
        cpu = _filled(B, H, 512, dtype, g)
        a, b = _to(cpu), _to(cpu)
        start = torch.tensor([60, 126, 0], dtype=torch.int32, device=DEV)
        lens = start.clone()
        q, k, v = (_rows(g, B, 1, H, 128).to(DEV) for _ in range(3))

        def step(cache, n):
            return flash_attn_with_kvcache_q8(q, cache, k, v, n)

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(_to(cpu), lens)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(a, lens)
            lens.add_(1)
        a_start = [x.clone() for x in b]
        for x, y in zip(a, a_start):
            x.copy_(y)
        lens.copy_(start)
        eager = start.clone()
        for i in range(8):
            for x in (q, k, v):
                x.copy_(_rows(g, B, 1, H, 128))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, step(b, eager)), i
            eager.add_(1)
            _same_cache(a, [x.cpu() for x in b], i)


def test_other_stream_compile_and_both_host_paths():
    B, H = 2, 2
    g = torch.Generator().manual_seed(110)
    cpu = _filled(B, H, 256, torch.float8_e4m3fn, g)
    q, k, v = (_rows(g, B, 1, H, 128).to(DEV) for _ in range(3))
    lens = torch.tensor([63, 130], dtype=torch.int32, device=DEV)
    a, b, c, d = (_to(cpu) for _ in range(4))
    want = flash_attn_with_kvcache_q8(q, a, k, v, lens)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = flash_attn_with_kvcache_q8(q, b, k, v, lens)
    s.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(kvcache_q8_attn(q, k, v, *c, lens, 0, False, 128 ** -0.5), want)

    @torch.compile(dynamic=False, fullgraph=True)
    def step(q, k, v, cache, lens):
        return flash_attn_with_kvcache_q8(q, cache, k, v, lens)

    assert torch.equal(step(q, k, v, d, lens), want)
    for other in (b, c, d):
        _same_cache(other, [x.cpu() for x in a])


def test_repeats_bitwise():
    g = torch.Generator().manual_seed(120)
    for S in (1, 9):
        q, k, v = (_rows(g, 2, S, 3, 128).to(DEV) for _ in range(3))
        cpu = _filled(2, 3, 1024, torch.int8, g)
        outs = [flash_attn_with_kvcache_q8(q, _to(cpu), k, v, 1000) for _ in range(3)]
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_close_to_the_bf16_cache():
    """Against the bf16 cache's own call the rounding of K and V to 8 bits is what differs: the error of
    e4m3 rows is uniform within 2^-4 relative (2^-4 / sqrt(3) at most in the mean square), and the
    outputs average it over their keys; the bound takes no averaging."""
    B, H, n = 2, 4, 500
    g = torch.Generator().manual_seed(130)
    kc, vc = (_rows(g, B, 1024, H, 128).to(DEV) for _ in range(2))
    q, k, v = (_rows(g, B, 1, H, 128).to(DEV) for _ in range(3))
    cache = kvcache_q8(B, 1024, H)
    flash_attn_with_kvcache_q8(kc[:, :n], cache, kc[:, :n], vc[:, :n], 0)
    got = flash_attn_with_kvcache_q8(q, cache, k, v, n).double()
    want = flash_attn_with_kvcache(q, kc, vc, k=k, v=v, cache_seqlens=n).double()
    assert (got - want).abs().mean().item() <= 2.0 ** -4            # |v| about 1, weights that sum to 1
    assert (got - want).abs().max().item() > 0


def test_refusals_on_the_gpu():
    B, H = 2, 2
    q = torch.zeros(B, 1, H, 128, dtype=torch.bfloat16, device=DEV)
    good = kvcache_q8(B, 128, H)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)

    def refuse(needle, cache=good, q=q, k=None, v=None, lens=lens, error=ValueError):
        with pytest.raises(error, match=needle):
            flash_attn_with_kvcache_q8(q, cache, k, v, lens)

    refuse("bf16", q=q.float())
    refuse("together", k=q)
    refuse("must be", k=q[:1], v=q[:1])
    refuse("q must be", q=q[:, :0])
    refuse("k_codes", cache=good._replace(k_codes=good.k_codes.view(torch.uint8)))
    refuse("k_codes must be", cache=kvcache_q8(B + 1, 128, H))
    refuse("v_codes must be", cache=good._replace(v_codes=good.v_codes.view(torch.int8)))
    refuse("k_scale must be", cache=good._replace(k_scale=good.k_scale[..., :1].contiguous()))
    refuse("v_recent must be", cache=good._replace(v_recent=good.v_recent.float()))
    refuse("contiguous", cache=good._replace(v_recent=good.v_recent.transpose(2, 3).contiguous().transpose(2, 3)))
    refuse("multiple of 64", cache=good._replace(k_codes=good.k_codes[:, :, :100].contiguous()))
    refuse("overlap", cache=good._replace(v_codes=good.k_codes))
    refuse("cache_seqlens", lens=lens[:1])
    refuse("cache_seqlens", lens=lens.float())
    refuse("outside", lens=129)
    refuse("outside", lens=-1)
    a = flash_attn_with_kvcache_q8(q, good, q, q, torch.tensor([3, 5], device=DEV))          # int64 lengths
    assert a.shape == q.shape


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("S", [2, 33, 65])
def test_every_end_of_a_tile(S, dtype):
    """Lengths at which the codes, the bf16 rows and the splits end at every place of a tile."""
    print(f"[case] ends {S} {dtype}", flush=True)
    H, Smax = 1, 256
    lens = torch.cat((torch.arange(0, Smax - S, 5), torch.tensor([Smax - S]))).int()
    g = torch.Generator().manual_seed(77 + S)
    B = lens.numel()
    q, k, v = (_rows(g, B, S, H, 128) for _ in range(3))
    cache = _filled(B, H, Smax, dtype, g)
    _check(q, cache, k, v, lens, True, "causal")
    _check(q, cache, k, v, lens, False, "all")
    _check(q, cache, None, None, lens, True, "alone")


@pytest.mark.parametrize("S", [7, 64, 100])
def test_one_row_with_many_splits(S):
    """One batch row and a long cache: the most splits, whose ends fall into codes, ring and new rows."""
    print(f"[case] splits {S}", flush=True)
    g = torch.Generator().manual_seed(S)
    q, k, v = (_rows(g, 1, S, 2, 128) for _ in range(3))
    cache = _filled(1, 2, 4096, torch.float8_e4m3fn, g)
    for n in (0, 64, 1000, 2047, 4096 - S):
        _check(q, cache, k, v, torch.tensor([n], dtype=torch.int32), True, n)
