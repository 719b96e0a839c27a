"""GPU: the 8-bit cache by the sizes that choose its kernels, captured calls of several queries, batches
of uneven lengths, and rows taken back.

Tolerances (u = 2^-24, of the sum of p |v|): a score's 128 products, off by 140 u of their magnitudes,
change a weight twice; n keys add n u and joins 100 u; several queries multiply the probabilities' 24 bits;
half a bf16 step of the output. Caches are equal bit for bit."""
import math

import pytest
import torch

from oracle import kvcache8_oracle as oracle
from prefixlm import KVCacheQ8, flash_attn_with_kvcache_q8, kvcache_q8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24
CODES = [torch.float8_e4m3fn, torch.int8]


def _rows(g, *shape):
    return torch.randn(*shape, generator=g).bfloat16()


def _filled(B, H, Smax, dtype, g):
    """Random codes, scales and rows, the same for every fourth (batch row, head)."""
    cache = oracle.empty(B, H, Smax, dtype)
    n = min(4, B * H)
    for c in range(2):
        x = torch.randn(n, Smax // 64, 64, 128, generator=g)
        codes, scales = zip(*(oracle.round_block(b.bfloat16(), dtype) for b in x.view(-1, 64, 128)))
        codes, scales = torch.stack(codes).view(torch.uint8).view(n, Smax, 128), torch.stack(scales).view(n, Smax // 64)
        at = torch.arange(B * H) % n
        cache[c] = codes[at].view(B, H, Smax, 128).view(dtype)
        cache[2 + c] = scales[at].view(B, H, Smax // 64).contiguous()
        cache[4 + c] = _rows(g, n, 128, 128)[at].view(B, H, 128, 128)
    return cache


def _to(cache):
    return KVCacheQ8(*(x.to(DEV).clone() for x in cache))


def _bits(x):
    return x.contiguous().view(torch.uint8)


def _tol(q, cache, k, mag, want):
    top = max(float(cache[2].abs().max()) * oracle.code_max(cache[0].dtype), float(cache[4].float().abs().max()),
              float(k.float().abs().max()) if k is not None else 0.0)
    A = q.double().abs().sum(-1, keepdim=True) * top / math.sqrt(128)
    return 2.0 ** -8 * want.abs() + (2 * 140 * U * A + (cache[0].shape[2] + 100) * U) * mag + 1e-30


def _check(q, cache, k, v, lens, causal, only=None):
    """`only`: the batch rows that are compared."""
    dev = _to(cache)
    out = flash_attn_with_kvcache_q8(q.to(DEV), dev, k.to(DEV) if k is not None else None,
                                     v.to(DEV) if v is not None else None, lens.to(DEV), causal=causal)
    at = list(range(q.shape[0])) if only is None else only
    sub = [x[at] for x in cache]
    args = [x[at] if x is not None else None for x in (k, v)]
    want, mag, new = oracle.attend(q[at], sub, *args, lens[at], causal)
    over = (out[at].double().cpu() - want).abs() - _tol(q[at], sub, args[0], mag, want)
    assert over.max().item() <= 0, over.max().item()
    for name, a, b in zip(KVCacheQ8._fields, dev, new):
        assert torch.equal(_bits(a[at].cpu()), _bits(b)), name


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("B,H,Smax", [(40, 16, 512), (130, 4, 256), (32, 16, 512), (33, 16, 64), (40, 16, 576), (3, 2, 1536),
                                      (3, 2, 1600), (2, 1, 1984), (12, 16, 2048), (11, 17, 2048)])
def test_decode_by_its_sizes(B, H, Smax, dtype):
    """One split with four waves (many pairs, short caches) and with eight, several splits."""
    print(f"[case] {B} {H} {Smax} {dtype}", flush=True)
    g = torch.Generator().manual_seed(B)
    q, k, v = (_rows(g, B, 1, H, 128) for _ in range(3))
    cache = _filled(B, H, Smax, dtype, g)
    lens = torch.randint(0, Smax, (B,), generator=g, dtype=torch.int32)
    lens[0], lens[1], lens[-1] = Smax - 1, 63, Smax
    _check(q, cache, k, v, lens, False, only=[0, 1, B // 2, B - 1])


@pytest.mark.parametrize("S", [1, 7, 100])
def test_one_long_sequence_among_short_ones(S):
    B, H, Smax = 16, 16, 8192
    g = torch.Generator().manual_seed(S)
    q, k, v = (_rows(g, B, S, H, 128) for _ in range(3))
    cache = _filled(B, H, Smax, torch.int8, g)
    lens = torch.tensor([0, 1, 63, 64, 65, 100, 127, 128] + [5] * 7 + [Smax - S], dtype=torch.int32)
    _check(q, cache, k, v, lens, True, only=[0, 3, 15])


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("S,Smax", [(2, 512), (8, 512), (33, 1024), (64, 1024), (65, 1024), (130, 2048)])
def test_captured_calls_of_several_queries(S, Smax, dtype):
    """The speculative step and the chunk: replayed with lengths that move on the device, forth by S and
    back by up to 64, between eager calls."""
    print(f"[case] {S} {dtype}", flush=True)
    B, H = 3, 2
    g = torch.Generator().manual_seed(S)
    cpu = _filled(B, H, Smax, dtype, g)
    a, b = _to(cpu), _to(cpu)
    lens = torch.tensor([60, 126, 0], dtype=torch.int32, device=DEV)
    q, k, v = (_rows(g, B, S, H, 128).to(DEV) for _ in range(3))

    def step(cache, n):
        return flash_attn_with_kvcache_q8(q, cache, k, v, n, causal=True)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(_to(cpu), lens)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a, lens)
    for x, y in zip(a, _to(cpu)):
        x.copy_(y)
    for i in range(6):
        for x in (q, k, v):
            x.copy_(_rows(g, B, S, H, 128))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(b, lens.clone())), i
        for name, x, y in zip(KVCacheQ8._fields, a, b):
            assert torch.equal(_bits(x), _bits(y)), (i, name)
        lens.add_(S - min(64, (i * 17) % (S + 1)))


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("furthest", [191, 192, 200, 129])
def test_rows_taken_back_from_the_furthest_length(furthest, dtype):
    """Lengths go back, again and again, to the block before the furthest length's incomplete one, and
    to whole blocks anywhere; the result is that of a cache that took the rows once."""
    H, Smax = 2, 320
    g = torch.Generator().manual_seed(furthest)
    rows = [_rows(g, 1, 320, H, 128) for _ in range(2)]          # the sequence as it stands
    dev = kvcache_q8(1, Smax, H, dtype=dtype)

    def bring(at, k, v):
        for x, new in zip(rows, (k, v)):
            x[:, at:at + new.shape[1]] = new
        q = _rows(g, 1, k.shape[1], H, 128)
        lens = torch.tensor([at], dtype=torch.int32, device=DEV)
        out = flash_attn_with_kvcache_q8(q.to(DEV), dev, k.to(DEV), v.to(DEV), lens, causal=True).double().cpu()
        held = oracle.empty(1, H, Smax, dtype)
        for c, x in enumerate(rows):
            for h in range(H):
                for blk in range(at // 64):
                    codes, scale = oracle.round_block(x[0, blk * 64:blk * 64 + 64, h], dtype)
                    held[c][0, h, blk * 64:blk * 64 + 64], held[2 + c][0, h, blk] = codes, scale
                for j in range(at // 64 * 64, at):
                    held[4 + c][0, h, j % 128] = x[0, j, h]
        want, mag, _ = oracle.attend(q, held, k, v, at, True)
        assert ((out - want).abs() <= _tol(q, held, k, mag, want)).all(), at

    for at in range(0, furthest, 50):
        n = min(50, furthest - at)
        bring(at, *(x[:, at:at + n].clone() for x in rows))
    low, end = furthest // 64 * 64 - 64, furthest
    for at, n in ((furthest - 64, 5), (furthest - 63, 4), (low + 3, 5), (low + 1, 5), (low, 7), (low + 4, 60), (low + 40, 3),
                  (0, 64), (64, 1), (0, 70)):
        assert at <= end                                          # rows behind the last call's are gone
        n = min(furthest - at, n)
        bring(at, _rows(g, 1, n, H, 128), _rows(g, 1, n, H, 128))
        end = at + n


def test_back_to_a_whole_block_and_on():
    """Far below the window, to multiples of 64: from there the window counts anew."""
    H, Smax, dtype = 1, 512, torch.int8
    g = torch.Generator().manual_seed(5)
    k, v = (_rows(g, 1, Smax, H, 128) for _ in range(2))
    k2, v2 = (_rows(g, 1, Smax, H, 128) for _ in range(2))
    got, want = kvcache_q8(1, Smax, H, dtype=dtype), kvcache_q8(1, Smax, H, dtype=dtype)

    def call(cache, at, n, k, v):
        d = [x[:, at:at + n].to(DEV) for x in (k, k, v)]
        return flash_attn_with_kvcache_q8(d[0], cache, d[1], d[2], torch.tensor([at], dtype=torch.int32, device=DEV), causal=True)

    call(got, 0, 300, k, v)
    call(want, 0, 128, k, v)
    for at, n in ((128, 5), (133, 64), (197, 30), (130, 3), (133, 1)):      # 130: two blocks below 227's is 128
        assert torch.equal(call(got, at, n, k2, v2), call(want, at, n, k2, v2)), at
    call(want, 0, 64, k, v)
    assert torch.equal(call(got, 64, 9, k2, v2), call(want, 64, 9, k2, v2))
