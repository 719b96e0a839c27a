"""GPU: prompts into an empty cache whose rows lie too far apart for the forward's 32-bit offsets take
the extend kernel. One head of a wide projection, on both sides of the limit.

Tolerances (u = 2^-24, of the sum of p |v|): scores here are below 2^7 in magnitudes, off by 2 * 140 u
of that; n keys add n u, joins 100 u; below the limit the probabilities are rounded to bf16, 2^-8, and
their exponents' argument with it; half a bf16 step of the output. Rows in the cache are equal."""
import math

import pytest
import torch

from prefixlm import flash_attn_with_kvcache, flash_attn_with_kvcache_q8, kvcache_q8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24
WIDE = 65536                       # (S + 256) rows of it reach 2^31 bytes at S = 16128


@pytest.fixture(scope="module")
def wide():
    x = torch.zeros(16200, WIDE, dtype=torch.bfloat16, device=DEV)
    x[:, :384] = torch.randn(16200, 384, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    yield x
    del x


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("S", [16127, 16128, 16200])
@pytest.mark.parametrize("kind", ["bf16", "e4m3", "int8"])
def test_prompts_on_both_sides_of_the_limit(wide, kind, S, causal):
    print(f"[case] {kind} {S} {causal}", flush=True)
    Smax = 16256
    q, k, v = (wide[:S, 128 * i:128 * i + 128].reshape(1, S, 1, 128) for i in range(3))
    assert q.stride(1) == WIDE and q.data_ptr() == wide.data_ptr()
    near = [x.contiguous() for x in (q, k, v)]
    if kind == "bf16":
        caches = [tuple(torch.zeros(1, Smax, 1, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)) for _ in range(2)]
        out = flash_attn_with_kvcache(q, *caches[0], k=k, v=v, cache_seqlens=0, causal=causal)
        flash_attn_with_kvcache(near[0], *caches[1], k=near[1], v=near[2], cache_seqlens=0, causal=causal)
        assert torch.equal(caches[0][0][:, :S], near[1]) and torch.equal(caches[0][1][:, :S], near[2])
    else:
        dtype = torch.int8 if kind == "int8" else torch.float8_e4m3fn
        caches = [kvcache_q8(1, Smax, 1, dtype=dtype) for _ in range(2)]
        out = flash_attn_with_kvcache_q8(q, caches[0], k, v, 0, causal=causal)
        flash_attn_with_kvcache_q8(near[0], caches[1], near[1], near[2], 0, causal=causal)
    for a, b in zip(*caches):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    rows = torch.cat((torch.arange(0, S, 997), torch.tensor([1, 31, 32, S - 2, S - 1]))).to(DEV)
    score = near[0][0, rows, 0].double() @ near[1][0, :, 0].double().t() / math.sqrt(128)
    if causal:
        score = score.masked_fill(torch.arange(S, device=DEV)[None] > rows[:, None], -math.inf)
    p = torch.softmax(score, -1)
    want, mag = p @ near[2][0, :, 0].double(), p @ near[2][0, :, 0].double().abs()
    rel = 2 * 140 * U * 128 + (S + 100) * U + (2.0 ** -7 if S < 16128 else 0.0)
    assert ((out[0, rows, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + rel * mag).all()
