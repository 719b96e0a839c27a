"""GPU: prompts into an empty cache with softmax scales of every sign, given as a length of 0 (an int)
and as a tensor of lengths.

Tolerances (u = 2^-24, of the sum of p |v|): a score's 128 products, off by 140 u of their magnitudes,
change a weight twice; 500 keys 500 u, joins 100 u; the training forward, which calls with a positive
scale run, rounds the probabilities to bf16, 2^-8, and their exponents' argument with it; half a bf16
step of the output."""
import pytest
import torch

from oracle import kvcache8_oracle as oracle
from prefixlm import KVCacheQ8, flash_attn_with_kvcache, flash_attn_with_kvcache_q8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24


@pytest.mark.parametrize("as_int", [True, False])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.1, -1.5, 2.0 ** -40, 0.7])
@pytest.mark.parametrize("kind", ["bf16", "e4m3", "int8"])
def test_prompts_with_scales_of_every_sign(kind, scale, causal, as_int):
    B, S, H, Smax = 2, 150, 2, 192
    g = torch.Generator().manual_seed(11)
    q, k, v = (torch.randn(B, S, H, 128, generator=g).bfloat16() for _ in range(3))
    empty = oracle.empty(B, H, Smax, torch.int8 if kind == "int8" else torch.float8_e4m3fn)
    want, mag, _ = oracle.attend(q, empty, k, v, 0, causal, scale)
    lens = 0 if as_int else torch.zeros(B, dtype=torch.int32, device=DEV)
    d = [x.to(DEV) for x in (q, k, v)]
    if kind == "bf16":
        kc, vc = (torch.zeros(B, Smax, H, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        out = flash_attn_with_kvcache(d[0], kc, vc, k=d[1], v=d[2], cache_seqlens=lens, softmax_scale=scale, causal=causal)
    else:
        out = flash_attn_with_kvcache_q8(d[0], KVCacheQ8(*(x.to(DEV) for x in empty)), d[1], d[2], lens, scale, causal)
    A = q.double().abs().sum(-1, keepdim=True) * k.float().abs().max().item() * abs(scale)
    rel = 2 * 140 * U * A + 600 * U + (2.0 ** -7 if as_int and scale > 0 else 0.0)
    got = out.double().cpu()
    assert torch.isfinite(got).all()
    over = (got - want).abs() - (2.0 ** -8 * want.abs() + rel * mag)
    assert over.max().item() <= 0, (got - want).abs().max().item()
