"""GPU: several queries over the 8-bit cache multiply the probabilities with their fp32 bits: sums that
cancel to 2^-17 of their terms keep them.

Tolerance (u = 2^-24): an exponent's argument below 6 has the scale's two roundings, the product's and the
difference's, 4 u * 6 relative to 1, so the weight 4 * 6 * ln 2 u < 17 u; the exponential itself 2 u;
products with bf16 rows of its terms are exact but for their sums, 9 adds of u; the sum of the weights,
its reciprocal and the last product 6 u: 34 u of the sum of p |v|, and half a bf16 step of the output."""
import math

import pytest
import torch

from oracle import kvcache8_oracle as oracle
from prefixlm import flash_attn_with_kvcache_q8, kvcache_q8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("S", [4, 40, 100])
def test_several_queries_keep_the_bits_of_the_probabilities(S, causal):
    """Three keys with v = (hi, -1, lo) and weights (1, p, 1): hi + lo is p to 2^-17, so the output is
    what is left of p beyond that. The other new rows are masked or have no weight."""
    B, H = 16, 8
    g = torch.Generator().manual_seed(S)
    y = -(torch.rand(B, H, generator=g) * 3.0).bfloat16()               # scores y / sqrt(128) * 8
    q, k, v = (torch.zeros(B, S, H, 128).bfloat16() for _ in range(3))
    q[..., 0] = 8.0
    q[..., 1] = 64.0
    k[:, 1, :, 0] = y
    k[:, 3:, :, 1] = -60.0                                               # e^-339
    p = torch.exp(y.double() * 8.0 / math.sqrt(128))
    hi = p.bfloat16()
    lo = (p - hi.double()).bfloat16()
    v[:, 0], v[:, 1], v[:, 2] = hi[..., None], -1.0, lo[..., None]
    cache = oracle.empty(B, H, 128, torch.int8)
    dev = kvcache_q8(B, 128, H, dtype=torch.int8)
    lens = torch.zeros(B, dtype=torch.int32)
    out = flash_attn_with_kvcache_q8(q.to(DEV), dev, k.to(DEV), v.to(DEV), lens.to(DEV), causal=causal).double().cpu()
    want, mag, _ = oracle.attend(q, cache, k, v, lens, causal)
    last = slice(2, S)                                                   # the queries that see all three
    assert (want[:, last].abs() <= 2.0 ** -16 * mag[:, last]).all()
    over = ((out - want).abs() - (2.0 ** -8 * want.abs() + 34 * U * mag))[:, last]
    assert over.max().item() <= 0, ((out - want).abs() / mag)[:, last].max().item() / U
