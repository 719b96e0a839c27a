"""GPU: attention over pages multiplies the weights with their fp32 bits, however many rows share the keys: sums that
cancel to 2^-16 of their terms keep them.

Tolerance (u = 2^-24). An exponent is at most 14 + 1.75: its argument takes log2 e's rounding and the product's, 1.75 u each, and
its last one, half a step below 16, 8 u; times ln 2 that is 8 u of the weight, and the exponential itself 2 u. A weight's terms
times bf16 values are exact; nine of them are added up, each addition off by 2 u of at most half the sum of p |v|; the joins
2 u. That is 21 u of the sum of p |v|, and half a bf16 step of what is left. Two bf16 terms a weight, each rounded to
nearest, leave at least 60 u of the weights chosen here, with the opposite sign on the other side of the sum."""
import pytest
import torch

from oracle import paged_oracle as oracle
from prefixlm import PagedKVCache, flash_attn_with_paged_kvcache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24


def _scores():
    """(left, right): scores whose weights two bf16 terms miss by at least 60 u, from below and from above."""
    y = torch.arange(-1.2, -0.2, 2.0 ** -10, dtype=torch.float64).bfloat16().double().unique()
    w = torch.exp(y)
    hi = w.bfloat16().double()
    off = (w - hi - (w - hi).bfloat16().double()) / w / U
    return y[off >= 60], y[off <= -60]


# rows that share keys: one, up to 16, blocks of 64 and of 128; units whole and in pieces
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D,ps", [(128, 16), (128, 64), (64, 32), (64, 256)])
@pytest.mark.parametrize("S,G,B,H,cap", [(1, 1, 4, 4, 256), (1, 1, 4, 4, 4096), (4, 4, 4, 4, 256), (4, 4, 4, 4, 1024), (20, 1, 4, 4, 256),
                                         (8, 8, 4, 4, 1024), (12, 8, 4, 4, 256), (12, 8, 4, 4, 1024), (12, 8, 16, 16, 256)])
def test_weights_keep_their_bits(S, G, B, H, cap, D, ps, causal):
    """Keys with v = (1, -hi, -lo) and weights (p, r, r), where hi + lo is p / r to 2^-17; the others weigh 1 and are 0."""
    left, right = _scores()
    assert left.numel() >= 16 and right.numel() >= 16
    g = torch.Generator().manual_seed(S + G)
    a = left[torch.randint(0, left.numel(), (B, H), generator=g)]
    b = right[torch.randint(0, right.numel(), (B, H), generator=g)]
    ratio = torch.exp(a - b)
    hi = ratio.bfloat16()
    n = 7
    lens = torch.full((B,), n, dtype=torch.int32)
    cache = oracle.dealt(1, B * 2 + 3, H, ps, D, B, cap // ps, [n + S] * B, g)
    cache[0].zero_(), cache[1].zero_()
    page = cache[3][:, 0].long()
    keys, values = (torch.zeros(B, H, n, dtype=torch.bfloat16) for _ in range(2))
    keys[..., 1], keys[..., 2], keys[..., 5] = a.bfloat16(), b.bfloat16(), b.bfloat16()
    values[..., 1], values[..., 2], values[..., 5] = 1.0, -hi, -(ratio - hi.double()).bfloat16()
    cache[0][0, page, :, :n, 3] = keys
    cache[1][0, page, :, :n] = values[..., None].expand(B, H, n, D)
    q, k, v = torch.zeros(B, S, H * G, D).bfloat16(), torch.zeros(B, S, H, D).bfloat16(), torch.zeros(B, S, H, D).bfloat16()
    q[..., 3] = 8.0
    dev = PagedKVCache(*(x.to(DEV) for x in cache))
    out = flash_attn_with_paged_kvcache(q.to(DEV), dev, k.to(DEV), v.to(DEV), lens.to(DEV), 0.125, causal).double().cpu()
    few = [0, B - 1]
    want, mag, _ = oracle.attend(q[few], [*cache[:3], cache[3][few]], k[few], v[few], lens[few], causal, 0.125)
    assert (want.abs() <= 2.0 ** -16 * mag).all()
    over = (out[few] - want).abs() - (2.0 ** -8 * want.abs() + 21 * U * mag)
    assert over.max().item() <= 0, ((out[few] - want).abs() / mag).max().item() / U
