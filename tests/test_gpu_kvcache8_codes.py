"""GPU: the codes of blocks that hold an infinity or NaN, which are ``round(row / scale)`` as all others."""
import math

import pytest
import torch

from oracle import kvcache8_oracle as oracle
from prefixlm import flash_attn_with_kvcache_q8, kvcache_q8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
CODES = [torch.float8_e4m3fn, torch.int8]


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("S", [1, 3, 64, 65, 128])
def test_codes_of_blocks_that_are_not_finite(S, dtype):
    """Blocks with one infinity of either sign, with a NaN, with both, of infinities alone, and beside
    them finite ones, completed by calls of 1 to 128 rows."""
    B, H, n = 1, 7, 128
    g = torch.Generator().manual_seed(S)
    k, v = (torch.randn(B, n, H, 128, generator=g).bfloat16() for _ in range(2))
    k[0, 10, 0, 3], k[0, 70, 1, 100] = math.inf, -math.inf
    k[0, 63, 2, 127], k[0, 64, 3, 0] = math.nan, math.nan
    k[0, 5, 4, 5], k[0, 6, 4, 6] = math.inf, math.nan
    k[0, :64, 5] = -math.inf
    k[0, 127, 6, 1], k[0, 100, 6, 2] = math.inf, -0.0
    v = torch.where(torch.isfinite(k.flip(2)), v, k.flip(2))
    dev, want = kvcache_q8(B, n, H, dtype=dtype), oracle.empty(B, H, n, dtype)
    for at in range(0, n, S):
        m = min(S, n - at)
        piece = [x[:, at:at + m] for x in (k, v)]
        lens = torch.full((B,), at, dtype=torch.int32)
        flash_attn_with_kvcache_q8(piece[0].to(DEV), dev, piece[0].to(DEV), piece[1].to(DEV), lens.to(DEV))
    for c, x in enumerate((k, v)):
        for h in range(H):
            for blk in range(2):
                codes, scale = oracle.round_block(x[0, blk * 64:blk * 64 + 64, h], dtype)
                want[c][0, h, blk * 64:blk * 64 + 64], want[2 + c][0, h, blk] = codes, scale
    for a, b in zip((dev.k_scale, dev.v_scale), want[2:4]):
        assert torch.equal(a.cpu().nan_to_num(-1.0), b.nan_to_num(-1.0))
    for name, a, b in zip(("keys", "values"), (dev.k_codes, dev.v_codes), want[:2]):
        a, b = a.cpu().float(), b.float()
        off = ~((a == b) | (torch.isnan(a) & torch.isnan(b)))
        assert not off.any(), (name, int(off.sum()), off.nonzero()[:4].tolist())
        assert torch.equal(torch.signbit(a) & (a == 0), torch.signbit(b) & (b == 0)), name
