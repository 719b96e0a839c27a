"""GPU: attention over pages with more rows than a launch of a wave for each could take, where no such launch is made.

Tolerance: as in tests/test_gpu_paged_holes.py."""
import math

import pytest
import torch

from prefixlm import PagedKVCache, flash_attn_with_paged_kvcache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24


def test_more_rows_than_a_wave_each():
    """2^26 rows over 40 keys: whole units, which no second launch joins."""
    S, H, ps, D, n = 1 << 22, 16, 64, 64, 40
    g = torch.Generator().manual_seed(1)
    kp, vp = (torch.randn(1, 2, H, ps, D, generator=g).bfloat16() for _ in range(2))
    cache = PagedKVCache(kp.to(DEV), vp.to(DEV), torch.ones(2, dtype=torch.int32, device=DEV), torch.tensor([[1]], dtype=torch.int32, device=DEV))
    room = torch.randn(8 * S + H * D, generator=g).bfloat16().to(DEV)
    q = room.as_strided((1, S, H, D), (room.numel() // 8 * 8, 8, D, 1))      # query i begins 8 i elements into it
    out = flash_attn_with_paged_kvcache(q, cache, cache_seqlens=n)
    at = torch.tensor([0, 1, 127, 128, 65535, 1 << 20, (1 << 21) + 77, S - 129, S - 1])
    rows, got = q[0, at.to(DEV)].double().cpu(), out[0, at.to(DEV)].double().cpu()
    for h in range(H):
        keys, values = kp[0, 1, h, :n].double(), vp[0, 1, h, :n].double()
        s = 1.0 / math.sqrt(D)
        p = torch.softmax(rows[:, h] @ keys.t() * s, -1)
        want, mag = p @ values, p @ values.abs()
        A = (rows[:, h].abs() @ keys.abs().t()).amax(-1, keepdim=True) * s
        tol = 2.0 ** -8 * want.abs() + (2 * 140 * U * A + (n + 100) * U) * mag + 1e-30
        assert ((got[:, h] - want).abs() - tol).max().item() <= 0, h
    # all others: equal queries have equal rows, wherever they lie
    room.copy_(room[:16].repeat(room.numel() // 16 + 1)[:room.numel()])
    out = flash_attn_with_paged_kvcache(q, cache, cache_seqlens=n)
    for a in out[0].split(1 << 19):
        assert torch.equal(a, out[0, :2].repeat(a.shape[0] // 2, 1, 1))
