"""GPU: attention over pages with more rows than a launch of a wave for each could take, where no such launch is made, and
forks of the widest table.

Tolerance: as in tests/test_gpu_paged_holes.py."""
import math

import pytest
import torch

from prefixlm import PagedKVCache, flash_attn_with_paged_kvcache, paged_kvcache_fork

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


@pytest.mark.parametrize("columns", [1 << 26, (1 << 26) - 7])
def test_fork_of_2_to_30_rows(columns):
    g = torch.Generator().manual_seed(2)
    table = torch.full((2, columns), -1, dtype=torch.int32, device=DEV)
    at = torch.cat((torch.randint(0, columns, (1000,), generator=g), torch.tensor([0, 1 << 25, columns - 17, columns - 1]))).to(DEV)
    table[1, at] = torch.arange(at.numel(), dtype=torch.int32, device=DEV)
    table[0, columns - 2] = at.numel()
    P = at.numel() + 1
    refs = torch.bincount(table.clamp_min(-1).add(1).view(-1), minlength=P + 1)[1:].int()
    pages = [torch.zeros(1, P, 1, 16, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    cache = PagedKVCache(*pages, refs.clone(), table.clone())
    paged_kvcache_fork(cache, torch.tensor([1, 1], dtype=torch.int32, device=DEV))
    assert torch.equal(cache.page_table[0], table[1]) and torch.equal(cache.page_table[1], table[1])
    refs = torch.bincount(table[1].add(1), minlength=P + 1)[1:].int()
    assert torch.equal(cache.refs, 2 * refs)
