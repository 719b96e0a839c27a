"""GPU: attention over pages for 17 rows and more that share keys, where tiles, lengths and references can go wrong; operands
that lie in what a call writes.

Tolerances: those of tests/test_gpu_paged.py, where they are derived.
"""
import math

import pytest
import torch

from oracle import paged_oracle as oracle
from prefixlm import (PagedKVCache, _native, flash_attn_with_paged_kvcache, paged_kvcache_copy, paged_kvcache_fork, paged_kvcache_free,
                      paged_kvcache_reserve)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24


def _rows(g, *shape):
    return torch.randn(*shape, generator=g).bfloat16()


def _to(cache):
    return PagedKVCache(*(x.to(DEV) for x in cache))


def _check(q, cache, k, v, lens, causal, softmax_scale=None, at=None, k_dev=None, v_dev=None):
    """at: the sequences that are compared."""
    at = list(range(q.shape[0])) if at is None else at
    out = flash_attn_with_paged_kvcache(q.to(DEV), _to(cache), k.to(DEV) if k_dev is None else k_dev, v.to(DEV) if v_dev is None else v_dev,
                                        lens.to(DEV), softmax_scale, causal)
    want, mag, _ = oracle.attend(q[at], [*cache[:3], cache[3][at]], k[at], v[at], lens[at], causal, softmax_scale)
    s = 1.0 / math.sqrt(q.shape[-1]) if softmax_scale is None else abs(softmax_scale)
    A = q[at].double().abs().sum(-1, keepdim=True) * max(float(x.abs().max().float()) for x in (cache[0], k)) * s
    n = cache[3].shape[1] * cache[0].shape[3]
    over = (out[at].double().cpu() - want).abs() - (2.0 ** -8 * want.abs() + (2 * 140 * U * A + (n + 100 + 256) * U) * mag + 1e-30)
    assert over.max().item() <= 0, over.max().item()
    return out


@pytest.mark.parametrize("D,ps", [(128, 64), (64, 16), (64, 128), (128, 32)])
@pytest.mark.parametrize("B,H,S,G,most", [(1, 40, 450, 1, 200), (3, 9, 333, 4, 150), (16, 16, 40, 1, 600), (64, 8, 20, 1, 700),
                                          (65, 8, 20, 2, 400), (17, 4, 520, 1, 90)])
def test_a_workgroup_for_each_unit(B, H, S, G, most, D, ps):
    """Sequences of any lengths, some the same, none and one row among them, in grids that fill the chip once, less and more."""
    g = torch.Generator().manual_seed(B + S)
    M = -(-(most + S) // ps)
    lens = torch.randint(0, most, (B,), generator=g, dtype=torch.int32)
    lens[:: 5] = lens[0]
    lens[B // 2], lens[-1] = 0, 1 if B > 1 else most
    cache = oracle.dealt(1, B * M, H, ps, D, B, M, (lens + S).tolist(), g)
    q, k, v = _rows(g, B, S, H * G, D), _rows(g, B, S, H, D), _rows(g, B, S, H, D)
    # a few sequences and two heads of each in 64 bits; the others against calls of their own
    out = flash_attn_with_paged_kvcache(q.to(DEV), _to(cache), k.to(DEV), v.to(DEV), lens.to(DEV), causal=True)
    at = sorted({0, B // 2, B - 1})
    for h in (0, H - 1):
        heads = slice(h * G, h * G + G)
        sub = [x[:, :, h:h + 1].contiguous() for x in cache[:2]] + [cache[2], cache[3][at]]
        want, mag, _ = oracle.attend(q[at][:, :, heads], sub, k[at][:, :, h:h + 1], v[at][:, :, h:h + 1], lens[at], True)
        A = q[at][:, :, heads].double().abs().sum(-1, keepdim=True) * max(float(x.abs().max().float()) for x in (cache[0], k)) / math.sqrt(D)
        over = (out[at][:, :, heads].double().cpu() - want).abs() \
            - (2.0 ** -8 * want.abs() + (2 * 140 * U * A + (M * ps + 100 + 256) * U) * mag + 1e-30)
        assert over.max().item() <= 0, (h, over.max().item())
    dev = _to(cache)
    for b in range(B):
        one = dev._replace(page_table=dev.page_table[b:b + 1])
        got = flash_attn_with_paged_kvcache(q[b:b + 1].to(DEV), one, k[b:b + 1].to(DEV), v[b:b + 1].to(DEV), int(lens[b]), causal=True)
        # both are within their rounding and a little of one value
        assert ((got[0].float() - out[b].float()).abs() <= 2 * 2.0 ** -8 * out[b].float().abs() + 1e-2).all(), b


@pytest.mark.parametrize("stride", [(1 << 23) - 8, 1 << 23, 0, 64])
@pytest.mark.parametrize("S", [40, 70])
def test_strides_of_the_new_rows(S, stride):
    """Rows as far apart as 32 bits reach over a tile, further, all the same one, and over each other."""
    ps, D, M = 64, 128, 4
    g = torch.Generator().manual_seed(S)
    lens = torch.tensor([100], dtype=torch.int32)
    cache = oracle.dealt(1, 6, 1, ps, D, 1, M, [100 + S], g)
    q, k_dev, v_dev = _rows(g, 1, S, 1, D), None, None
    made = []
    for i in range(2):
        room = torch.empty((S - 1) * stride + D, dtype=torch.bfloat16, device=DEV)
        x = room.as_strided((1, S, 1, D), (room.numel() // 8 * 8, stride, D, 1))
        for j in range(S):
            x[0, j, 0].copy_(_rows(g, D))
        made.append(x)
    k_dev, v_dev = made
    _check(q, cache, k_dev.cpu(), v_dev.cpu(), lens, True, k_dev=k_dev, v_dev=v_dev)


@pytest.mark.parametrize("scale", [1.0, -1.0])
@pytest.mark.parametrize("step", [0.02, 0.125, 0.5, -0.25])
@pytest.mark.parametrize("S", [40, 150])
def test_scores_that_rise_from_key_to_key(S, step, scale):
    """What the weights are relative to follows the scores, up or down, slowly and fast."""
    ps, D, M = 32, 64, 12
    g = torch.Generator().manual_seed(S)
    lens = torch.tensor([200, 33], dtype=torch.int32)
    cache = oracle.dealt(1, 30, 1, ps, D, 2, M, (lens + S).tolist(), g)
    q, k, v = torch.zeros(2, S, 1, D).bfloat16(), torch.zeros(2, S, 1, D).bfloat16(), _rows(g, 2, S, 1, D)
    q[..., 0] = (torch.arange(S) % 7 / 4.0 - 0.5)[None, :, None] * scale
    cache[0].zero_()
    for b in range(2):
        for j in range(int(lens[b])):
            cache[0][0, cache[3][b, j // ps], 0, j % ps, 0] = j * step
        k[b, :, 0, 0] = (torch.arange(S) + int(lens[b])) * step
    _check(q, cache, k, v, lens, True, softmax_scale=scale)


@pytest.mark.parametrize("S", [20, 140])
def test_values_near_the_range_end(S):
    ps, D, M = 64, 128, 4
    g = torch.Generator().manual_seed(S)
    lens = torch.tensor([110], dtype=torch.int32)
    cache = oracle.dealt(1, 6, 1, ps, D, 1, M, [110 + S], g)
    q, k, v = _rows(g, 1, S, 1, D), _rows(g, 1, S, 1, D), torch.full((1, S, 1, D), 1.5e38).bfloat16()
    cache[1][:] = 1.5e38
    out = _check(q, cache, k, v, lens, True)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("path", ["native", "python"])
def test_operands_in_what_a_call_writes(path, monkeypatch):
    assert _native.calls() is not None
    if path == "python":
        monkeypatch.setattr(_native, "_module", None)
    g = torch.Generator().manual_seed(1)
    c = _to(oracle.dealt(1, 12, 2, 16, 64, 4, 3, [40, 20, 3, 0], g))
    row, counts, pages = c.page_table.view(-1)[:4], c.refs[:4], c.k_pages.view(-1)[:8].view(torch.int32)
    q = torch.zeros(4, 1, 2, 64, dtype=torch.bfloat16, device=DEV)
    ones = torch.ones(4, dtype=torch.int32, device=DEV)
    for call in (lambda: paged_kvcache_reserve(c, row, 1), lambda: paged_kvcache_reserve(c, 0, counts), lambda: paged_kvcache_fork(c, row),
                 lambda: paged_kvcache_free(c, counts), lambda: paged_kvcache_copy(c, pages, ones), lambda: paged_kvcache_copy(c, ones, pages),
                 lambda: flash_attn_with_paged_kvcache(q, c, q, q, pages), lambda: flash_attn_with_paged_kvcache(q, c, cache_seqlens=row)):
        before = [x.clone() for x in c]
        with pytest.raises(ValueError, match="overlap"):
            call()
        for x, y in zip(before, c):
            assert torch.equal(x, y)
