"""GPU: prompts into an empty cache whose rows hold infinities, NaN or values whose scores pass fp32's
range before the softmax scale: a query has the result of the keys that it sees, whatever the rows
behind it hold.

Tolerances (u = 2^-24, of the sum of p |v|): the training forward rounds the probabilities to bf16,
2^-8, and their exponents' argument with it; a score's 128 products 2 * 140 u of their magnitudes; n keys
n u; half a bf16 step of the output."""
import math

import pytest
import torch

from oracle import kvcache8_oracle as oracle
from prefixlm import flash_attn_with_kvcache, flash_attn_with_kvcache_q8, kvcache_q8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24
KINDS = ["bf16", "e4m3", "int8"]


def _prompt(kind, q, k, v, causal):
    B, S, H, _ = q.shape
    Smax = (S + 63) // 64 * 64
    q, k, v = (x.to(DEV) for x in (q, k, v))
    if kind == "bf16":
        kc, vc = (torch.zeros(B, Smax, H, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        return flash_attn_with_kvcache(q, kc, vc, k=k, v=v, cache_seqlens=0, causal=causal).double().cpu()
    cache = kvcache_q8(B, Smax, H, dtype=torch.int8 if kind == "int8" else torch.float8_e4m3fn)
    return flash_attn_with_kvcache_q8(q, cache, k, v, 0, causal=causal).double().cpu()


def _want(q, k, v, causal):
    B, S, H, _ = q.shape
    want, mag, _ = oracle.attend(q, oracle.empty(B, H, (S + 63) // 64 * 64, torch.int8), k, v, 0, causal)
    return want, mag


def _check(got, want, mag, A, tag):
    nan, inf = torch.isnan(want), torch.isinf(want)
    assert torch.equal(torch.isnan(got), nan), (tag, (torch.isnan(got) != nan).nonzero()[:4].tolist())
    assert torch.equal(got[inf], want[inf]), tag
    ok = torch.isfinite(want)
    over = ((got - want).abs() - (2.0 ** -8 * want.abs() + (2 * 140 * U * A + (want.shape[1] + 100) * U + 2.0 ** -7) * mag))[ok]
    assert (over <= 0).all(), (tag, (got - want).abs()[ok].max().item())


def _data(B, S, H, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, S, H, 128, generator=g).bfloat16() for _ in range(3)]


def _A(q, k):
    return q.double().abs().sum(-1, keepdim=True) * k.float().nan_to_num(0, 0, 0).abs().max().item() / math.sqrt(128)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B,S,H", [(2, 40, 2), (2, 131, 3), (1, 300, 2), (8, 260, 20)])
@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_are_not_finite(kind, B, S, H, causal):
    """One sequence and head with a NaN value, one with an infinite one, one with a NaN key, one with an
    infinite key; 8 x 3 x 20 workgroups have one group of keys each, the others two."""
    print(f"[case] {kind} {B} {S} {H} {causal}", flush=True)
    q, k, v = _data(B, S, H, S)
    clean = _prompt(kind, q, k, v, causal)
    hit = [(0, 0), (0, 1), (B - 1, 0), (B - 1, 1)]
    rows = [S - 3, S // 2, S // 2 + 1, S - 7]
    if B == 1:
        hit = hit[:2]
    for n, ((b, h), j) in enumerate(zip(hit, rows)):
        if n == 0:
            v[b, j, h] = math.nan
        elif n == 1:
            v[b, j, h, 5], v[b, j, h, 6] = math.inf, -math.inf
        elif n == 2:
            k[b, j, h, 3] = math.nan
        else:
            k[b, j, h, 9] = math.inf
    got = _prompt(kind, q, k, v, causal)
    for b, h in hit:
        one = [x[b:b + 1, :, h:h + 1] for x in (q, k, v)]
        want, mag = _want(*one, causal)
        _check(got[b:b + 1, :, h:h + 1], want, mag.nan_to_num(0, 0, 0), _A(one[0], one[1]), (b, h))
        got[b, :, h] = clean[b, :, h]
    assert torch.equal(got, clean)                     # the other heads have their bits


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kind", KINDS)
def test_scores_past_the_range_before_the_scale(kind, causal):
    """Raw scores of 1.2e39 are finite once scaled: far above all others, far below, and for all keys."""
    B, S, H = 1, 140, 4
    q, k, v = _data(B, S, H, 7)
    q[..., 0] = 4.0
    k[:, 30, 0, 0] = 3e38
    k[:, 30, 1, 0] = -3e38
    q[:, :, 2], k[:, :, 2] = 0, 0
    q[:, :, 2, 0], k[:, :, 2, 0] = 4.0, -3e38
    got = _prompt(kind, q, k, v, causal)
    want, mag = _want(q, k, v, causal)
    assert torch.isfinite(want).all() and torch.isfinite(got).all()
    # scores of 1e38 differ by more than any rounding or are equal: the tolerance is of the other keys'
    small = k.clone()
    small[..., 0] = torch.where(small[..., 0].abs() > 1e37, torch.zeros_like(small[..., 0]), small[..., 0])
    _check(got, want, mag, _A(q, small), "overflow")


@pytest.mark.parametrize("kind", KINDS)
def test_queries_that_are_not_finite(kind):
    q, k, v = _data(2, 70, 2, 9)
    clean = _prompt(kind, q, k, v, True)
    q[0, 13, 0, 2], q[1, 69, 1, 100] = math.nan, math.inf
    got = _prompt(kind, q, k, v, True)
    assert not torch.isfinite(got[0, 13, 0]).any() and not torch.isfinite(got[1, 69, 1]).any()
    got[0, 13, 0], got[1, 69, 1] = clean[0, 13, 0], clean[1, 69, 1]
    assert torch.equal(got, clean)
