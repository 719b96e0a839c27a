"""GPU: the log probabilities' kernels by the sizes that choose them: gradients with non-temporal accesses
(logits and gradient of more than 192 MB together) with rows that begin at any element, rows in several
workgroups with targets that do not count, and rows of few finite logits.

Tolerances as in tests/test_gpu_logprob.py (u = 2^-24): ln S is off by (V / 512 + 32) u; a probability by
that, and by (3 |ln p| + 2 ln S + 8) u, relative; a gradient by that of its terms' magnitudes and by half
a step of its type."""
import math

import pytest
import torch

from oracle import logprob_oracle as oracle
from prefixlm import token_logprobs

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24


def _grad_tol(x, g, h, want):
    V = x.shape[1]
    logp = torch.log_softmax(x.double(), -1)
    ent = -(logp.exp() * logp).sum(-1, keepdim=True)
    span = math.log(V)                                     # ln S is at most that
    rel = (V / 512 + 32) * U + (3 * (logp.abs() + span) + 2 * span + 8) * U
    w = g.abs().double()[:, None] + (h.abs().double()[:, None] * (logp.abs() + ent + 2) if h is not None else 0.0)
    half = 2.0 ** -8 if x.dtype == torch.bfloat16 else 4 * U
    return 2 * logp.exp() * w * rel + want.abs() * half + 1e-37


@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("dtype,rows,V", [(torch.bfloat16, 1003, 50257), (torch.float32, 801, 32003), (torch.bfloat16, 1049, 48000),
                                          (torch.float32, 999, 25200)])
def test_large_gradients(dtype, rows, V, entropy):
    """Just above the threshold (the last two: a row fewer is below it)."""
    print(f"[case] {dtype} {rows} {V} {entropy}", flush=True)
    size = 2 if dtype == torch.bfloat16 else 4
    assert 2 * rows * V * size > 192 << 20
    gen = torch.Generator(device=DEV).manual_seed(V)
    x = (torch.randn(rows, V, generator=gen, device=DEV) * 2).to(dtype).requires_grad_()
    t = torch.randint(0, V, (rows,), generator=gen, device=DEV)
    t[1], t[2], t[rows - 1] = 0, V - 1, -100
    g, h = (torch.randn(rows, generator=gen, device=DEV) for _ in range(2))
    r = token_logprobs(x, t, entropy=entropy)
    heads, given = ((r.logprob, r.entropy), (g, h)) if entropy else ((r.logprob,), (g,))
    d, = torch.autograd.grad(heads, (x,), given)
    at = [0, 1, 2, 3, 7, 8, rows // 2, rows - 3, rows - 2, rows - 1]
    xs, ts = x.detach()[at].cpu(), t[at].cpu()
    gs, hs = g[at].cpu(), h[at].cpu() if entropy else None
    want = oracle.backward(xs, ts, gs, hs)
    gs[-1] = 0
    over = (d[at].double().cpu() - want).abs() - _grad_tol(xs, gs, hs, want)
    assert over.max().item() <= 0, over.max().item()
    # half of the rows, their edges included, against a call of their own, which is below the threshold
    half = x.detach()[rows // 2:].clone().requires_grad_()
    r2 = token_logprobs(half, t[rows // 2:], entropy=entropy)
    heads = (r2.logprob, r2.entropy) if entropy else (r2.logprob,)
    d2, = torch.autograd.grad(heads, (half,), tuple(y[rows // 2:] for y in given))
    assert torch.equal(d[rows // 2:], d2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V", [(5, 131072), (64, 131079), (1, 262145)])
def test_split_rows_with_targets_that_do_not_count(rows, V, dtype):
    print(f"[case] {rows} {V} {dtype}", flush=True)
    g = torch.Generator().manual_seed(rows)
    x = (torch.randn(rows, V, generator=g) * 2).to(dtype)
    t = torch.randint(0, V, (rows,), generator=g)
    t[0] = -100
    if rows > 1:
        t[1], t[2], t[3], t[4] = V, -1, V - 1, 0
    for entropy, top in ((False, 0), (True, 0), (False, 3), (True, 3)):
        xd = x.to(DEV).requires_grad_()
        r = token_logprobs(xd, t.to(DEV), entropy=entropy, top_k=top)
        lp, ent, _, tv, ti = oracle.forward(x, t, top)
        tol = (V / 512 + 32) * U + 4 * U * 64
        got = r.logprob.detach().double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(lp)) and got[0] == 0
        ok = ~torch.isnan(lp)
        assert ((got - lp).abs()[ok] <= tol).all()
        if entropy:
            assert ((r.entropy.detach().double().cpu() - ent).abs() <= 40 * tol).all()
        if top:
            assert torch.equal(r.top_ids.cpu(), ti) and ((r.top_logprobs.double().cpu() - tv).abs() <= tol).all()
        give = torch.randn(rows, generator=g)
        d, = torch.autograd.grad(r.logprob, (xd,), give.to(DEV))
        want = oracle.backward(x, t, give, None)
        assert torch.equal(torch.isnan(d.cpu()), torch.isnan(want))
        give[0] = 0
        over = ((d.double().cpu() - want).abs() - _grad_tol(x, give, None, want))[ok]
        assert over.max().item() <= 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [100, 9001, 65536, 131072])
def test_fewer_finite_logits_than_alternatives(V, dtype):
    """A grammar's mask: ten tokens can be. Behind them come the lowest ids, with -inf."""
    g = torch.Generator().manual_seed(V)
    allowed = torch.randperm(V, generator=g)[:10]
    x = torch.full((3, V), -math.inf)
    x[:, allowed] = torch.randn(3, 10, generator=g)
    x[2] = torch.randn(V, generator=g)
    x = x.to(dtype)
    t = allowed[:3].clone()
    for top in (10, 11, 20, 64):
        r = token_logprobs(x.to(DEV), t.to(DEV), entropy=True, top_k=top)
        lp, ent, _, tv, ti = oracle.forward(x, t, top)
        assert torch.equal(r.top_ids.cpu(), ti), top
        got, inf = r.top_logprobs.double().cpu(), torch.isinf(tv)
        assert torch.equal(torch.isinf(got), inf) and ((got - tv).abs()[~inf] <= (V / 512 + 32 + 200) * U).all()
        assert ((r.logprob.double().cpu() - lp).abs() <= (V / 512 + 32 + 200) * U).all()
        assert ((r.entropy.double().cpu() - ent).abs() <= 40 * (V / 512 + 32 + 200) * U).all()
