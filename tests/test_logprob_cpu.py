"""token_logprobs without a GPU: the oracle against torch's float64 log_softmax, its autograd and
finite differences; refusals of the operator and of the C entry points."""
import ctypes
import os

import pytest
import torch

from oracle import logprob_oracle as oracle
from prefixlm import _build, _capi, token_logprobs


def _x(rows=5, V=23, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rows, V, generator=g, dtype=torch.float64) * 2, torch.randint(0, V, (rows,), generator=g)


def test_oracle_matches_log_softmax_and_autograd():
    x, t = _x()
    t[2] = -100
    x[3, 4] = -float("inf")
    x.requires_grad_()
    logp = torch.log_softmax(x, -1)
    want = torch.where(t == -100, 0.0, logp.gather(1, t.clamp_min(0)[:, None])[:, 0])
    ent = torch.distributions.Categorical(logits=x).entropy()
    lp, e, lse, top, ids = oracle.forward(x.detach(), t, 4)
    torch.testing.assert_close(lp, want.detach(), rtol=1e-13, atol=1e-13)
    torch.testing.assert_close(e, ent.detach(), rtol=1e-13, atol=1e-13)
    torch.testing.assert_close(lse, torch.logsumexp(x, -1).detach())
    assert torch.equal(ids, torch.topk(x, 4).indices)
    torch.testing.assert_close(top, torch.topk(logp, 4).values.detach())
    g, h = torch.randn(5, dtype=torch.float64), torch.randn(5, dtype=torch.float64)
    d, = torch.autograd.grad((want, ent), (x,), (g, torch.where(torch.arange(5) == 3, 0.0, h)))
    got = oracle.backward(x.detach(), t, g, torch.where(torch.arange(5) == 3, 0.0, h))
    torch.testing.assert_close(got, torch.nan_to_num(d), rtol=1e-12, atol=1e-13)


def test_oracle_gradient_matches_differences():
    x, t = _x(2, 7, 1)
    g, h = torch.tensor([0.7, -1.3], dtype=torch.float64), torch.tensor([-0.4, 0.9], dtype=torch.float64)

    def f(y):
        lp, e, _, _, _ = oracle.forward(y, t)
        return (g * lp + h * e).sum()

    d = oracle.backward(x, t, g, h)
    for i in range(2):
        for j in range(7):
            up, down = x.clone(), x.clone()
            up[i, j] += 1e-6
            down[i, j] -= 1e-6
            assert abs((f(up) - f(down)) / 2e-6 - d[i, j]) < 1e-8


def test_oracle_orders_ties_by_index():
    x = torch.tensor([[1.0, 3.0, 3.0, -0.0, 0.0, 3.0]])
    assert oracle.forward(x, None, 5)[4].tolist() == [[1, 2, 5, 0, 3]]


def test_planted_mistake_is_caught():
    """The gradient without the entropy's constant fails the difference check."""
    x, t = _x(1, 5, 2)
    h = torch.ones(1, dtype=torch.float64)
    logp = torch.log_softmax(x, -1)
    wrong = -(logp.exp() * logp)
    up, down = x.clone(), x.clone()
    up[0, 0] += 1e-6
    down[0, 0] -= 1e-6
    diff = (oracle.forward(up)[1] - oracle.forward(down)[1]) / 2e-6
    assert abs(diff[0] - oracle.backward(x, t, None, h)[0, 0]) < 1e-8
    assert abs(diff[0] - wrong[0, 0]) > 1e-3


@pytest.mark.parametrize("logits,kw,needle", [
    (torch.zeros(2, 8), {"top_k": 1}, "GPU tensor"),
    (torch.zeros(2, 8, dtype=torch.float16), {"entropy": True}, "bf16 or fp32"),
    (torch.zeros(2, 8), {}, "neither"),
])
def test_refusals(logits, kw, needle):
    with pytest.raises(ValueError, match=needle):
        token_logprobs(logits, **kw)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_build.LIB_PATH):
        _build.build()
    return _capi.load()


def _args(**kw):
    fake = 1 << 20   # never dereferenced: validation fails first
    a = dict(x=fake, targets=fake, logprob=fake, stats=fake, x_stride=1000, dx_stride=1000, rows=300, vocab=1000,
             ignore_index=-100, dx=fake)
    a.update(kw)
    return _capi.LogprobArgs(**a)


@pytest.mark.parametrize("kw,needle", [
    (dict(vocab=0), "vocab"), (dict(rows=-1), "rows"), (dict(x=0), "x is null"), (dict(x=(1 << 20) + 1), "x is null"),
    (dict(x=(1 << 20) + 2, x_fp32=1), "aligned"), (dict(x_stride=-1), "x_stride"), (dict(stats=0), "stats"),
    (dict(targets=0), "targets"), (dict(logprob=0), "logprob"), (dict(top_k=65), "top_k"),
    (dict(top_k=-1), "top_k"), (dict(top_k=3), "top_logprobs"), (dict(rows=4, vocab=200000), "workspace"),
])
def test_forward_entry_point_rejects(lib, kw, needle):
    assert lib.prefixlm_logprob_fwd(ctypes.byref(_args(**kw)), None) == 1
    assert needle in _capi.last_error()


@pytest.mark.parametrize("kw,needle", [
    (dict(dx=0), "dx"), (dict(dx_stride=999), "dx_stride"), (dict(dlogprob=1 << 20, targets=0, logprob=0), "targets"),
    (dict(dentropy=1 << 20), "entropy"), (dict(stats=0), "stats"),
])
def test_backward_entry_point_rejects(lib, kw, needle):
    assert lib.prefixlm_logprob_bwd(ctypes.byref(_args(**kw)), None) == 1
    assert needle in _capi.last_error()


def test_null_args_and_empty_calls(lib):
    assert lib.prefixlm_logprob_fwd(None, None) == 1 and lib.prefixlm_logprob_bwd(None, None) == 1
    assert lib.prefixlm_logprob_fwd(ctypes.byref(_args(rows=0, x=0)), None) == 0
    assert lib.prefixlm_logprob_workspace_size(300, 1000, 5) == 0     # one workgroup a row
    assert lib.prefixlm_logprob_workspace_size(1, 100000, 5) > 0
    assert lib.prefixlm_logprob_workspace_size(0, 100, 0) == 0
