"""embedding without a GPU: the oracle against F.embedding and its autograd, refusals of the operator
and of the C entry points."""
import ctypes
import os

import pytest
import torch
import torch.nn.functional as F

from oracle import embedding_oracle as oracle
from prefixlm import _build, _capi, embedding


def test_oracle_matches_torch():
    g = torch.Generator().manual_seed(0)
    table = torch.randn(11, 8, generator=g, dtype=torch.float64, requires_grad=True)
    ids = torch.randint(0, 11, (3, 7), generator=g)
    dy = torch.randn(3, 7, 8, generator=g, dtype=torch.float64)
    y = F.embedding(ids, table, padding_idx=4) * 2.5
    torch.testing.assert_close(oracle.forward(ids, table.detach(), 2.5), y.detach())
    want, = torch.autograd.grad(y, (table,), dy)
    grad, mag = oracle.backward(ids, dy, 11, 2.5, padding_idx=4)
    torch.testing.assert_close(grad, want)
    assert (mag >= grad.abs() - 1e-12).all() and not grad[4].any()


def test_planted_mistake_is_caught():
    """A gradient that drops repeated ids differs from autograd's."""
    ids, dy = torch.tensor([1, 1, 2]), torch.ones(3, 8, dtype=torch.float64)
    grad, _ = oracle.backward(ids, dy, 4, 1.0)
    wrong = torch.zeros(4, 8, dtype=torch.float64)
    wrong[ids] = dy
    assert grad[1, 0] == 2 and not torch.equal(grad, wrong)


@pytest.mark.parametrize("ids,table,kw,needle", [
    (torch.zeros(2, dtype=torch.int64), torch.zeros(4, 8), {}, "GPU tensor"),
    (torch.zeros(2, dtype=torch.int64), torch.zeros(4, 8, dtype=torch.float16), {}, "bf16 or fp32"),
    (torch.zeros(2, dtype=torch.int64), torch.zeros(4, 8), {"padding_idx": 4}, "padding_idx"),
    (torch.zeros(2, dtype=torch.int64), torch.zeros(4, 8), {"padding_idx": -1}, "padding_idx"),
])
def test_refusals(ids, table, kw, needle):
    with pytest.raises(ValueError, match=needle):
        embedding(ids, table, **kw)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_build.LIB_PATH):
        _build.build()
    return _capi.load()


def _args(**kw):
    fake = 1 << 20   # never dereferenced: validation fails first
    a = dict(ids=fake, table=fake, y=fake, dy=fake, grad=fake, table_stride=64, y_stride=64, dy_stride=64, tokens=10,
             vocab=100, padding_id=-1, cols=64, scale=1.0)
    a.update(kw)
    return _capi.EmbeddingArgs(**a)


@pytest.mark.parametrize("kw,needle", [
    (dict(tokens=-1), "tokens"), (dict(vocab=0), "vocab"), (dict(vocab=1 << 27), "vocab"), (dict(cols=60), "cols"),
    (dict(cols=0), "cols"), (dict(ids=0), "ids"), (dict(table=0), "table"), (dict(y=(1 << 20) + 8), "y is null"),
    (dict(table_stride=56), "table"), (dict(y_stride=68), "row stride of y"), (dict(y_stride=0), "row stride of y"),
])
def test_forward_entry_point_rejects(lib, kw, needle):
    assert lib.prefixlm_embedding_fwd(ctypes.byref(_args(**kw)), None) == 1
    assert needle in _capi.last_error()


@pytest.mark.parametrize("kw,needle", [
    (dict(), "workspace"), (dict(grad=0), "grad"), (dict(dy=0), "dy"), (dict(ids=0), "ids"), (dict(dy_stride=63), "dy"),
    (dict(workspace=1 << 20, workspace_bytes=100), "workspace"), (dict(workspace=(1 << 20) + 4, workspace_bytes=1 << 30), "workspace"),
])
def test_backward_entry_point_rejects(lib, kw, needle):
    assert lib.prefixlm_embedding_bwd(ctypes.byref(_args(**kw)), None) == 1
    assert needle in _capi.last_error()


def test_null_args_and_empty_calls(lib):
    assert lib.prefixlm_embedding_fwd(None, None) == 1 and lib.prefixlm_embedding_bwd(None, None) == 1
    assert lib.prefixlm_embedding_fwd(ctypes.byref(_args(tokens=0, ids=0, y=0)), None) == 0
    assert lib.prefixlm_embedding_workspace_size(0, 100, 64) == 0
    assert lib.prefixlm_embedding_workspace_size(1, 100, 64) > 0
