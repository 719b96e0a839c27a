"""The stack's ``score`` with PyTorch's elementwise operations takes the targets that ``token_logprobs``
takes: int32 ones, ignored ones, and ones outside the vocabulary, which give NaN."""
import pytest
import torch
import torch.nn.functional as F

from oracle import logprob_oracle
from prefixlm.hrm_stack import HRMStack, HRMStackConfig


def _model():
    return HRMStack(HRMStackConfig(hidden_size=64, num_heads=2, vocab_size=50, max_seq_len=64)).init_weights(5)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("ignore", [-100, 3])
def test_targets_of_every_kind(dtype, ignore):
    model, T = _model(), 12
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, 50, (T,), generator=g)
    targets = torch.randint(0, 50, (T,), generator=g).to(dtype)
    targets[0], targets[1], targets[2], targets[3] = ignore, 50, -1, 49
    attn = lambda q, k, v, c, **_: v  # noqa: E731
    r = model.score(ids, targets, torch.arange(T), attn, {}, entropy=True, top_k=2, ignore_index=ignore)
    hidden = model(model.embed_tokens(ids), torch.arange(T), attn, {})
    logits = F.linear(hidden, model.head).detach()
    lp, ent, _, top, tid = logprob_oracle.forward(logits, targets, 2, ignore)
    assert torch.equal(torch.isnan(r.logprob.detach()), torch.isnan(lp)) and torch.isnan(lp).sum() == 2
    ok = ~torch.isnan(lp)
    # float32 sums over 50 logits of magnitude below 4: below 1e-5
    assert (r.logprob.detach().double()[ok] - lp[ok]).abs().max() <= 1e-5 and r.logprob[0] == 0
    assert (r.entropy.detach().double() - ent).abs().max() <= 1e-5 and torch.equal(r.top_ids, tid)
    # a target outside the vocabulary has a gradient of NaN, an ignored one none
    assert torch.isnan(torch.autograd.grad(r.logprob[1], (model.head,), retain_graph=True)[0]).any()
    targets[1:3] = 7
    r = model.score(ids, targets, torch.arange(T), attn, {}, ignore_index=ignore)
    head, = torch.autograd.grad(r.logprob.sum(), (model.head,))
    want = logprob_oracle.backward(logits, targets, torch.ones(T), None, ignore).t() @ hidden.detach().double()
    assert torch.isfinite(head).all() and (head.double() - want).abs().max() <= 1e-4
