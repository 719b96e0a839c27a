"""CPU/fp64 oracle for token log probabilities -- TEST INFRASTRUCTURE.

Only tests may import this module; the product path never calls it.

Restates, row by row and from the definitions, what ``token_logprobs`` gives for logits x and a
target t: ``x_t - lse`` with ``lse = ln sum_j e^x_j`` (the negative of the reference's cross entropy,
models/lm_head.py:52), the entropy ``-sum_j p_j ln p_j``, the k largest logits in order with the
lower index first among equal ones, and the closed-form gradient. Pinned by torch's own float64
``log_softmax``, its autograd and finite differences (tests/test_logprob_cpu.py).
"""
from __future__ import annotations

import torch

__all__ = ["forward", "backward"]


def forward(x, targets=None, top_k=0, ignore_index=-100):
    """(logprob, entropy, lse, top_logprobs, top_ids) in float64 of logits [rows, V]."""
    x = x.double()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    s = e.sum(-1)
    lse = m[:, 0] + torch.log(s)
    p = e / s[:, None]
    logp = (x - m) - torch.log(s)[:, None]
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    lp = None
    if targets is not None:
        lp = torch.zeros(x.shape[0], dtype=torch.float64)
        for i, t in enumerate(targets.tolist()):
            if t != ignore_index:
                lp[i] = logp[i, t] if 0 <= t < x.shape[1] else float("nan")
    top = ids = None
    if top_k:
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top_k]
        top = torch.gather(logp, 1, ids)
    return lp, entropy, lse, top, ids


def backward(x, targets, g, h, ignore_index=-100):
    """d x in float64 for the gradients g of the log probabilities and h of the entropies (None: 0)."""
    _, entropy, _, _, _ = forward(x, None)
    x = x.double()
    m = x.amax(-1, keepdim=True)
    logp = (x - m) - torch.exp(x - m).sum(-1, keepdim=True).log()
    p = logp.exp()
    d = torch.zeros_like(x)
    if g is not None:
        for i, t in enumerate(targets.tolist()):
            if t == ignore_index:
                continue
            d[i] = -g[i].double() * p[i]
            if 0 <= t < x.shape[1]:
                d[i, t] += g[i].double()
            else:
                d[i] = float("nan")
    if h is not None:
        d = d - h.double()[:, None] * torch.where(p > 0, p * (logp + entropy[:, None]), torch.zeros_like(p))
    return d
