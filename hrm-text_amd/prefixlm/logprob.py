"""Log probabilities of given tokens, with their entropy and the top alternatives.

The reference's head computes the cross entropy of its logits in fp32
(models/lm_head.py:52); scoring and sampling want the same row statistics with a little
more: the chosen token's log probability, the distribution's entropy, the few most likely
tokens. ``token_logprobs`` gives all of them from one pass over the logits, in bf16 or
fp32, with fp32 statistics and without a copy of the logits in fp32; its backward is one
pass that reads the logits and writes their gradient.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor

from . import _capi
from .op import _native_calls, _ptr, _stream

__all__ = ["TokenLogprobs", "token_logprobs", "token_logprobs_fwd", "token_logprobs_bwd"]

MAX_TOP_K = 64


class TokenLogprobs(NamedTuple):
    """What was asked for, float32 and int64 in the shape of the logits' rows; else None."""
    logprob: Optional[Tensor]        # [...]
    entropy: Optional[Tensor]        # [...]
    top_logprobs: Optional[Tensor]   # [..., k], largest first
    top_ids: Optional[Tensor]        # [..., k]


def _logit_rows(x: Tensor) -> Tensor:
    """x as a bf16 or fp32 [rows, V] GPU view with unit stride over V."""
    if x.dtype not in (torch.bfloat16, torch.float32) or x.device.type != "cuda" or x.dim() < 1:
        raise ValueError(f"logits must be a bf16 or fp32 GPU tensor [..., V] (got {x.dtype} {tuple(x.shape)} on {x.device})")
    if x.shape[-1] < 1:
        raise ValueError("logits have no vocabulary")
    x2 = x.reshape(-1, x.shape[-1]) if x.numel() else x.new_empty((0, x.shape[-1]))
    return x2 if x2.stride(-1) == 1 or x2.shape[1] == 1 else x2.contiguous()


def _target_rows(t: Tensor, x: Tensor) -> Tensor:
    if t.dtype not in (torch.int64, torch.int32) or tuple(t.shape) != tuple(x.shape[:-1]) or t.device != x.device:
        raise ValueError(f"targets must be int64 or int32 {tuple(x.shape[:-1])} on {x.device} "
                         f"(got {t.dtype} {tuple(t.shape)} on {t.device})")
    return t.reshape(-1).contiguous()


def _check_top_k(top_k: int, V: int) -> None:
    if not 0 <= top_k <= min(MAX_TOP_K, V):
        raise ValueError(f"top_k must be between 0 and min({MAX_TOP_K}, V = {V}) (got {top_k})")


@torch.library.custom_op("prefixlm::token_logprobs_fwd", mutates_args=())
def token_logprobs_fwd(logits: Tensor, targets: Optional[Tensor], entropy: bool, top_k: int,
                       ignore_index: int) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(logprob, entropy, stats, top_logprobs, top_ids), empty where not asked for; stats [..., 2]: the
    largest logit and the log of the sum of e^(logit - largest)."""
    x2 = _logit_rows(logits)
    rows, V = x2.shape
    _check_top_k(top_k, V)
    t = _target_rows(targets, logits) if targets is not None else None
    lib, dev, shape = _capi.load(), logits.device, logits.shape[:-1]
    f32 = dict(dtype=torch.float32, device=dev)
    lp = torch.empty(shape if t is not None else (0,), **f32)
    ent = torch.empty(shape if entropy else (0,), **f32)
    stats = torch.empty((*shape, 2), **f32)
    top = torch.empty((*shape, top_k) if top_k else (0,), **f32)
    ids = torch.empty((*shape, top_k) if top_k else (0,), dtype=torch.int64, device=dev)
    n = lib.prefixlm_logprob_workspace_size(rows, V, top_k)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    a = _capi.LogprobArgs(
        _ptr(x2), _ptr(t), _ptr(lp) if t is not None else None, _ptr(ent) if entropy else None, _ptr(stats),
        _ptr(top) if top_k else None, _ptr(ids) if top_k else None, None, None, None, x2.stride(0), 0, rows, V,
        ignore_index, top_k, int(logits.dtype == torch.float32), int(t is not None and t.dtype == torch.int32), _ptr(ws), n)
    with torch.cuda.device(dev):
        _capi.check(lib.prefixlm_logprob_fwd(ctypes.byref(a), _stream(dev)), "prefixlm_logprob_fwd")
    return lp, ent, stats, top, ids


@token_logprobs_fwd.register_fake
def _token_logprobs_fwd_fake(logits, targets, entropy, top_k, ignore_index):
    shape = logits.shape[:-1]
    f = lambda s: logits.new_empty(s, dtype=torch.float32)  # noqa: E731
    return (f(shape if targets is not None else (0,)), f(shape if entropy else (0,)), f((*shape, 2)),
            f((*shape, top_k) if top_k else (0,)),
            logits.new_empty((*shape, top_k) if top_k else (0,), dtype=torch.int64))


@torch.library.custom_op("prefixlm::token_logprobs_bwd", mutates_args=())
def token_logprobs_bwd(logits: Tensor, targets: Optional[Tensor], stats: Tensor, entropy: Tensor,
                       dlogprob: Optional[Tensor], dentropy: Optional[Tensor], ignore_index: int) -> Tensor:
    """The gradient of the logits, in their type, contiguous."""
    x2 = _logit_rows(logits)
    rows, V = x2.shape
    t = _target_rows(targets, logits) if targets is not None else None
    lib, dev = _capi.load(), logits.device

    def row_values(x, name, each=1):
        if x is None:
            return None
        if x.dtype != torch.float32 or x.numel() != rows * each or x.device != dev:
            raise ValueError(f"{name} must be float32 [{rows * each}] on {dev} (got {x.dtype} {tuple(x.shape)} on {x.device})")
        return x.reshape(-1).contiguous()

    g, h = row_values(dlogprob, "dlogprob") if t is not None else None, row_values(dentropy, "dentropy")
    stats = row_values(stats, "stats", 2)
    ent = row_values(entropy, "entropy") if h is not None else None
    dx = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    a = _capi.LogprobArgs(_ptr(x2), _ptr(t), None, _ptr(ent), _ptr(stats), None, None, _ptr(g), _ptr(h), _ptr(dx),
                          x2.stride(0), V, rows, V, ignore_index, 0, int(logits.dtype == torch.float32),
                          int(t is not None and t.dtype == torch.int32), None, 0)
    with torch.cuda.device(dev):
        _capi.check(lib.prefixlm_logprob_bwd(ctypes.byref(a), _stream(dev)), "prefixlm_logprob_bwd")
    return dx


@token_logprobs_bwd.register_fake
def _token_logprobs_bwd_fake(logits, targets, stats, entropy, dlogprob, dentropy, ignore_index):
    return logits.new_empty(logits.shape)


class TokenLogprobsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, entropy, top_k, ignore_index):
        lp, ent, stats, top, ids = token_logprobs_fwd(logits, targets, entropy, top_k, ignore_index)
        ctx.save_for_backward(logits, targets, stats, ent)
        ctx.ignore_index, ctx.with_entropy = ignore_index, entropy
        ctx.mark_non_differentiable(top, ids, *(() if targets is not None else (lp,)), *(() if entropy else (ent,)))
        ctx.set_materialize_grads(False)
        return lp, ent, top, ids

    @staticmethod
    def backward(ctx, g, h, *_):
        logits, targets, stats, ent = ctx.saved_tensors
        if g is None and h is None:
            return None, None, None, None, None
        return token_logprobs_bwd(logits, targets, stats, ent, g, h if ctx.with_entropy else None,
                                  ctx.ignore_index), None, None, None, None


def token_logprobs(logits: Tensor, targets: Optional[Tensor] = None, *, entropy: bool = False, top_k: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Row statistics of log_softmax(logits, -1), fp32, from one pass over bf16 or fp32 logits [..., V].

    ``targets`` (int64 or int32 [...]): ``logprob`` is their log probability, 0 where the target is
    ``ignore_index`` and NaN where it is any other index outside the vocabulary (its gradient too).
    ``entropy``: the distribution's, in nats. ``top_k`` (to 64): the k most likely tokens' log
    probabilities and ids, largest first, of equal ones the lower id first. ``logprob`` and
    ``entropy`` carry gradients, the alternatives do not. The mean cross entropy is
    ``-r.logprob.sum() / (targets != ignore_index).sum()``."""
    entropy, top_k, ignore_index = bool(entropy), int(top_k), int(ignore_index)
    if targets is None and not entropy and not top_k:
        raise ValueError("token_logprobs: neither targets, entropy nor top_k are asked for")
    native = _native_calls()
    out = native.token_logprobs(logits, targets, entropy, top_k, ignore_index) if native is not None else None
    lp, ent, top, ids = out if out is not None else TokenLogprobsFunction.apply(logits, targets, entropy, top_k,
                                                                              ignore_index)
    return TokenLogprobs(lp if targets is not None else None, ent if entropy else None, top if top_k else None,
                         ids if top_k else None)
