"""Scaled embedding lookup, with its gradient by sorted tokens.

The reference's head looks its tokens up in a table and multiplies the rows by a scale
(models/lm_head.py:34-43). ``embedding`` does both in one pass, from a bf16 or fp32 table
into bf16 or fp32 rows with one rounding. The backward sorts the tokens by id and adds each
id's rows in fp32, chunk by chunk of the sorted tokens, so that the gradient is bitwise the same
every time, and writes the whole table's gradient, zero rows included.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor

from . import _capi
from .op import _native_calls, _ptr, _stream

__all__ = ["embedding", "embedding_fwd", "embedding_bwd"]

_TYPES = (torch.bfloat16, torch.float32)


def _check_ids(ids: Tensor, dev) -> Tensor:
    if ids.dtype not in (torch.int64, torch.int32) or ids.device != dev:
        raise ValueError(f"ids must be int64 or int32 on {dev} (got {ids.dtype} on {ids.device})")
    return ids.reshape(-1).contiguous()


def _check_table(table_dtype, shape, device, dtype) -> None:
    if table_dtype not in _TYPES or len(shape) != 2 or device.type != "cuda":
        raise ValueError(f"table must be a bf16 or fp32 [V, D] GPU tensor (got {table_dtype} {tuple(shape)} on {device})")
    if shape[1] % 8 or shape[1] == 0 or not 1 <= shape[0] < 1 << 27:
        raise ValueError(f"table [V, D] = {tuple(shape)}: D must be a positive multiple of 8 and V in [1, 2^27)")
    if dtype not in _TYPES:
        raise ValueError(f"dtype must be bfloat16 or float32 (got {dtype})")


def _rows16(x: Tensor) -> Tensor:
    """x with unit column stride and 16-byte rows."""
    ok = x.stride(-1) == 1 and x.stride(0) * x.element_size() % 16 == 0 and x.data_ptr() % 16 == 0 \
        and (x.stride(0) >= x.shape[1] or x.stride(0) == 0)
    return x if ok else x.clone(memory_format=torch.contiguous_format)


@torch.library.custom_op("prefixlm::embedding_fwd", mutates_args=())
def embedding_fwd(ids: Tensor, table: Tensor, scale: float, dtype: torch.dtype) -> Tensor:
    """scale * table[ids], [..., D] in dtype."""
    _check_table(table.dtype, table.shape, table.device, dtype)
    dev = table.device
    flat, t2 = _check_ids(ids, dev), _rows16(table)
    V, D = table.shape
    y = torch.empty((*ids.shape, D), dtype=dtype, device=dev)
    a = _capi.EmbeddingArgs(_ptr(flat), _ptr(t2), _ptr(y), None, None, t2.stride(0), D, 0, flat.numel(), V, -1, D,
                            int(table.dtype == torch.float32), int(dtype == torch.float32),
                            int(ids.dtype == torch.int32), scale, None, 0)
    with torch.cuda.device(dev):
        _capi.check(_capi.load().prefixlm_embedding_fwd(ctypes.byref(a), _stream(dev)), "prefixlm_embedding_fwd")
    return y


@embedding_fwd.register_fake
def _embedding_fwd_fake(ids, table, scale, dtype):
    return table.new_empty((*ids.shape, table.shape[1]), dtype=dtype)


@torch.library.custom_op("prefixlm::embedding_bwd", mutates_args=())
def embedding_bwd(ids: Tensor, dy: Tensor, num_rows: int, scale: float, dtype: torch.dtype, padding_idx: int) -> Tensor:
    """The table's gradient [num_rows, D] in dtype; padding_idx < 0: none."""
    dev, D = dy.device, dy.shape[-1]
    _check_table(dtype, (num_rows, D), dev, dy.dtype)
    if tuple(dy.shape[:-1]) != tuple(ids.shape):
        raise ValueError(f"ids {tuple(ids.shape)} and dy {tuple(dy.shape)} do not match")
    flat = _check_ids(ids, dev)
    d2 = _rows16(dy.reshape(-1, D) if dy.numel() else dy.new_empty((0, D)))
    lib, T = _capi.load(), flat.numel()
    grad = torch.empty((num_rows, D), dtype=dtype, device=dev)
    n = lib.prefixlm_embedding_workspace_size(T, num_rows, D)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    a = _capi.EmbeddingArgs(_ptr(flat), None, None, _ptr(d2), _ptr(grad), 0, 0, d2.stride(0), T, num_rows, padding_idx, D,
                            int(dtype == torch.float32), int(dy.dtype == torch.float32),
                            int(ids.dtype == torch.int32), scale, _ptr(ws), n)
    with torch.cuda.device(dev):
        _capi.check(lib.prefixlm_embedding_bwd(ctypes.byref(a), _stream(dev)), "prefixlm_embedding_bwd")
    return grad


@embedding_bwd.register_fake
def _embedding_bwd_fake(ids, dy, num_rows, scale, dtype, padding_idx):
    return dy.new_empty((num_rows, dy.shape[-1]), dtype=dtype)


class EmbeddingFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, dtype, padding_idx):
        ctx.save_for_backward(ids)
        ctx.args = (table.shape[0], scale, table.dtype, padding_idx)
        return embedding_fwd(ids, table, scale, dtype)

    @staticmethod
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        return None, embedding_bwd(ids, dy, *ctx.args), None, None, None


def embedding(ids: Tensor, table: Tensor, scale: float = 1.0, *, dtype: Optional[torch.dtype] = None,
              padding_idx: Optional[int] = None) -> Tensor:
    """``scale * table[ids]`` [..., D] for ids [...] (int64 or int32) and a bf16 or fp32 table [V, D].

    ``dtype`` (bf16 or fp32, default the table's) is the rows' type; the product is rounded once.
    An id outside the table gives a row of NaN and no gradient. ``padding_idx``: this id's rows add
    nothing to the gradient. The table's gradient is dense, in its type. It is added in fp32: the
    tokens are sorted by id, those of one id in their order, and each 16 or 32 sorted ones are added one
    after another, then their sums in order. The same call gives the same bits; other ids' tokens move
    an id's place among the sorted ones, and with it its last bits."""
    scale, dtype = float(scale), table.dtype if dtype is None else dtype
    if padding_idx is not None and not 0 <= padding_idx < table.shape[0]:
        raise ValueError(f"padding_idx must be in [0, {table.shape[0]}) (got {padding_idx})")
    padding = -1 if padding_idx is None else int(padding_idx)
    native = _native_calls()
    y = native.embedding(ids, table, scale, dtype == torch.float32 if dtype in _TYPES else None, padding) \
        if native is not None else None
    return EmbeddingFunction.apply(ids, table, scale, dtype, padding) if y is None else y
