"""KV-cache attention over a cache held in 8 bits, with one scale for each 64 rows and head.

``flash_attn_with_kvcache_q8`` takes the place of ``flash_attn_with_kvcache`` in an engine that
wants half the cache's memory, and half the bytes of a decode step (the reference's loop:
simple_inference_engine.py:105-112, models/layers.py:147-151). Same queries, new rows, lengths and
masks; the cache is a ``KVCacheQ8``.

A row is attended in bf16 while its block of 64 is incomplete, and by the call that brings it.
When its block is complete the block is rounded once, straight from bf16: the scale is the block's
largest magnitude times the fp32 value of 1/448 (e4m3) or 1/127 (int8), at least 2^-126, and
``code = round(row / scale)``, to nearest, ties to even. So what the cache holds does not depend on how many rows each call
brought. The last 64 to 127 rows stay in bf16 as well: a caller may take rows back (rejected draft
tokens) by passing a smaller length. How far counts from the furthest length that the cache has had,
taken back since or not: to ``furthest // 64 * 64 - 64`` (64 rows at least). Below that the bf16 rows have
been overwritten, which the call cannot see; only a multiple of 64, 0 among them, needs none of them and
may be gone back to at any time. The furthest length then counts anew, and what lies below that
multiple is reached at multiples of 64 only.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional, Union

import torch
from torch import Tensor

from . import _capi
from .kvcache import _check4
from .op import _native_calls, _ptr, _stream

__all__ = ["KVCacheQ8", "kvcache_q8", "flash_attn_with_kvcache_q8", "kvcache_q8_attn"]

BLOCK = 64
RECENT = 128
_CODES = (torch.float8_e4m3fn, torch.int8)


class KVCacheQ8(NamedTuple):
    """The tensors of an 8-bit cache, each contiguous (``kvcache_q8`` makes an empty one). Row j of
    (batch row, head) is ``scale[j // 64] * codes[j]`` once its block is complete."""
    k_codes: Tensor     # float8_e4m3fn or int8 [B, H, Smax, 128]
    v_codes: Tensor
    k_scale: Tensor     # float32 [B, H, Smax / 64]
    v_scale: Tensor
    k_recent: Tensor    # bfloat16 [B, H, 128, 128]: row j in slot j % 128
    v_recent: Tensor


def kvcache_q8(batch: int, max_seqlen: int, num_heads: int, head_dim: int = 128,
               dtype: torch.dtype = torch.float8_e4m3fn, device="cuda") -> KVCacheQ8:
    """An empty cache for up to max_seqlen rows, which is rounded up to a multiple of 64."""
    if head_dim != 128:
        raise ValueError(f"head_dim must be 128 (got {head_dim})")
    if dtype not in _CODES:
        raise ValueError(f"dtype must be float8_e4m3fn or int8 (got {dtype})")
    if batch < 1 or max_seqlen < 1 or num_heads < 1:
        raise ValueError(f"batch={batch}, max_seqlen={max_seqlen} and num_heads={num_heads} must be >= 1")
    n = -(-max_seqlen // BLOCK)
    lead = (batch, num_heads)
    return KVCacheQ8(
        *(torch.zeros((*lead, n * BLOCK, head_dim), dtype=torch.uint8, device=device).view(dtype) for _ in range(2)),
        *(torch.zeros((*lead, n), dtype=torch.float32, device=device) for _ in range(2)),
        *(torch.zeros((*lead, RECENT, head_dim), dtype=torch.bfloat16, device=device) for _ in range(2)))


def _span(x: Tensor):
    """The addresses that x's elements lie in."""
    n = sum((n - 1) * s for n, s in zip(x.shape, x.stride())) + 1
    return x.data_ptr(), x.data_ptr() + n * x.element_size()


def _check_cache(c, B: int, H: int, D: int, dev, others) -> int:
    """Smax of a cache that fits q and shares no memory with it and the new rows."""
    codes = c[0]
    if codes.dtype not in _CODES or codes.dim() != 4:
        raise ValueError(f"k_codes must be float8_e4m3fn or int8 [B, H, Smax, 128] (got {codes.dtype} {tuple(codes.shape)})")
    Smax = codes.shape[2]
    if Smax < 1 or Smax % BLOCK:
        raise ValueError(f"the cache's rows must be a positive multiple of {BLOCK} (got {Smax})")
    want = [((B, H, Smax, D), codes.dtype)] * 2 + [((B, H, Smax // BLOCK), torch.float32)] * 2 \
        + [((B, H, RECENT, D), torch.bfloat16)] * 2
    at = []
    for name, x, (shape, dtype) in zip(KVCacheQ8._fields, c, want):
        if tuple(x.shape) != shape or x.dtype != dtype or x.device != dev:
            raise ValueError(f"{name} must be {dtype} {shape} on {dev} (got {x.dtype} {tuple(x.shape)} on {x.device})")
        if not x.is_contiguous() or x.data_ptr() % (4 if dtype == torch.float32 else 16):
            raise ValueError(f"{name} must be contiguous and 16-byte aligned (got strides {x.stride()})")
        at.append(_span(x))
    at.sort()
    if any(a[1] > b[0] for a, b in zip(at, at[1:])):
        raise ValueError("the cache's tensors overlap")
    # they are read while the cache is written
    if any(a[0] < s[1] and s[0] < a[1] for s in map(_span, others) for a in at):
        raise ValueError("q, k or v overlap the cache")
    return Smax


@torch.library.custom_op("prefixlm::kvcache_q8_attn", mutates_args=("k_codes", "v_codes", "k_scale", "v_scale", "k_recent",
                                                                   "v_recent"))
def kvcache_q8_attn(q: Tensor, k: Optional[Tensor], v: Optional[Tensor], k_codes: Tensor, v_codes: Tensor,
                    k_scale: Tensor, v_scale: Tensor, k_recent: Tensor, v_recent: Tensor,
                    cache_seqlens: Optional[Tensor], cache_seqlen: int, causal: bool, softmax_scale: float) -> Tensor:
    """out [B, S, H, D] bf16; the cache's tensors updated in place."""
    _check4(q, "q")
    B, S, H, D = q.shape
    if D != 128 or q.numel() == 0:
        raise ValueError(f"q must be [B, S, H, 128], none of them 0 (got {tuple(q.shape)})")
    dev = q.device
    cache = (k_codes, v_codes, k_scale, v_scale, k_recent, v_recent)
    if (k is None) != (v is None):
        raise ValueError("k and v must be given together")
    Smax = _check_cache(cache, B, H, D, dev, (q,) if k is None else (q, k, v))
    if k is not None:
        k, v = (x.clone(memory_format=torch.contiguous_format) if x.data_ptr() % 16 else x for x in (k, v))
        for name, x in (("k", k), ("v", v)):
            _check4(x, name)
            if tuple(x.shape) != (B, S, H, D) or x.device != dev:
                raise ValueError(f"{name} must be [{B}, {S}, {H}, {D}] on {dev} (got {tuple(x.shape)} on {x.device})")
    if cache_seqlens is not None:
        if cache_seqlens.dtype not in (torch.int32, torch.int64) or cache_seqlens.numel() != B:
            raise ValueError(f"cache_seqlens must hold {B} int32 (got {cache_seqlens.dtype} {tuple(cache_seqlens.shape)})")
        if cache_seqlens.dtype == torch.int64:   # outside int32 is outside the cache
            cache_seqlens = cache_seqlens.clamp(0, Smax)
        cache_seqlens = cache_seqlens.to(device=dev, dtype=torch.int32).contiguous()
    elif not 0 <= cache_seqlen <= Smax:
        raise ValueError(f"cache_seqlens = {cache_seqlen} is outside [0, {Smax}]")
    lib = _capi.load()
    out = torch.empty((B, S, H, D), dtype=q.dtype, device=dev)
    n = lib.prefixlm_kvcache8_workspace_size(B, S, H, Smax)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    z = (0, 0, 0)
    a = _capi.Kvcache8Args(
        _ptr(q), _ptr(k), _ptr(v), *(_ptr(x) for x in cache), _ptr(out), *q.stride()[:3],
        *(k.stride()[:3] if k is not None else z), *(v.stride()[:3] if v is not None else z), *out.stride()[:3],
        _ptr(cache_seqlens), int(cache_seqlen), B, S, H, D, Smax, int(k_codes.dtype == torch.int8), 1 if causal else 0,
        float(softmax_scale), _ptr(ws), n)
    with torch.cuda.device(dev):
        _capi.check(lib.prefixlm_kvcache8_fwd(ctypes.byref(a), _stream(dev)), "prefixlm_kvcache8_fwd")
    return out


@kvcache_q8_attn.register_fake
def _kvcache_q8_attn_fake(q, k, v, k_codes, v_codes, k_scale, v_scale, k_recent, v_recent, cache_seqlens, cache_seqlen,
                          causal, softmax_scale):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


def flash_attn_with_kvcache_q8(q: Tensor, cache: KVCacheQ8, k: Optional[Tensor] = None, v: Optional[Tensor] = None,
                               cache_seqlens: Union[int, Tensor, None] = None, softmax_scale: Optional[float] = None,
                               causal: bool = False) -> Tensor:
    """Attention of q [B, S, H, 128] bf16 over an 8-bit cache, which takes the new rows k, v
    [B, S, H, 128] (or None: the cache only) behind its first ``cache_seqlens`` rows (an int, or int32
    [B] on the GPU, where values outside [0, Smax] count as the nearest of the two; None = 0). Rows
    past the cache's end are dropped. A prompt into an empty cache (the int 0 or None) runs the training
    forward, which rounds the probabilities to bf16; with a tensor of zeros, as in every other call, they
    keep their fp32 bits. ``causal``: query i sees keys j <= rows - S + i, as in
    ``flash_attn_with_kvcache``. A query that sees no key gives a row of 0. Forward only: the call has
    no gradient."""
    if cache_seqlens is None:
        cache_seqlens = 0
    native = _native_calls()
    if native is not None:
        out = native.kvcache_q8(q, *cache, k, v, cache_seqlens, softmax_scale, causal)
        if out is not None:
            return out
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(q.shape[-1])
    lens, n = (None, cache_seqlens) if isinstance(cache_seqlens, int) else (cache_seqlens, 0)
    return kvcache_q8_attn(q, k, v, *cache, lens, n, bool(causal), float(softmax_scale))
