"""A key-value cache in pages, and the attention that reads it.

``flash_attn_with_paged_kvcache`` takes the place of ``flash_attn_with_kvcache`` in an engine whose
sequences have very different lengths, or share what they begin with (the reference's loop:
simple_inference_engine.py:105-112, models/layers.py:147-151, keeps max_seqlen rows for every
sequence). Same queries, new rows, lengths and masks; several query heads may share a key-value head. The
cache is a ``PagedKVCache``: a pool of pages for each layer and one table for all layers, which gives
each sequence its pages.

An engine's step, all on the device and without a wait, so that it may be captured into a graph::

    short = paged_kvcache_reserve(cache, lens, 1)       # pages of their own for the new rows
    for i, layer in enumerate(layers):
        ... flash_attn_with_paged_kvcache(q, cache, k, v, lens, causal=True, layer=i)
    lens += 1

``paged_kvcache_fork`` makes sequences copies of others by sharing their pages (samples of one prompt,
beams); the next ``reserve`` gives each a page of its own for its new rows, with what an incomplete
page holds copied. ``paged_kvcache_free`` gives pages up (a sequence that ended, rejected draft tokens),
``paged_kvcache_compact`` moves those in use to the pool's front, ``paged_kvcache_copy`` copies pages within
a pool or into another one.
"""
from __future__ import annotations

import ctypes
import math
import operator
from typing import NamedTuple, Optional, Union

import torch
from torch import Tensor

from . import _capi
from .kvcache import _check4
from .kvcache8 import _span
from .op import _native_calls, _ptr, _stream

__all__ = ["PagedKVCache", "paged_kvcache", "flash_attn_with_paged_kvcache", "paged_kvcache_reserve", "paged_kvcache_fork",
           "paged_kvcache_free", "paged_kvcache_compact", "paged_kvcache_copy", "paged_kvcache_attn"]

MAX_SEQUENCES = 8192


class PagedKVCache(NamedTuple):
    """The tensors of a cache in pages (``paged_kvcache`` makes an empty one). Row j of sequence b is row
    ``j % page_size`` of page ``page_table[b, j // page_size]``."""
    k_pages: Tensor      # bfloat16 [layers, num_pages, num_kv_heads, page_size, head_dim]
    v_pages: Tensor
    refs: Tensor         # int32 [num_pages]: entries of the table that hold the page; 0: free
    page_table: Tensor   # int32 [batch, columns]; no page: -1


def paged_kvcache(num_pages: int, page_size: int, batch: int, max_seqlen: int, num_kv_heads: int, head_dim: int = 128,
                  layers: int = 1, device="cuda") -> PagedKVCache:
    """An empty cache: ``num_pages`` pages of ``page_size`` rows (a power of two, 16 to 1024) for each layer, and
    a table for ``batch`` sequences of up to ``max_seqlen`` rows, which is rounded up to whole pages."""
    if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two from 16 to 1024 (got {page_size})")
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128 (got {head_dim})")
    if min(num_pages, batch, max_seqlen, num_kv_heads, layers) < 1:
        raise ValueError(f"num_pages={num_pages}, batch={batch}, max_seqlen={max_seqlen}, num_kv_heads={num_kv_heads} and "
                         f"layers={layers} must be >= 1")
    shape = (layers, num_pages, num_kv_heads, page_size, head_dim)
    return PagedKVCache(*(torch.zeros(shape, dtype=torch.bfloat16, device=device) for _ in range(2)),
                        torch.zeros(num_pages, dtype=torch.int32, device=device),
                        torch.full((batch, -(-max_seqlen // page_size)), -1, dtype=torch.int32, device=device))


def _check_pages(k_pages: Tensor, v_pages: Tensor) -> None:
    for name, x in (("k_pages", k_pages), ("v_pages", v_pages)):
        if x.dtype != torch.bfloat16 or x.dim() != 5 or x.device.type != "cuda" or not x.numel():
            raise ValueError(f"{name} must be a bf16 [layers, num_pages, num_kv_heads, page_size, head_dim] GPU tensor "
                             f"(got {x.dtype} {tuple(x.shape)} on {x.device})")
        if not x.is_contiguous() or x.data_ptr() % 16:
            raise ValueError(f"{name} must be contiguous and 16-byte aligned (got strides {x.stride()})")
    if k_pages.shape != v_pages.shape or k_pages.device != v_pages.device:
        raise ValueError(f"k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)} differ")
    page_size, head_dim = k_pages.shape[3:]
    if page_size < 16 or page_size > 1024 or page_size & (page_size - 1) or head_dim not in (64, 128):
        raise ValueError(f"page_size must be a power of two from 16 to 1024 and head_dim 64 or 128 (got {page_size}, {head_dim})")


def _check_table(refs: Tensor, page_table: Tensor, num_pages: Optional[int], dev, most: int = 0) -> None:
    if refs.dtype != torch.int32 or refs.dim() != 1 or not refs.is_contiguous() or refs.device != dev \
            or (num_pages is not None and refs.shape[0] != num_pages) or not refs.numel():
        raise ValueError(f"refs must be int32 [{'num_pages' if num_pages is None else num_pages}], contiguous, on {dev} "
                         f"(got {refs.dtype} {tuple(refs.shape)} on {refs.device})")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or not page_table.numel() or page_table.device != dev:
        raise ValueError(f"page_table must be int32 [batch, columns] on {dev} (got {page_table.dtype} {tuple(page_table.shape)} "
                         f"on {page_table.device})")
    N, M = page_table.shape
    if (M > 1 and page_table.stride(1) != 1) or (N > 1 and page_table.stride(0) < M):
        raise ValueError(f"page_table's rows must be contiguous and apart (got strides {page_table.stride()})")
    if most and N > most:
        raise ValueError(f"page_table holds {N} sequences, at most {most} here")


def _apart(tensors, others=()) -> None:
    """The cache's tensors share no memory with each other and the other operands."""
    at = sorted(map(_span, tensors))
    if any(a[1] > b[0] for a, b in zip(at, at[1:])):
        raise ValueError("the cache's tensors overlap")
    if any(a[0] < s[1] and s[0] < a[1] for s in map(_span, others) for a in at):
        raise ValueError("an operand overlaps the cache")


def _pool(k_pages: Optional[Tensor], v_pages: Optional[Tensor], refs: Tensor, page_table: Tensor, shape=None) -> _capi.PagePool:
    L, P, H, ps, D = k_pages.shape if shape is None else shape
    N, M = page_table.shape
    return _capi.PagePool(_ptr(k_pages), _ptr(v_pages), _ptr(refs), _ptr(page_table), page_table.stride(0) if N > 1 else M,
                          L, P, H, ps, D, N, M)


def _whole(x, name: str) -> int:
    try:
        return operator.index(x)
    except TypeError:
        raise ValueError(f"{name} must be a whole number or a tensor (got {x!r})") from None


def _rows(x: Union[int, Tensor, None], n: int, dev, name: str):
    """(int32 [n] on dev, or None; the constant in its place)."""
    if not isinstance(x, Tensor):
        return None, max(-1, min(_whole(x, name), 2**31 - 1))
    if x.dtype not in (torch.int32, torch.int64) or x.numel() != n or x.device != dev:
        raise ValueError(f"{name} must be an int or int32 [{n}] on {dev} (got {x.dtype} {tuple(x.shape)} on {x.device})")
    if x.dtype == torch.int64:   # outside int32 is outside every cache
        x = x.clamp(-2**31, 2**31 - 1).to(torch.int32)
    return x.reshape(-1).contiguous(), 0


def _given(x: Optional[Tensor], n: int, dev, name: str) -> Optional[Tensor]:
    return None if x is None else _rows(x, n, dev, name)[0]


# ---- attention ------------------------------------------------------------------------------
@torch.library.custom_op("prefixlm::paged_kvcache_attn", mutates_args=("k_pages", "v_pages"))
def paged_kvcache_attn(q: Tensor, k: Optional[Tensor], v: Optional[Tensor], k_pages: Tensor, v_pages: Tensor, refs: Tensor,
                       page_table: Tensor, cache_seqlens: Optional[Tensor], cache_seqlen: int, layer: int, causal: bool,
                       softmax_scale: float) -> Tensor:
    """out [B, S, Hq, D] bf16; the pages updated in place."""
    _check4(q, "q")
    _check_pages(k_pages, v_pages)
    dev = q.device
    B, S, Hq, D = q.shape
    L, P, Hkv, ps, _ = k_pages.shape
    if k_pages.device != dev:
        raise ValueError(f"q is on {dev}, the cache on {k_pages.device}")
    _check_table(refs, page_table, P, dev)
    if page_table.shape[0] != B or k_pages.shape[4] != D or Hq % Hkv or q.numel() == 0:
        raise ValueError(f"q must be [{page_table.shape[0]}, S, a multiple of {Hkv} heads, {k_pages.shape[4]}] (got {tuple(q.shape)})")
    cap = page_table.shape[1] * ps
    if not 0 <= layer < L:
        raise ValueError(f"layer = {layer} is outside [0, {L})")
    if (k is None) != (v is None):
        raise ValueError("k and v must be given together")
    if k is not None:
        k, v = (x.clone(memory_format=torch.contiguous_format) if x.data_ptr() % 16 else x for x in (k, v))
        for name, x in (("k", k), ("v", v)):
            _check4(x, name)
            if tuple(x.shape) != (B, S, Hkv, D) or x.device != dev:
                raise ValueError(f"{name} must be [{B}, {S}, {Hkv}, {D}] on {dev} (got {tuple(x.shape)} on {x.device})")
    lens = _given(cache_seqlens, B, dev, "cache_seqlens")
    _apart((k_pages, v_pages, refs, page_table), [x for x in (q, k, v, lens) if x is not None])
    if lens is None and not 0 <= cache_seqlen <= cap:
        raise ValueError(f"cache_seqlens = {cache_seqlen} is outside [0, {cap}]")
    lib = _capi.load()
    out = torch.empty((B, S, Hq, D), dtype=q.dtype, device=dev)
    n = lib.prefixlm_paged_workspace_size(B, S, Hq, Hkv, D, ps, page_table.shape[1])
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    z = (0, 0, 0)
    a = _capi.PagedArgs(
        _pool(k_pages, v_pages, refs, page_table), _ptr(q), _ptr(k), _ptr(v), _ptr(out), *q.stride()[:3],
        *(k.stride()[:3] if k is not None else z), *(v.stride()[:3] if v is not None else z), *out.stride()[:3],
        _ptr(lens), int(cache_seqlen), int(layer), S, Hq, 1 if causal else 0, float(softmax_scale), _ptr(ws), n)
    with torch.cuda.device(dev):
        _capi.check(lib.prefixlm_paged_fwd(ctypes.byref(a), _stream(dev)), "prefixlm_paged_fwd")
    return out


@paged_kvcache_attn.register_fake
def _paged_kvcache_attn_fake(q, k, v, k_pages, v_pages, refs, page_table, cache_seqlens, cache_seqlen, layer, causal,
                             softmax_scale):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


def flash_attn_with_paged_kvcache(q: Tensor, cache: PagedKVCache, k: Optional[Tensor] = None, v: Optional[Tensor] = None,
                                  cache_seqlens: Union[int, Tensor, None] = None, softmax_scale: Optional[float] = None,
                                  causal: bool = False, layer: int = 0) -> Tensor:
    """Attention of q [B, S, Hq, D] bf16 over one layer of a cache in pages, one table row for each of q's
    batch; Hq is a multiple of the cache's heads Hkv, and query head h reads key-value head
    ``h // (Hq // Hkv)``. k, v [B, S, Hkv, D] (or None: the cache only) are new rows behind the first
    ``cache_seqlens`` rows (an int in [0, columns * page_size], or int32 [B] on the GPU, where values outside count
    as the nearest of the two; None = 0). They are attended as given, and stored where the sequence holds the
    page alone (``paged_kvcache_reserve`` sees to it); rows past the table's end are dropped. All S rows count in
    every sequence: where sequences have fewer and are padded behind, pass ``causal``, with which no row sees those
    behind it; without it the padding is seen as keys, so only sequences with the same number of new rows go into one
    call. Cached rows without a page are not seen. ``causal``: query i sees keys j <= rows - S + i, as in
    ``flash_attn_with_kvcache``. A query that sees no key gives a row of 0. Forward only: the call has
    no gradient."""
    if cache_seqlens is None:
        cache_seqlens = 0
    native = _native_calls()
    if native is not None:
        out = native.paged(q, *cache, k, v, cache_seqlens, softmax_scale, causal, layer)
        if out is not None:
            return out
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(q.shape[-1])
    lens, n = (cache_seqlens, 0) if isinstance(cache_seqlens, Tensor) else (None, _whole(cache_seqlens, "cache_seqlens"))
    return paged_kvcache_attn(q, k, v, *cache, lens, n, int(layer), bool(causal), float(softmax_scale))


# ---- the pages --------------------------------------------------------------------------------
def _call(name: str, dev, pool: _capi.PagePool, workspace: bool = False, **args) -> None:
    lib = _capi.load()
    ws = None
    if workspace:
        n = lib.prefixlm_pages_workspace_size(ctypes.byref(pool))
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        args.update(workspace=_ptr(ws), workspace_bytes=n)
    a = _capi.PagesArgs(pool=pool, **args)
    with torch.cuda.device(dev):
        _capi.check(getattr(lib, name)(ctypes.byref(a), _stream(dev)), name)


@torch.library.custom_op("prefixlm::paged_kvcache_reserve", mutates_args=("k_pages", "v_pages", "refs", "page_table"))
def _reserve(k_pages: Tensor, v_pages: Tensor, refs: Tensor, page_table: Tensor, cache_seqlens: Optional[Tensor],
             cache_seqlen: int, new_rows: Optional[Tensor], new_row: int) -> Tensor:
    _check_pages(k_pages, v_pages)
    dev, N = k_pages.device, page_table.shape[0]
    _check_table(refs, page_table, k_pages.shape[1], dev, MAX_SEQUENCES)
    lens, new = _given(cache_seqlens, N, dev, "cache_seqlens"), _given(new_rows, N, dev, "new_rows")
    _apart((k_pages, v_pages, refs, page_table), [x for x in (lens, new) if x is not None])
    short = torch.empty(N, dtype=torch.int32, device=dev)
    _call("prefixlm_pages_reserve", dev, _pool(k_pages, v_pages, refs, page_table), True, rows=_ptr(lens), row_const=cache_seqlen,
          new_rows=_ptr(new), new_row_const=new_row, result=_ptr(short))
    return short


@_reserve.register_fake
def _reserve_fake(k_pages, v_pages, refs, page_table, cache_seqlens, cache_seqlen, new_rows, new_row):
    return page_table.new_empty(page_table.shape[0])


def paged_kvcache_reserve(cache: PagedKVCache, cache_seqlens: Union[int, Tensor, None], new_rows: Union[int, Tensor]) -> Tensor:
    """Gives each sequence pages of its own for rows ``cache_seqlens .. cache_seqlens + new_rows - 1`` (each an
    int, or int32 [batch] on the GPU; a sequence with no new rows gets none), as far as the table reaches. Columns of
    these rows without a page, or with one that others hold too, get the lowest free pages, in the order of
    sequences and columns; of a page whose holders all ask for it in this call the first keeps it. Where a
    shared page is left, its rows below ``cache_seqlens`` are copied, in every layer. Returns int32 [batch]:
    how many columns are left without a page of their own, 0 as long as pages last; new rows in these are not stored
    by ``flash_attn_with_paged_kvcache``. Rows below ``cache_seqlens`` that no page held, such as these, hold what their
    page held before once they are given one. At most 8192 sequences."""
    if cache_seqlens is None:
        cache_seqlens = 0
    native = _native_calls()
    if native is not None:
        short = native.pages_reserve(*cache, cache_seqlens, new_rows)
        if short is not None:
            return short
    lens, n = _rows(cache_seqlens, cache.page_table.shape[0], cache.page_table.device, "cache_seqlens")
    new, m = _rows(new_rows, cache.page_table.shape[0], cache.page_table.device, "new_rows")
    return _reserve(*cache, lens, n, new, m)


@torch.library.custom_op("prefixlm::paged_kvcache_fork", mutates_args=("refs", "page_table"))
def _fork(refs: Tensor, page_table: Tensor, parents: Tensor) -> None:
    dev = page_table.device
    if dev.type != "cuda":
        raise ValueError(f"the cache must be on a GPU (got {dev})")
    _check_table(refs, page_table, None, dev, MAX_SEQUENCES)
    src = _given(parents, page_table.shape[0], dev, "parents")
    _apart((refs, page_table), (src,))
    _call("prefixlm_pages_fork", dev, _pool(None, None, refs, page_table, (1, refs.shape[0], 1, 16, 64)), src=_ptr(src))


@_fork.register_fake
def _fork_fake(refs, page_table, parents):
    return None


def paged_kvcache_fork(cache: PagedKVCache, parents: Tensor) -> None:
    """Sequence b becomes a copy of sequence ``parents[b]`` (int32 [batch] on the GPU), all at once: it gives up
    its pages and holds its parent's. Entries that are b itself or outside [0, batch) leave their sequence as
    it is. No rows are copied: the lengths are the caller's to copy, and ``paged_kvcache_reserve`` gives
    each sequence a page of its own before it takes new rows. At most 8192 sequences."""
    if not isinstance(parents, Tensor):
        raise ValueError(f"parents must be int32 [{cache.page_table.shape[0]}] (got {type(parents).__name__})")
    native = _native_calls()
    if native is None or native.pages_fork(cache.refs, cache.page_table, parents) is None:
        _fork(cache.refs, cache.page_table, parents)


@torch.library.custom_op("prefixlm::paged_kvcache_free", mutates_args=("refs", "page_table"))
def _free(refs: Tensor, page_table: Tensor, page_size: int, keep_rows: Optional[Tensor], keep_row: int) -> None:
    dev = page_table.device
    if dev.type != "cuda":
        raise ValueError(f"the cache must be on a GPU (got {dev})")
    _check_table(refs, page_table, None, dev)
    keep = _given(keep_rows, page_table.shape[0], dev, "keep_rows")
    _apart((refs, page_table), () if keep is None else (keep,))
    _call("prefixlm_pages_free", dev, _pool(None, None, refs, page_table, (1, refs.shape[0], 1, page_size, 64)), rows=_ptr(keep),
          row_const=keep_row)


@_free.register_fake
def _free_fake(refs, page_table, page_size, keep_rows, keep_row):
    return None


def paged_kvcache_free(cache: PagedKVCache, keep_rows: Union[int, Tensor] = 0) -> None:
    """Each sequence keeps the pages of its first ``keep_rows`` rows (an int, or int32 [batch] on the GPU) and
    gives up the others: 0 for a sequence that ended, its length to give up what draft tokens took, any
    number from columns * page_size on for one that keeps everything. A page that no one holds any more is free."""
    page_size = cache.k_pages.shape[3]
    native = _native_calls()
    if native is not None and native.pages_free(cache.refs, cache.page_table, page_size, keep_rows) is not None:
        return
    keep, n = _rows(keep_rows, cache.page_table.shape[0], cache.page_table.device, "keep_rows")
    _free(cache.refs, cache.page_table, page_size, keep, n)


@torch.library.custom_op("prefixlm::paged_kvcache_compact", mutates_args=("k_pages", "v_pages", "refs", "page_table"))
def _compact(k_pages: Tensor, v_pages: Tensor, refs: Tensor, page_table: Tensor) -> Tensor:
    _check_pages(k_pages, v_pages)
    dev = k_pages.device
    _check_table(refs, page_table, k_pages.shape[1], dev)
    _apart((k_pages, v_pages, refs, page_table))
    used = torch.empty(1, dtype=torch.int32, device=dev)
    _call("prefixlm_pages_compact", dev, _pool(k_pages, v_pages, refs, page_table), True, result=_ptr(used))
    return used


@_compact.register_fake
def _compact_fake(k_pages, v_pages, refs, page_table):
    return page_table.new_empty(1)


def paged_kvcache_compact(cache: PagedKVCache) -> Tensor:
    """Moves the pages in use, U of them, to numbers below U, in every layer, and the table with them: the i-th used
    page from U on goes to the i-th free one below U. Returns U, int32 [1]: a pool of U pages holds it all
    (``paged_kvcache_copy``)."""
    native = _native_calls()
    used = native.pages_compact(*cache) if native is not None else None
    return _compact(*cache) if used is None else used


@torch.library.custom_op("prefixlm::paged_kvcache_copy", mutates_args=("k_pages", "v_pages"))
def _copy(k_pages: Tensor, v_pages: Tensor, k_source: Optional[Tensor], v_source: Optional[Tensor], src: Tensor,
          dst: Tensor) -> None:
    _check_pages(k_pages, v_pages)
    dev = k_pages.device
    pools = [k_pages, v_pages]
    if k_source is not None:
        _check_pages(k_source, v_source)
        pools += [k_source, v_source]
        if k_source.device != dev or any(k_source.shape[i] != k_pages.shape[i] for i in (0, 2, 3, 4)):
            raise ValueError(f"the pools {tuple(k_source.shape)} on {k_source.device} and {tuple(k_pages.shape)} on {dev} may differ "
                             "in their numbers of pages only")
    if src.dim() != 1 or src.shape != dst.shape:
        raise ValueError(f"src {tuple(src.shape)} and dst {tuple(dst.shape)} must be lists of the same length")
    n = src.numel()
    src, dst = _given(src, n, dev, "src"), _given(dst, n, dev, "dst")
    if not n:
        return
    _apart(pools, (src, dst))
    word = torch.empty((1, 1), dtype=torch.int32, device=dev)   # neither table nor refs are read
    pool = _pool(k_pages, v_pages, word, word)
    source = _pool(k_source, v_source, word, word) if k_source is not None else None
    _call("prefixlm_pages_copy", dev, pool, from_=ctypes.pointer(source) if source is not None else None, src=_ptr(src),
          dst=_ptr(dst), n=n)


@_copy.register_fake
def _copy_fake(k_pages, v_pages, k_source, v_source, src, dst):
    return None


def paged_kvcache_copy(cache: PagedKVCache, src: Tensor, dst: Tensor, source: Optional[PagedKVCache] = None) -> None:
    """Copies pages ``src[i]`` of ``source`` (None: of the cache itself) to pages ``dst[i]`` of the cache, in every
    layer; src and dst are int32 [n] on the GPU. Pairs with a page outside its pool are skipped. The pages of dst
    differ from each other, and within one pool from those of src: else what they hold afterwards is not
    defined. Tables and refs stay as they are."""
    native = _native_calls()
    if native is not None and native.pages_copy(*cache, *((None,) * 4 if source is None else source), src, dst) is not None:
        return
    _copy(cache.k_pages, cache.v_pages, *((source.k_pages, source.v_pages) if source is not None else (None, None)), src, dst)
