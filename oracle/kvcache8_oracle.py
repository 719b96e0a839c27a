"""CPU/fp64 oracle for attention over an 8-bit KV cache -- TEST INFRASTRUCTURE.

Only tests may import this module; the product path never calls it.

``attend`` is the definition, sequence by sequence: the rows that query i sees are the complete
blocks' ``scale * code``, then the incomplete block's bf16 rows from the ring, then the call's new
rows; a float64 softmax over them; and the cache afterwards, its blocks rounded in float32 by the
stated formula (the codes and scales are exact quantities: equal or wrong). Queries, lengths and
masks are those of ``oracle.kvcache_oracle``, which pins this one where nothing is rounded
(tests/test_kvcache8_cpu.py).
"""
from __future__ import annotations

import math

import torch

__all__ = ["BLOCK", "RECENT", "code_max", "round_block", "empty", "rows_of", "attend"]

BLOCK, RECENT = 64, 128


def code_max(dtype):
    return 127.0 if dtype == torch.int8 else 448.0


def round_block(x, dtype):
    """(codes, scale) of one block [64, D] of bf16 rows, in float32."""
    x = x.float()
    inv = torch.tensor(1.0 / code_max(dtype), dtype=torch.float32)
    scale = torch.clamp_min(x.abs().max() * inv, torch.tensor(2.0 ** -126))
    y = x / scale
    if dtype == torch.int8:
        y = y.round()                       # 127 at most, unless the block is not finite
        y = torch.where(y.abs() <= 127, y, torch.zeros_like(y))
    return y.to(dtype), scale


def empty(B, H, Smax, dtype, D=128):
    return [torch.zeros(B, H, Smax, D, dtype=torch.uint8).view(dtype) for _ in range(2)] \
        + [torch.zeros(B, H, Smax // BLOCK) for _ in range(2)] \
        + [torch.zeros(B, H, RECENT, D, dtype=torch.bfloat16) for _ in range(2)]


def rows_of(cache, n, b, h, length):
    """float64 [length, D]: the rows that a call sees of keys (n = 0) or values (n = 1)."""
    codes, scale, recent = cache[n], cache[2 + n], cache[4 + n]
    full = length // BLOCK * BLOCK
    old = codes[b, h, :full].float().double() * scale[b, h, :full // BLOCK].double().repeat_interleave(BLOCK)[:, None]
    slots = torch.arange(full, length) % RECENT
    return torch.cat((old, recent[b, h, slots].double()))


def attend(q, cache, k=None, v=None, lens=0, causal=False, softmax_scale=None):
    """(out float64 [B, S, H, D], sum of p |v| of the same shape, the new cache); the inputs are not
    modified."""
    B, S, H, D = q.shape
    Smax = cache[0].shape[2]
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else softmax_scale
    lens = [lens] * B if isinstance(lens, int) else [min(max(int(x), 0), Smax) for x in lens.tolist()]
    new = [x.clone() for x in cache]
    out = torch.zeros(B, S, H, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for b, n in enumerate(lens):
        s_new = S if k is not None else 0
        end = min(Smax, n + s_new)
        for h in range(H):
            rows = [rows_of(cache, i, b, h, n) for i in range(2)]
            if k is not None:
                rows = [torch.cat((r, x[b, :end - n, h].double())) for r, x in zip(rows, (k, v))]
            for i in range(S):
                seen = min(end, n + s_new - S + i + 1) if causal else end
                if seen <= 0:
                    continue
                p = torch.softmax(rows[0][:seen] @ q[b, i, h].double() * scale, 0)
                out[b, i, h] = p @ rows[1][:seen]
                mag[b, i, h] = p @ rows[1][:seen].abs()
            if k is None:
                continue
            for c, x in enumerate((k, v)):
                given = x[b, :, h]
                row = lambda j: given[j - n] if j >= n else cache[4 + c][b, h, j % RECENT]  # noqa: B023, E731
                for blk in range(n // BLOCK, end // BLOCK):
                    whole = torch.stack([row(j) for j in range(blk * BLOCK, blk * BLOCK + BLOCK)])
                    new[c][b, h, blk * BLOCK:(blk + 1) * BLOCK], new[2 + c][b, h, blk] = round_block(whole, cache[c].dtype)
                for j in range(max(n, end // BLOCK * BLOCK - BLOCK), end):
                    new[4 + c][b, h, j % RECENT] = given[j - n]
    return out, mag, new
