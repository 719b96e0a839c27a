"""CPU/fp64 oracle for the scaled embedding -- TEST INFRASTRUCTURE.

Only tests may import this module; the product path never calls it.

``scale * table[ids]`` (models/lm_head.py:34-43) and the table's gradient, token by token in
float64. Pinned by ``F.embedding`` and its autograd (tests/test_embedding_cpu.py).
"""
from __future__ import annotations

import torch

__all__ = ["forward", "backward"]


def forward(ids, table, scale):
    return table.double()[ids] * scale


def backward(ids, dy, num_rows, scale, padding_idx=-1):
    """(gradient, sum of the magnitudes that went into each of its elements), float64 [num_rows, D]."""
    dy = dy.double().reshape(-1, dy.shape[-1])
    grad = torch.zeros(num_rows, dy.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(grad)
    for i, v in enumerate(ids.reshape(-1).tolist()):
        if 0 <= v < num_rows and v != padding_idx:
            grad[v] += dy[i]
            mag[v] += dy[i].abs()
    return grad * scale, mag * abs(scale)
