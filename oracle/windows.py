"""Oracle of attention with a window and sinks, and of rotary positions with several axes.

TEST INFRASTRUCTURE ONLY -- nothing in the product imports this module.

The operators' definitions in 64 bits on CPU tensors, by loops over requests and rows.  Pinned by
(tests/test_oracle_windows.py): the causal oracle where the window holds everything, a dense masked softmax, hand-worked
masks, and rotations in the complex plane.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch
from torch import Tensor


def visible(pos: int, length: int, window: int, sinks: int) -> List[int]:
    """The tokens that a row at position ``pos`` of a request of ``length`` tokens sees."""
    return [k for k in range(min(pos + 1, length)) if k > pos - window or k < sinks]


def window_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, cu: Sequence[int], lens: Sequence[int], table: Tensor,
                     window: int, sinks: int, scale: float, k_scales: Optional[Tensor] = None,
                     v_scales: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """(result, sum of probability times |value|, sum of |value|), fp64 ``[T, Hq, d]``; rows ``cu[r] : cu[r + 1]`` are the
    last tokens of request r.  ``k_cache`` / ``v_cache`` hold values (of an fp8 cache: the e4m3 numbers).  A value that a row
    does not see has no part in it, whatever it is; table entries are kept inside the cache, lengths inside the table."""
    T, Hq, d = q.shape
    N, C, Hkv, _ = k_cache.shape
    G = Hq // Hkv
    out, size, total = (torch.zeros(T, Hq, d, dtype=torch.float64) for _ in range(3))
    for r in range(len(cu) - 1):
        n, length = cu[r + 1] - cu[r], max(0, min(lens[r], table.size(1) * C))
        chunks = table[r].long().clamp(0, N - 1)
        for i in range(n):
            keys = visible(length - n + i, length, window, sinks)
            if not keys:
                continue
            at = torch.tensor(keys)
            ids, loc = chunks[at // C], at % C
            K, V = k_cache[ids, loc].double(), v_cache[ids, loc].double()   # [keys, Hkv, d]
            if k_scales is not None:
                K, V = K * k_scales[ids].double()[..., None], V * v_scales[ids].double()[..., None]
            x = torch.einsum("khd,hgd->hgk", K, q[cu[r] + i].double().view(Hkv, G, d)) * scale
            p = torch.softmax(x, -1)
            out[cu[r] + i] = torch.einsum("hgk,khd->hgd", p, V).reshape(Hq, d)
            size[cu[r] + i] = torch.einsum("hgk,khd->hgd", p, V.abs()).reshape(Hq, d)
            total[cu[r] + i] = V.abs().sum(0).repeat_interleave(G, 0)
    return out, size, total


def axes_of_pairs(sections: Sequence[int], alternate: bool = False) -> List[int]:
    """The axis of every rotary pair: the axes' sections one after the other, or (``alternate``) the axes in turn as far as
    each section goes, and the first axis for the rest."""
    if not alternate:
        return [axis for axis, n in enumerate(sections) for _ in range(n)]
    out, n = [0] * sum(sections), len(sections)
    for axis in range(1, n):
        for j in range(sections[axis]):
            if axis + n * j < len(out):
                out[axis + n * j] = axis
    return out


def norm_rotate(x: Tensor, positions: Tensor, table: Tensor, axes: Sequence[int], *, norm: Optional[str] = None,
                weight: Optional[Tensor] = None, eps: float = 1e-5, interleaved: bool = False, mscale: float = 1.0) -> Tensor:
    """Head norm and rotation of ``x`` ``[T, H, d]`` in 64 bits: pair i turns by ``table[positions[axes[i]], column of i]``."""
    y, pairs = x.double().clone(), len(axes)
    if norm in ("rms", "l2"):
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
    if norm == "rms" and weight is not None:
        y = y * weight.double()
    out = y.clone()
    for i, axis in enumerate(axes):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        angle = table[positions[axis], a].double()[:, None]
        c, s = torch.cos(angle) * mscale, torch.sin(angle) * mscale
        # (the two halves of the table's row may differ: the second element turns by its own)
        angle_b = table[positions[axis], b].double()[:, None]
        cb, sb = torch.cos(angle_b) * mscale, torch.sin(angle_b) * mscale
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * cb + y[..., a] * sb
    return out
