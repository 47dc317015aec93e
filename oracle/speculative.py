"""Oracle for a step of speculative decoding: attention of drafted tokens, their verification, the cache afterwards.

TEST INFRASTRUCTURE ONLY -- nothing in the product imports this module.

The reference has no counterpart (its dynamic engine decodes one token per request and step), so everything here is the
operators' definition, in 64 bits on CPU tensors and by explicit loops over requests, nodes and tokens.  Pinned by
(tests/test_oracle_speculative.py): the causal oracle for chains, a dense masked softmax, the distribution of accepted and
drawn tokens against the target's own by counting, and hand-worked trees.
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

import torch
from torch import Tensor


def ancestors(parents: Sequence[int]) -> List[int]:
    """A row of bits per node: its ancestors and itself (Python integers, bit j = node j)."""
    bits: List[int] = []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
    return bits


def mask_rows(bits: Sequence[int], words: int) -> Tensor:
    """Rows of ``words`` int64 words."""
    def signed(w):
        return w - (1 << 64) if w >> 63 else w
    return torch.tensor([[signed(b >> 64 * w & (1 << 64) - 1) for w in range(words)] for b in bits],
                        dtype=torch.int64).view(len(bits), words)


def position(table_row: Sequence[int], chunk: int, n_chunks: int, pos: int) -> Optional[Tuple[int, int]]:
    """(chunk id, local position) of a request's position, None where the table names no chunk of the cache."""
    if pos < 0 or pos >= len(table_row) * chunk:
        return None
    c = table_row[pos // chunk]
    return (c, pos % chunk) if 0 <= c < n_chunks else None


def tree_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, cu: Sequence[int], lens: Sequence[int], table: Tensor,
                   bits: Sequence[int], scale: float, k_scales: Optional[Tensor] = None,
                   v_scales: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """(result, sum of probability times |value|), both fp64 ``[T, Hq, d]``; ``k_cache`` / ``v_cache`` hold values (of an fp8
    cache: the e4m3 numbers).  A value that a row does not see has no part in it, whatever it is."""
    T, Hq, d = q.shape
    N, C, Hkv, _ = k_cache.shape
    G, rows = Hq // Hkv, table.tolist()
    out, size = torch.zeros(T, Hq, d, dtype=torch.float64), torch.zeros(T, Hq, d, dtype=torch.float64)
    for r in range(len(cu) - 1):
        n = cu[r + 1] - cu[r]
        length = max(0, min(lens[r], len(rows[r]) * C))
        first = length - n
        places = [position(rows[r], C, N, k) for k in range(length)]
        for i in range(n):
            keys = [k for k in range(length) if places[k] is not None and (k < first or bits[cu[r] + i] >> (k - first) & 1)]
            if not keys:
                continue
            at = torch.tensor([places[k] for k in keys])
            K, V = k_cache[at[:, 0], at[:, 1]].double(), v_cache[at[:, 0], at[:, 1]].double()   # [keys, Hkv, d]
            if k_scales is not None:
                K, V = K * k_scales[at[:, 0]].double()[..., None], V * v_scales[at[:, 0]].double()[..., None]
            for h in range(Hq):
                x = (K[:, h // G] @ q[cu[r] + i, h].double()) * scale
                p = torch.softmax(x, 0)
                out[cu[r] + i, h] = p @ V[:, h // G]
                size[cu[r] + i, h] = p @ V[:, h // G].abs()
    return out, size


def scaled_logits(logits: Tensor, temperature: float) -> Tensor:
    if temperature == 1.0:
        return logits.float()
    inv = torch.tensor(1.0) / torch.tensor(temperature, dtype=torch.float32)
    return (logits.float() * inv).to(logits.dtype).float()


def verify(logits: Tensor, tokens: Sequence[int], parents: Sequence[int], cu: Sequence[int], max_path: int, *,
           greedy: bool = False, draft_probs: Optional[Tensor] = None, uniform: Optional[Sequence[float]] = None,
           temperature: float = 1.0, cut: Optional[Sequence[float]] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """``(tokens [R, max_path], rows [R, max_path], counts [R])`` by walking each tree."""
    R, V = len(cu) - 1, logits.size(1)
    out = torch.full((R, max_path), -1, dtype=torch.int64)
    rows = torch.full((R, max_path), -1, dtype=torch.int32)
    counts = torch.zeros(R, dtype=torch.int32)
    for r in range(R):
        base, n = cu[r], cu[r + 1] - cu[r]
        if n == 0:
            continue
        node, path, new = 0, [base], []
        while True:
            x = logits[base + node].float() if greedy else scaled_logits(logits[base + node], temperature)
            if greedy:
                best = int(torch.argmax(x))
                p = torch.zeros(V, dtype=torch.float64)
                p[best] = 1.0
            else:
                z = x.double()
                if cut is not None:
                    z = torch.where(x < cut[base + node], torch.tensor(-math.inf, dtype=torch.float64), z)
                p = torch.softmax(z, 0)
            target, following = p.clone(), None
            for i in range(node + 1, n if len(path) < max_path else 0):
                if parents[base + i] != node:
                    continue
                t = tokens[base + i]
                w = float(p[t]) if 0 <= t < V else 0.0
                if greedy:
                    ok = w > 0
                elif draft_probs is None:
                    ok = uniform[base + i] * float(p.sum()) < w
                else:
                    q = draft_probs[base + node].double()
                    ok = uniform[base + i] * (float(q[t]) if 0 <= t < V else 0.0) * float(p.sum()) < w
                if ok:
                    following = i
                    break
                if greedy:
                    continue
                if draft_probs is None:
                    if 0 <= t < V:
                        p[t] = 0
                else:
                    p = (p / p.sum() - q).clamp(min=0)
            if following is None:
                if not float(p.sum()) > 1e-13:
                    p = target
                cdf = p.cumsum(0)
                u = 0.0 if greedy else uniform[base] * float(cdf[-1])
                new.append(int((cdf <= u).sum()))
                break
            node = following
            path.append(base + node)
            new.append(tokens[base + node])
        counts[r] = len(path)
        out[r, :len(new)] = torch.tensor(new)
        rows[r, :len(path)] = torch.tensor(path, dtype=torch.int32)
    return out, rows, counts


def keep_accepted(cache: Tensor, rows: Tensor, counts: Sequence[int], cu: Sequence[int], lens: Sequence[int],
                  table: Tensor, scales: Optional[Tensor] = None) -> Tensor:
    """One cache ``[layers, N, C, H, d]`` (of an fp8 cache: the e4m3 numbers as fp32) after the move, entry by entry."""
    cache, t = cache.clone(), table.tolist()
    _, N, C = cache.shape[:3]
    for r in range(len(cu) - 1):
        n = cu[r + 1] - cu[r]
        for i in range(1, counts[r]):
            node = int(rows[r, i]) - cu[r]
            if not 0 <= node < n:
                continue
            a, b = position(t[r], C, N, lens[r] - n + node), position(t[r], C, N, lens[r] - n + i)
            if a is None or b is None or a == b:
                continue
            moved = cache[:, a[0], a[1]].clone()
            if scales is not None and a[0] != b[0]:
                f = scales[:, a[0]] / scales[:, b[0]]
                moved = (moved * f[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).float()
            cache[:, b[0], b[1]] = moved
    return cache
