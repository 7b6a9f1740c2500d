"""Drafting operators in 64 bits, sequence by sequence, on the CPU (test infrastructure).

Written from the formulas alone: attention of a drafted tree over a cache, the
commit of an accepted path with its attention weights, eviction by them, and
products with 4-bit weights.  Inputs are CPU tensors of any floating type.
"""

from __future__ import annotations

import math

import torch


def chains(parents):
    """Each node's path from the root down to itself; None where it is not there."""
    got = []
    for t, p in enumerate(int(x) for x in parents):
        above = [] if p == -1 else got[p] if 0 <= p < t else None
        got.append(None if above is None else above + [t])
    return got


def _logits(q, qpos, k, kpos, scale, bias):
    """q (N, d), k (L, d), positions (N,), (L,); bias (buckets,) -> (N, L) float64."""
    x = scale * (q.double() @ k.double().T)
    if bias is not None:
        far = (qpos[:, None] - kpos[None, :]).clamp(0, bias.shape[0] - 1)
        x = x + bias.double()[far]
    return x


def tree_attention(q, k_new, v_new, k, v, length, parents, scale=1.0, bias=None, pos=None, next_pos=None):
    """-> out (rows, nodes, heads, d), lse (rows, nodes, heads), both float64."""
    rows, nodes, heads, d = q.shape
    kv_heads, cap = k.shape[1], k.shape[2]
    n = heads // kv_heads
    out = torch.zeros((rows, nodes, heads, d), dtype=torch.float64)
    lse = torch.full((rows, nodes, heads), -math.inf, dtype=torch.float64)
    for b in range(rows):
        L = min(max(int(length[b]), 0), cap)
        paths = chains(parents[b] if parents.dim() == 2 else parents)
        first = L if pos is None else int(next_pos[b])
        for h in range(heads):
            g = h // n
            kpos = torch.arange(L) if pos is None else pos[b, g, :L].long()
            row = None if bias is None else bias[h]
            for t, path in enumerate(paths):
                if path is None:
                    continue
                at = torch.tensor([len(path) - 1])
                x = torch.cat([_logits(q[b, t, h][None], first + at, k[b, g, :L], kpos, scale, row),
                               _logits(q[b, t, h][None], at, k_new[b, path, g], torch.arange(len(path)), scale, row)], 1)[0]
                lse[b, t, h] = torch.logsumexp(x, 0)
                out[b, t, h] = torch.softmax(x, 0) @ torch.cat([v[b, g, :L], v_new[b, path, g]]).double()
    return out, lse
