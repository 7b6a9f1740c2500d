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


def accepted_prefix(nodes_of, nodes, room):
    """The longest prefix of ascending ids in [0, nodes) that fits."""
    path = []
    for t in (int(x) for x in nodes_of):
        if t <= (path[-1] if path else -1) or t >= nodes or len(path) >= room:
            break
        path.append(t)
    return path


def cache_commit(k, v, length, k_new, v_new, accepted, q=None, lse=None, score=None, score_out=None, scale=1.0, bias=None,
                 pos=None, next_pos=None):
    """-> dict of the new k, v, pos, length, next_pos, score (float64; score_out's values past the entries)."""
    rows, kv_heads, cap, _ = k.shape
    out = dict(k=k.clone(), v=v.clone(), pos=None if pos is None else pos.clone(), length=[], next_pos=[],
               score=None if q is None else score_out.double().clone())
    for b in range(rows):
        L = min(max(int(length[b]), 0), cap)
        path = accepted_prefix(accepted[b], k_new.shape[1], cap - L)
        n, first = len(path), L if pos is None else int(next_pos[b])
        out["length"].append(L + n)
        out["next_pos"].append(first + n)
        for g in range(kv_heads):
            for i, t in enumerate(path):
                out["k"][b, g, L + i], out["v"][b, g, L + i] = k_new[b, t, g], v_new[b, t, g]
                if pos is not None:
                    out["pos"][b, g, L + i] = first + i
            if q is None:
                continue
            total = torch.zeros(L + n, dtype=torch.float64)
            if score is not None:
                total[:L] = score[b, g, :L].double()
            share = q.shape[2] // kv_heads
            kpos = torch.arange(L + n) if pos is None else out["pos"][b, g, :L + n].long()
            for i, t in enumerate(path):
                for h in range(g * share, (g + 1) * share):
                    if float(lse[b, t, h]) == -math.inf:
                        continue
                    x = _logits(q[b, t, h][None], torch.tensor([first + i]), out["k"][b, g, :L + n], kpos, scale,
                                None if bias is None else bias[h])[0]
                    w = (x - float(lse[b, t, h])).exp()
                    w[L + i + 1:] = 0
                    total += w
            out["score"][b, g, :L + n] = total
    out["length"], out["next_pos"] = (torch.tensor(out[x], dtype=torch.int32) for x in ("length", "next_pos"))
    return out


def cache_evict(k, v, length, pos, next_pos, score, keep, recent, sinks):
    """-> dict of the new k, v, length, and (rows, kv_heads) lists of each head's new scores and positions."""
    rows, kv_heads, cap, _ = k.shape
    out = dict(k=k.clone(), v=v.clone(), length=[], score=[], pos=[])
    for b in range(rows):
        L = min(max(int(length[b]), 0), cap)
        m = min(L, keep)
        out["length"].append(m)
        for g in range(kv_heads):
            positions, scores = pos[b, g].tolist(), score[b, g].tolist()

            def rank(j):
                p, s = positions[j], scores[j]
                stays = p >= int(next_pos[b]) - recent or p < sinks
                return (not stays, math.inf if math.isnan(s) else -s, j)
            kept = sorted(sorted(range(L), key=rank)[:m])
            src, stay = list(range(m)), set(kept)
            holes = [j for j in range(m) if j not in stay]
            for to, at in zip(holes, [j for j in kept if j >= m]):
                src[to] = at
            out["k"][b, g, :m], out["v"][b, g, :m] = k[b, g, src], v[b, g, src]
            out["score"].append(score[b, g, src])
            out["pos"].append(pos[b, g, src])
    out["length"] = torch.tensor(out["length"], dtype=torch.int32)
    return out


def q4_weights(w, scales, biases):
    """The (n, k) float64 weights of 4-bit codes."""
    n, words = w.shape
    word = w.long() & 0xFFFFFFFF
    codes = torch.stack([(word >> (4 * i)) & 15 for i in range(8)], -1).reshape(n, words * 8)
    group = words * 8 // scales.shape[1]
    return codes.double() * scales.double().repeat_interleave(group, 1) + biases.double().repeat_interleave(group, 1)
