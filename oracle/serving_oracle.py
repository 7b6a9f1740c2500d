"""Operators of a server's step in 64 bits, sequence by sequence, on the CPU (test infrastructure).

Written from the formulas alone: entries of a cache in pages, quantised as they
are written, attention of the newest tokens over them, the verification of drafted
tokens, and products in 8-bit integers.  Inputs are CPU tensors.
"""

from __future__ import annotations

import math

import numpy as np
import torch

STEP = np.float32(1) / np.float32(127)


def quantise(x):
    """x (..., d) -> (codes int8, scales fp32 (...)): by definition fp32 products and quotients."""
    x = x.float().numpy().astype(np.float32)
    most = np.abs(x).max(-1)
    odd = ~np.isfinite(x).all(-1)
    with np.errstate(all="ignore"):
        scale = (most * STEP).astype(np.float32)
        q = np.where(scale[..., None] > 0, x / scale[..., None], np.float32(0))
    scale = np.where(odd, np.float32("nan"), scale)
    q = np.where(odd[..., None], 0, np.clip(np.rint(q), -127, 127))
    return torch.from_numpy(q.astype(np.int8)), torch.from_numpy(scale)


def entry_place(cache, b, e):
    """(page, slot) of entry e of sequence b, or None where it has no page."""
    page = cache["k"].shape[2]
    if not 0 <= e < cache["table"].shape[1] * page:
        return None
    at = int(cache["table"][b, e // page])
    return (at, e % page) if 0 <= at < cache["k"].shape[0] else None


def length_of(cache, b):
    return min(max(int(cache["length"][b]), 0), cache["table"].shape[1] * cache["k"].shape[2])


def fresh_of(fresh, b, tokens):
    return tokens if fresh is None else min(max(int(fresh[b]), 0), tokens)


def entries(cache, x, b, g, upto):
    """Values (upto, d) in 64 bits, and which entries have a page."""
    pool, scale = cache[x], cache[x + "_scale"]
    got, there = torch.zeros((upto, pool.shape[3]), dtype=torch.float64), torch.zeros(upto, dtype=torch.bool)
    for e in range(upto):
        at = entry_place(cache, b, e)
        if at is not None:
            there[e] = True
            got[e] = pool[at[0], g, at[1]].double()
            if scale is not None:
                got[e] *= scale[at[0], g, at[1]].double()
    return got, there


def paged_write(cache, k_new, v_new, fresh=None):
    """-> the cache's new pools and scales, and the new lengths."""
    out = {n: x.clone() if isinstance(x, torch.Tensor) else x for n, x in cache.items()}
    rows, tokens = k_new.shape[:2]
    room, lengths = cache["table"].shape[1] * cache["k"].shape[2], []
    for b in range(rows):
        n, length = fresh_of(fresh, b, tokens), length_of(cache, b)
        lengths.append(min(length + n, room))
        for t in range(n):
            at = entry_place(cache, b, length + t)
            if at is None:
                continue
            for x, new in (("k", k_new), ("v", v_new)):
                if cache[x + "_scale"] is None:
                    out[x][at[0], :, at[1]] = new[b, t]
                else:
                    out[x][at[0], :, at[1]], out[x + "_scale"][at[0], :, at[1]] = quantise(new[b, t])
    out["length_out"] = torch.tensor(lengths, dtype=torch.int32)
    return out


def paged_read(cache, k_out, v_out, start=None):
    """k_out, v_out (rows, kv_heads, tokens, d) with the entries put in, in their own type."""
    got = []
    for x, out in (("k", k_out), ("v", v_out)):
        out = out.clone()
        for b in range(out.shape[0]):
            for t in range(out.shape[2]):
                e = t + (0 if start is None else int(start[b]))
                at = entry_place(cache, b, e) if 0 <= e < length_of(cache, b) else None
                if at is None:
                    continue
                v = cache[x][at[0], :, at[1]]
                if cache[x + "_scale"] is not None:
                    v = v.float() * cache[x + "_scale"][at[0], :, at[1]][:, None]
                out[b, :, t] = v.to(out.dtype)
        got.append(out)
    return got


def paged_attention(q, cache, fresh=None, scale=1.0, bias=None):
    """-> out (rows, tokens, heads, d), lse (rows, tokens, heads), both float64."""
    rows, tokens, heads, d = q.shape
    n = heads // cache["k"].shape[1]
    out = torch.zeros((rows, tokens, heads, d), dtype=torch.float64)
    lse = torch.full((rows, tokens, heads), -math.inf, dtype=torch.float64)
    room = cache["table"].shape[1] * cache["k"].shape[2]
    for b in range(rows):
        new, length = fresh_of(fresh, b, tokens), length_of(cache, b)
        if new == 0:
            continue
        end = min(length + new, room)
        for g in range(heads // n):
            k, there = entries(cache, "k", b, g, end)
            v, _ = entries(cache, "v", b, g, end)
            for h in range(g * n, (g + 1) * n):
                for t in range(new):
                    at = torch.arange(end)
                    x = scale * (k @ q[b, t, h].double())
                    see = there & (at <= length + t)
                    if bias is not None:
                        by = bias[h].double()[(length + t - at).clamp(0, bias.shape[1] - 1)]
                        x, see = x + by, see & (by > -6.9e29)
                    if not see.any():
                        continue
                    lse[b, t, h] = torch.logsumexp(x[see], 0)
                    p = torch.softmax(x[see], 0)
                    out[b, t, h] = p @ v[see]
    return out, lse


def draft_verify(target, draft, tokens, uniforms, parents=None):
    """-> (paths, tokens that follow), whole numbers."""
    rows, slots, vocab = target.shape
    clean = lambda x: torch.where((x > 0) & (x < math.inf), x, torch.zeros_like(x)).double().numpy()  # noqa: E731
    paths, last = [], []
    for b in range(rows):
        up = list(range(-1, slots - 2)) if parents is None else [int(p) for p in (parents[b] if parents.dim() == 2 else parents)]
        node, path = -1, []
        while True:
            p = clean(target[b, node + 1])
            rest, z, took = p.copy(), 1.0, None
            kids = [t for t in range(node + 1, slots - 1) if up[t] == node and 0 <= int(tokens[b, t]) < vocab]
            q = clean(draft[b, node + 1]) if draft is not None and kids else None
            for t in kids:
                x, u = int(tokens[b, t]), float(uniforms[b, t])
                if u * z * (1.0 if q is None else q[x]) < rest[x]:
                    took = t
                    break
                if q is None:
                    z -= rest[x]
                    rest[x] = 0.0
                else:
                    rest = np.maximum(rest - z * q, 0.0)
                    z = rest.sum()
            if took is None:
                break
            node = took
            path.append(took)
        if not rest.sum() > 0:
            rest = p
        run = np.cumsum(rest)
        past = np.flatnonzero(run > max(float(uniforms[b, -1]) * run[-1], 0.0))
        some = np.flatnonzero(rest > 0)
        last.append(int(past[0]) if len(past) else int(some[-1]) if len(some) else -1)
        paths.append(path)
    return paths, last


def i8_matmul(x, x_scale, w, w_scale, add=None):
    y = (x.double() @ w.double().T) * x_scale.double()[:, None] * w_scale.double()
    return y if add is None else y + add.double()
