"""Serving operators over caller-owned caches and 4-bit weights: their cases, plain forms and 64-bit values.

Four operators, together a step of drafting decode: the drafting products from
4-bit weights (``q4_matmul``), the attention of a tree of drafted tokens over a
cache (``tree_attention``), the commit of the accepted path with the attention
weights its tokens gave to the cache's entries (``cache_commit``), and the
eviction of the entries with the least of it (``cache_evict``).

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges,
``prepare`` makes a case's inputs, ``run`` is one pass, ``work`` counts what a
pass cannot do without and ``exact`` evaluates a case in 64 bits.  With ``own``
false ``run`` computes in elementary torch operations in 32 bits.
"""

import functools
import math
import pathlib
import sys

import numpy as np
import torch

own = False

DEV = "cuda:0"
TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
MAX_NODES = 64


@functools.lru_cache(maxsize=None)
def _package():
    pkg = str(pathlib.Path(__file__).resolve().parents[1] / "magenta-realtime-mlx-cpp_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import mrt_df
    return mrt_df


# ---------------------------------------------------------------------------
# The cases.  rows: sequences (a CFG pair is two).  nodes: drafted tokens of a
# sequence.  length: entries in use of the longest sequence; ragged: the others
# hold fewer.  buckets: columns of the bias by distance (0: none).  evicted: the
# cache has had evictions, so that each entry's position is in an array.


def listed():
    return [
        # One token of one live stream against its frame cache: the smallest call, all latency.
        dict(name="tree_step", op="tree", dtype="bf16", rows=2, heads=16, kv_heads=16, d=64, nodes=1, length=49,
             buckets=128, ragged=False, evicted=False),
        # A frame's drafts, branching, over a 10 s context of a live stream.
        dict(name="tree_frame", op="tree", dtype="fp16", rows=2, heads=16, kv_heads=16, d=64, nodes=33, length=1006,
             buckets=0, ragged=False, evicted=False),
        # Few sequences with long caches and shared heads, some minutes of context.
        dict(name="tree_long", op="tree", dtype="bf16", rows=3, heads=32, kv_heads=8, d=128, nodes=15, length=65500,
             buckets=0, ragged=True, evicted=False),
        # A server's batch with the largest trees: many query rows for each cached entry.
        dict(name="tree_wide", op="tree", dtype="bf16", rows=16, heads=32, kv_heads=4, d=128, nodes=64, length=8191,
             buckets=0, ragged=True, evicted=False),
        # The 12-head configuration in fp32 with its bias by distance, on a cache held to a budget.
        dict(name="tree_fp32", op="tree", dtype="fp32", rows=4, heads=12, kv_heads=12, d=64, nodes=7, length=4099,
             buckets=128, ragged=True, evicted=True),
        # The accepted tokens of a frame into a live stream's cache.
        dict(name="commit_frame", op="commit", dtype="bf16", rows=2, heads=16, kv_heads=16, d=64, nodes=16, length=1006,
             buckets=0, ragged=False, evicted=True),
        # The same on long caches with shared heads.
        dict(name="commit_long", op="commit", dtype="fp16", rows=5, heads=32, kv_heads=8, d=128, nodes=16,
             length=40001, buckets=0, ragged=True, evicted=True),
        # 32 live streams held to the encoder's context length, a chunk's worth of entries over it.
        dict(name="evict_streams", op="evict", dtype="bf16", rows=64, heads=16, kv_heads=16, d=64, length=1056,
             keep=1006, recent=128, sinks=4),
        # Long caches halved.
        dict(name="evict_long", op="evict", dtype="bf16", rows=4, heads=32, kv_heads=8, d=128, length=65536,
             keep=32768, recent=1000, sinks=4),
        # The smallest product of a drafting step: one CFG pair through a gate and up projection.
        dict(name="q4_ffn", op="q4", dtype="bf16", rows=2, k=1024, n=5632, group=64),
        # The whole head for the nodes of a frame's drafts, in the model's largest type.
        dict(name="q4_head_fp32", op="q4", dtype="fp32", rows=5, k=1024, n=29824, group=32),
        # A large layer for a few drafted tokens.
        dict(name="q4_large", op="q4", dtype="bf16", rows=9, k=8192, n=28672, group=128),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(16, 16, 64), (12, 12, 64), (16, 16, 64), (32, 8, 128), (32, 4, 128), (28, 4, 128), (8, 1, 256), (6, 2, 96),
         (8, 8, 32), (15, 5, 64)]


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most:
            return c


def _draw(rng):
    op, dtype = rng.choice(["tree", "tree", "commit", "evict", "q4", "q4"]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "q4":
        group = rng.choice([32, 64, 128])
        return dict(op=op, dtype=dtype, rows=_log_int(rng, 1, 64), k=group * _log_int(rng, 1, 8192 // group),
                    n=_log_int(rng, 16, 30000), group=group)
    heads, kv_heads, d = rng.choice(HEADS)
    c = dict(op=op, dtype=dtype, rows=_log_int(rng, 1, 64), heads=heads, kv_heads=kv_heads, d=d,
             length=_log_int(rng, 1, 66000))
    if op == "evict":
        keep = max(1, int(c["length"] * rng.uniform(0.3, 1.0)))
        return dict(c, keep=keep, recent=rng.randrange(keep // 2 + 1), sinks=min(rng.choice([0, 1, 4]), keep // 4))
    return dict(c, nodes=_log_int(rng, 1, MAX_NODES), buckets=rng.choice([0, 0, 16, 128, 1000]),
                ragged=rng.random() < 0.5, evicted=rng.random() < 0.4)


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 4e12, w["flops"] / 5e14)


def work(case):
    e, m = BYTES[case["dtype"]], case["rows"]
    if case["op"] == "q4":
        k, n = case["k"], case["n"]
        return {"bytes": n * k // 2 + 2 * n * (k // case["group"]) * e + m * (k + n) * e, "flops": 2 * m * n * k}
    H, G, d, L = case["heads"], case["kv_heads"], case["d"], case["length"]
    if case["op"] == "evict":
        keep, free = case["keep"], L - min(L, case["recent"] + case["sinks"])
        gone = max(0, L - keep)
        # evicted entries fall evenly on the unprotected slots; those below `keep` are holes, filled from above it
        holes = gone * max(0, min(free, keep - case["sinks"])) // max(1, free)
        return {"bytes": m * G * (8 * L + 8 * min(L, keep) + 4 * holes * d * e), "flops": 0}
    T = case["nodes"]
    total = sum(_lengths(case))
    if case["op"] == "tree":
        small = m * T * (2 * H + 2 * G) * d * e + m * T * (4 + 4 * H) + 4 * H * case["buckets"]
        return {"bytes": 2 * total * G * d * e + (4 * total * G if case["evicted"] and case["buckets"] else 0) + small,
                "flops": 4 * T * H * d * total + 2 * m * T * T * H * d}
    A = (T + 1) // 2  # accepted tokens, about
    return {"bytes": total * G * (d * e + 8) + m * A * (H + 4 * G) * d * e, "flops": 2 * A * H * d * total}


def _lengths(case):
    """Entries in use of each sequence: equal, or spread from the whole length down to a seventh of it."""
    L, m = case["length"], case["rows"]
    return [L - (L - L // 7) * b // max(1, m - 1) if case["ragged"] else L for b in range(m)]


# ---------------------------------------------------------------------------
# Inputs


def _tree(rng, nodes):
    """Parents of a drafted tree: half of the nodes extend the newest branch, the others branch anywhere."""
    return [-1] + [t - 1 if rng.rand() < 0.5 else int(rng.randint(-1, t)) for t in range(1, nodes)]


def _path(rng, parents):
    """A path from a root child down, about half of the deepest one's length."""
    t, path = int(rng.randint(0, len(parents))), []
    while t >= 0:
        path.append(t)
        t = parents[t]
    return path[::-1][:(len(parents) + 1) // 2]


def prepare(case, seed):
    rng = np.random.RandomState(seed & 0x7FFFFFFF)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = TORCH[case["dtype"]]

    def normal(*shape, scale=1.0, to=dt):
        return torch.empty(shape, device=DEV, dtype=to).normal_(0.0, scale, generator=g)

    def on_device(v):
        return torch.from_numpy(np.ascontiguousarray(v)).to(DEV)

    s = dict(op=case["op"])
    m = case["rows"]
    if case["op"] == "q4":
        n, k, group = case["n"], case["k"], case["group"]
        w = torch.randint(-2 ** 31, 2 ** 31 - 1, (n, k // 8), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
        scales = (torch.rand((n, k // group), generator=g, device=DEV) * 0.5 + 0.5) / (8 * math.sqrt(k))
        s.update(x=normal(m, k), w=w, scales=scales.to(dt),
                 biases=(scales * (torch.randn((n, k // group), generator=g, device=DEV) * 0.5 - 7.5)).to(dt))
        return s
    H, G, d, L = case["heads"], case["kv_heads"], case["d"], case["length"]
    if case["op"] == "evict":
        C = L + 5
        # slots that evictions have filled again: positions out of order
        order = torch.arange(L, device=DEV) + torch.rand((m, G, L), generator=g, device=DEV) * (L / 4)
        # what accumulates: most entries little, some much
        score = torch.empty((m, G, C), device=DEV).normal_(0.0, 1.5, generator=g).exp_()
        s.update(k=normal(m, G, C, d), v=normal(m, G, C, d), score=score,
                 pos=torch.full((m, G, C), -1, dtype=torch.int32, device=DEV),
                 length=torch.full((m,), L, dtype=torch.int32, device=DEV),
                 next_pos=torch.full((m,), L, dtype=torch.int32, device=DEV),
                 keep=case["keep"], recent=case["recent"], sinks=case["sinks"])
        s["pos"][..., :L] = order.argsort(-1).to(torch.int32)
        s.update(length_out=torch.zeros_like(s["length"]), score_out=torch.zeros_like(score),
                 pos_out=torch.full_like(s["pos"], -1))
        return s
    T = case["nodes"]
    lengths = np.array(_lengths(case), dtype=np.int32)
    C = L + T + 5
    scale = 1.0 / math.sqrt(d)
    s.update(scale=scale, q=normal(m, T, H, d, scale=1.5), k_new=normal(m, T, G, d), v_new=normal(m, T, G, d),
             k=normal(m, G, C, d), v=normal(m, G, C, d), length=on_device(lengths), pos=None, next_pos=None, bias=None)
    if case["buckets"]:
        s["bias"] = normal(H, case["buckets"], to=torch.float32)
    if case["evicted"]:  # gaps where entries went: each position a few past the one before
        step = torch.randint(1, 4, (m, G, C), generator=g, device=DEV)
        pos = step.cumsum(-1)
        s["next_pos"] = (pos.amax((1, 2)) + 1).to(torch.int32)
        s["pos"] = pos.to(torch.int32)
    parents = [_tree(rng, T) for _ in range(m)]
    s["parents"] = on_device(np.array(parents, dtype=np.int32))
    if case["op"] == "commit":
        paths = [_path(rng, p) for p in parents]
        s["accepted"] = on_device(np.array([p + [-1] * (T - len(p)) for p in paths], dtype=np.int32))
        s["lse"] = _tree_attention(s)[1]
        s["score"] = torch.rand((m, G, C), generator=g, device=DEV) * 8
        s.update(score_out=s["score"].clone(), length_out=torch.zeros_like(s["length"]),
                 next_out=torch.zeros_like(s["length"]))
        if s["pos"] is None:
            s["next_out"] = None
    return s


# ---------------------------------------------------------------------------
# One pass


def run(s):
    if own:
        return _run_own(s)
    return {"tree": _tree_attention, "commit": _commit, "evict": _evict, "q4": _q4}[s["op"]](s)


def _run_own(s):
    mrt_df = _package()
    if s["op"] == "q4":
        return mrt_df.q4_matmul(s["x"], s["w"], s["scales"], s["biases"])
    if s["op"] == "tree":
        cache = mrt_df.KVCache(s["k"], s["v"], s["length"], pos=s["pos"], next_pos=s["next_pos"])
        return mrt_df.tree_attention(s["q"], s["k_new"], s["v_new"], cache, s["parents"], scale=s["scale"], bias=s["bias"])
    cache = mrt_df.KVCache(s["k"], s["v"], s["length"], pos=s["pos"], next_pos=s["next_pos"], score=s["score"])
    if s["op"] == "commit":
        mrt_df.cache_commit(cache, s["k_new"], s["v_new"], s["accepted"], s["length_out"], next_out=s["next_out"],
                            q=s["q"], lse=s["lse"], score_out=s["score_out"], scale=s["scale"], bias=s["bias"])
        return [s["k"], s["v"], s["pos"], s["length_out"], s["next_out"], s["score_out"]]
    mrt_df.cache_evict(cache, s["keep"], s["length_out"], s["score_out"], s["pos_out"], recent=s["recent"],
                       sinks=s["sinks"])
    return [s["k"], s["v"], s["length_out"], s["score_out"], s["pos_out"]]


def _visible(parents):
    """(sees (m, T, T), present (m, T), depth (m, T)) of the drafted nodes."""
    T = parents.shape[1]
    at = torch.arange(T, device=parents.device)
    known = (parents >= -1) & (parents < at)
    up = ((parents[..., None] == at) & known[..., None]).float()
    reach = torch.linalg.matrix_power(up + torch.eye(T, device=parents.device), MAX_NODES) > 0
    present = ~(reach & ~known[:, None, :]).any(-1)
    return reach & present[..., None], present, reach.sum(-1) - 1


def _positions(s):
    """Positions of the cache's slots and of the next token."""
    if s["pos"] is not None:
        return s["pos"].long(), s["next_pos"].long()
    m, G, C, _ = s["k"].shape
    return torch.arange(C, device=s["k"].device).expand(m, G, C), s["length"].long()


def _by_distance(bias, distance):
    """bias (H, M) at distance (m, G, N, C): (m, H, N, C), the last column for what lies further."""
    H, M = bias.shape
    m, G, N, C = distance.shape
    d = distance.clamp(0, M - 1)[:, :, None].expand(m, G, H // G, N, C).reshape(m, H, N, C)
    return bias[torch.arange(H, device=bias.device)[None, :, None, None], d]


def _tree_attention(s):
    q, k_new, v_new, k, v = (s[n].float() for n in ("q", "k_new", "v_new", "k", "v"))
    m, T, H, d = q.shape
    G, C = k.shape[1], k.shape[2]
    sees, present, depth = _visible(s["parents"])
    q = q.transpose(1, 2).reshape(m, G, H // G * T, d)
    k_new, v_new = (x.transpose(1, 2).contiguous() for x in (k_new, v_new))
    old = (q @ k.transpose(-1, -2).contiguous()).view(m, H, T, C) * s["scale"]
    new = (q @ k_new.transpose(-1, -2).contiguous()).view(m, H, T, T) * s["scale"]
    if s["bias"] is not None:
        pos, first = _positions(s)
        own_pos = first[:, None, None, None] + depth[:, None, :, None]
        old = old + _by_distance(s["bias"], own_pos - pos[:, :, None, :])
        new = new + _by_distance(s["bias"], (depth[:, :, None] - depth[:, None, :])[:, None].expand(m, G, T, T))
    used = torch.arange(C, device=k.device) < s["length"][:, None]
    old = old.masked_fill(~(used[:, None, :] & present[:, :, None])[:, None], -math.inf)
    new = new.masked_fill(~sees[:, None], -math.inf)
    top = torch.maximum(old.amax(-1, keepdim=True), new.amax(-1, keepdim=True)).clamp_min(-3e38)
    old, new = (old - top).exp_(), (new - top).exp_()
    total = old.sum(-1, keepdim=True) + new.sum(-1, keepdim=True)
    out = old.view(m, G, H // G * T, C) @ v + new.view(m, G, H // G * T, T) @ v_new
    out = out.view(m, H, T, d) / torch.where(total > 0, total, 1.0)
    lse = torch.where(total > 0, top + total.log(), -math.inf)
    return out.transpose(1, 2).to(s["q"].dtype).contiguous(), lse[..., 0].transpose(1, 2).contiguous()


def _commit(s):
    k, v, length = s["k"], s["v"], s["length"].long()
    m, T, H, d = s["q"].shape
    G, C = k.shape[1], k.shape[2]
    acc = s["accepted"].long()
    A = acc.shape[1]
    at = torch.arange(A, device=k.device)
    before = torch.cat([acc.new_full((m, 1), -1), acc[:, :-1]], 1)
    good = ((acc > before) & (acc < T) & (length[:, None] + at < C)).long().cumprod(1).bool()
    count = good.sum(1)
    slot = (length[:, None] + at).clamp(max=C - 1)
    row, node = torch.arange(m, device=k.device)[:, None], acc.clamp(0, T - 1)
    for cache, fresh in ((k, s["k_new"]), (v, s["v_new"])):
        cache[row, :, slot] = torch.where(good[..., None, None], fresh[row, node], cache[row, :, slot])
    pos, first = _positions(s)
    if s["pos"] is not None:
        s["pos"][row, :, slot] = torch.where(good, first[:, None] + at, 0).to(torch.int32)[..., None].where(
            good[..., None], s["pos"][row, :, slot])
        pos = s["pos"].long()
        s["next_out"].copy_(first + count)
    s["length_out"].copy_(length + count)
    q = s["q"][row, node].float().transpose(1, 2).reshape(m, G, H // G * A, d)
    logit = (q @ k.float().transpose(-1, -2).contiguous()).view(m, H, A, C) * s["scale"]
    if s["bias"] is not None:
        logit = logit + _by_distance(s["bias"], first[:, None, None, None] + at[:, None] - pos[:, :, None, :])
    lse = s["lse"][row, node].transpose(1, 2)[..., None]
    seen = (torch.arange(C, device=k.device) <= slot[..., None]) & good[..., None]
    weight = torch.where(seen[:, None], (logit - lse).exp(), 0.0).view(m, G, -1, C).sum(2)
    j = torch.arange(C, device=k.device)[None, None]
    end = length[:, None, None]
    s["score_out"].copy_(torch.where(j < end, s["score"] + weight,
                                     torch.where(j < end + count[:, None, None], weight, s["score_out"])))
    return [k, v, s["pos"], s["length_out"], s["next_out"], s["score_out"]]


def _evict(s):
    k, v, score, pos = s["k"], s["v"], s["score"], s["pos"]
    m, G, C, d = k.shape
    slot = torch.arange(C, device=k.device)
    valid = (slot < s["length"][:, None]).unsqueeze(1).expand(m, G, C)
    fixed = ((pos >= (s["next_pos"] - s["recent"])[:, None, None]) | (pos < s["sinks"])) & valid
    key = torch.where(score.isnan() | ~valid, -math.inf, score).masked_fill(fixed, math.inf)
    best = key.argsort(dim=-1, descending=True, stable=True)[..., :s["keep"]]
    kept = torch.zeros_like(valid).scatter_(-1, best, True) & valid
    end = s["length"].clamp(max=s["keep"]).long()
    low = slot < end[:, None, None]
    hole, mover = low & ~kept, ~low & kept
    rank = hole.cumsum(-1) - 1
    order = torch.where(mover, mover.cumsum(-1) - 1, C)
    by_rank = torch.zeros((m, G, C + 1), dtype=torch.long, device=k.device).scatter_(-1, order, slot.expand(m, G, C))
    src = torch.where(hole, by_rank.gather(-1, rank.clamp_min(0)), slot)[..., :s["keep"]]
    low = low[..., :s["keep"]]
    for cache in (k, v):
        cache[:, :, :s["keep"]] = cache.gather(2, src[..., None].expand(m, G, src.shape[2], d))
    for to, values in ((s["score_out"], score), (s["pos_out"], pos)):
        to[..., :s["keep"]] = torch.where(low, values.gather(-1, src), to[..., :s["keep"]])
    s["length_out"].copy_(end)
    return [k, v, s["length_out"], s["score_out"], s["pos_out"]]


def _q4(s):
    n, words = s["w"].shape
    groups = s["scales"].shape[1]
    q = (s["w"][..., None] >> torch.arange(0, 32, 4, device=s["w"].device, dtype=torch.int32)) & 15
    w = q.view(n, groups, -1).float() * s["scales"].float()[..., None] + s["biases"].float()[..., None]
    return (s["x"].float() @ w.view(n, -1).t().contiguous()).to(s["x"].dtype)


# ---------------------------------------------------------------------------
# 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _tree64, "commit": _commit64, "evict": _evict64, "q4": _q4_64}[case["op"]](s)


def _chains(parents):
    """Each node's path from the root, itself last; None where it has none."""
    got = []
    for t, p in enumerate(parents):
        above = [] if p == -1 else got[p] if 0 <= p < t else None
        got.append(None if above is None else above + [t])
    return got


def _logits64(s, b, g, q, qpos, keys, kpos):
    """(heads of group g, queries, keys) of sequence b: q (queries, H, d) at qpos, keys at kpos."""
    H = s["q"].shape[2]
    n = H // s["k"].shape[1]
    x = torch.stack([q[:, g * n + i].double() @ keys.double().t() for i in range(n)]) * s["scale"]
    if s["bias"] is None:
        return x
    M = s["bias"].shape[1]
    far = (qpos[:, None] - kpos[None]).clamp(0, M - 1)
    return x + s["bias"][g * n:(g + 1) * n].double()[:, far]


def _tree64(s):
    m, T, H, d = s["q"].shape
    G = s["k"].shape[1]
    n = H // G
    out = torch.zeros((m, T, H, d), dtype=torch.float64, device=DEV)
    lse = torch.full((m, T, H), -math.inf, dtype=torch.float64, device=DEV)
    for b, parents in enumerate(s["parents"].tolist()):
        end, chains = int(s["length"][b]), _chains(parents)
        here = [t for t in range(T) if chains[t] is not None]
        depth = torch.tensor([len(chains[t]) - 1 for t in here], device=DEV)
        mask = torch.tensor([[u in chains[t] for u in here] for t in here], device=DEV)
        at = torch.tensor(here, device=DEV)
        for g in range(G):
            pos = s["pos"][b, g, :end].long() if s["pos"] is not None else torch.arange(end, device=DEV)
            first = int(s["next_pos"][b]) if s["pos"] is not None else end
            q = s["q"][b, at]
            old = _logits64(s, b, g, q, first + depth, s["k"][b, g, :end], pos)
            new = _logits64(s, b, g, q, depth, s["k_new"][b, at, g], depth).masked_fill(~mask, -math.inf)
            x = torch.cat([old, new], -1)
            lse[b, at, g * n:(g + 1) * n] = torch.logsumexp(x, -1).t()
            p = torch.softmax(x, -1)
            values = torch.cat([s["v"][b, g, :end], s["v_new"][b, at, g]]).double()
            out[b, at, g * n:(g + 1) * n] = torch.stack([p[i] @ values for i in range(n)], 1)
    return out, lse


def _commit64(s):
    G = s["k"].shape[1]
    k, v, pos, score = s["k"].clone(), s["v"].clone(), s["pos"], s["score_out"].double()
    pos = None if pos is None else pos.clone()
    ends, nexts = [], []
    for b, nodes in enumerate(s["accepted"].tolist()):
        end, path = int(s["length"][b]), []
        for t in nodes:
            if t <= (path[-1] if path else -1) or t >= s["q"].shape[1] or end + len(path) >= k.shape[2]:
                break
            path.append(t)
        n, at = len(path), torch.tensor(path, device=DEV, dtype=torch.long)
        first = int(s["next_pos"][b]) if pos is not None else end
        qpos = first + torch.arange(n, device=DEV)
        ends.append(end + n)
        nexts.append(first + n)
        for g in range(G):
            k[b, g, end:end + n], v[b, g, end:end + n] = s["k_new"][b, at, g], s["v_new"][b, at, g]
            if pos is not None:
                pos[b, g, end:end + n] = qpos.to(torch.int32)
            kpos = pos[b, g, :end + n].long() if pos is not None else torch.arange(end + n, device=DEV)
            x = _logits64(s, b, g, s["q"][b, at], qpos, k[b, g, :end + n], kpos)
            x = x - s["lse"][b, at, g * x.shape[0]:(g + 1) * x.shape[0]].double().t()[..., None]
            late = torch.arange(end + n, device=DEV)[None] > end + torch.arange(n, device=DEV)[:, None]
            w = x.exp().masked_fill(late, 0.0).sum((0, 1))
            w[:end] += s["score"][b, g, :end].double()
            score[b, g, :end + n] = w
    whole = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return [k, v, pos, whole(ends), whole(nexts) if pos is not None else None, score]


def _evict64(s):
    m, G, C, d = s["k"].shape
    k, v = s["k"].clone(), s["v"].clone()
    score, pos = s["score_out"].double(), s["pos_out"].clone()
    scores, positions, ends = s["score"].cpu().numpy(), s["pos"].cpu().numpy(), []
    for b in range(m):
        end, first = int(s["length"][b]), int(s["next_pos"][b])
        keep = min(end, s["keep"])
        ends.append(keep)
        for g in range(G):
            p = positions[b, g, :end]
            fixed = (p >= first - s["recent"]) | (p < s["sinks"])
            order = np.lexsort((np.arange(end), -scores[b, g, :end].astype(np.float64), ~fixed))
            kept = np.zeros(end, dtype=bool)
            kept[order[:keep]] = True
            src = np.arange(keep)
            src[~kept[:keep]] = keep + np.flatnonzero(kept[keep:])
            at = torch.from_numpy(src).to(DEV)
            k[b, g, :keep], v[b, g, :keep] = s["k"][b, g, at], s["v"][b, g, at]
            score[b, g, :keep], pos[b, g, :keep] = s["score"][b, g, at].double(), s["pos"][b, g, at]
    return [k, v, torch.tensor(ends, dtype=torch.int32, device=DEV), score, pos]


def _q4_64(s):
    n, words = s["w"].shape
    k = words * 8
    group = k // s["scales"].shape[1]
    out = torch.empty((s["x"].shape[0], n), dtype=torch.float64, device=DEV)
    for lo in range(0, n, 4096):
        word = s["w"][lo:lo + 4096].long() & 0xFFFFFFFF
        w = torch.empty((word.shape[0], k), dtype=torch.float64, device=DEV)
        for i in range(8):
            w[:, i::8] = ((word >> (4 * i)) % 16).double()
        w = w * s["scales"][lo:lo + 4096].double().repeat_interleave(group, 1)
        w += s["biases"][lo:lo + 4096].double().repeat_interleave(group, 1)
        out[:, lo:lo + 4096] = s["x"].double() @ w.t()
    return out
