"""Serving operators over paged caches and 8-bit integers: their cases, plain forms and 64-bit values.

Together a server's step of drafting decode: products in 8-bit integers
(``i8_quantize``, ``i8_matmul``), new entries quantised into the pages of a cache
and read back (``paged_write``, ``paged_read``), the attention of new tokens
over the pages (``paged_attention``), and the verification of drafted tokens
against the target's probabilities (``draft_verify``).

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges,
``prepare`` makes a case's inputs, ``run`` is one pass, ``work`` counts what a
pass cannot do without and ``exact`` evaluates a case in 64 bits.  With ``own``
false ``run`` computes in elementary torch operations, in 32 bits; the sums over
a vocabulary that a drawn token depends on in 64.
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
STEP = float(np.float32(1) / np.float32(127))  # a scale is its vector's largest magnitude times this, in fp32


@functools.lru_cache(maxsize=None)
def _package():
    pkg = str(pathlib.Path(__file__).resolve().parents[1] / "magenta-realtime-mlx-cpp_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import mrt_df
    return mrt_df


# ---------------------------------------------------------------------------
# The cases.  rows: sequences (a CFG pair is two).  tokens: new tokens of a
# sequence.  length: entries before them of the longest sequence; ragged: the
# others hold fewer, and some bring fewer new tokens, or none.  i8: pages hold 8-bit
# codes with a scale for each entry and head, else values of the type.  buckets:
# columns of the bias by distance (0: none).


def listed():
    return [
        # One token of one live stream against its frame cache: the smallest call, all latency.
        dict(name="attn_step", op="attention", dtype="bf16", i8=False, rows=2, heads=16, kv_heads=16, d=64, tokens=1,
             length=49, page=16, buckets=128, ragged=False),
        # 32 live streams, a 10 s context each, in 8 bits, with the model's bias by distance.
        dict(name="attn_streams", op="attention", dtype="fp16", i8=True, rows=64, heads=16, kv_heads=16, d=64, tokens=1,
             length=1005, page=64, buckets=128, ragged=False),
        # The 12-head configuration in fp32 over 8-bit pages, a few drafted tokens.
        dict(name="attn_fp32", op="attention", dtype="fp32", i8=True, rows=4, heads=12, kv_heads=12, d=64, tokens=3,
             length=4099, page=32, buckets=128, ragged=True),
        # A server's batch over pages in the model's type, heads shared.
        dict(name="attn_serve", op="attention", dtype="bf16", i8=False, rows=48, heads=32, kv_heads=8, d=128, tokens=1,
             length=8191, page=16, buckets=0, ragged=True),
        # Few sequences with very long caches in 8 bits, a chain of drafts each.
        dict(name="attn_long", op="attention", dtype="bf16", i8=True, rows=3, heads=32, kv_heads=8, d=128, tokens=4,
             length=131000, page=128, buckets=0, ragged=True),
        # One token of each sequence of a batch into its page, and back as the values that it stands for.
        dict(name="store_step", op="store", dtype="bf16", i8=True, rows=64, kv_heads=8, d=128, tokens=1, length=1000,
             page=16, ragged=True),
        # Whole prompts into pages, and back.
        dict(name="store_prompt", op="store", dtype="fp16", i8=True, rows=16, kv_heads=8, d=128, tokens=4001, length=0,
             page=64, ragged=False),
        # A frame's 16 levels drafted as a chain over one codebook, a CFG pair's stream and another: latency.
        dict(name="verify_frame", op="verify", dtype="fp32", rows=2, tokens=16, vocab=1024, tree=False, sure=False),
        # A batch of trees over a large vocabulary.
        dict(name="verify_trees", op="verify", dtype="fp32", rows=16, tokens=31, vocab=131072, tree=True, sure=False),
        # The smallest product: one CFG pair through a gate and up projection.
        dict(name="i8_step", op="i8", dtype="bf16", rows=2, k=1024, n=5632, add=False),
        # The verifying pass of 32 streams' drafted frames through a down projection, onto the residual.
        dict(name="i8_verify", op="i8", dtype="fp16", rows=512, k=2816, n=1024, add=True),
        # A prompt's tokens through a large layer.
        dict(name="i8_large", op="i8", dtype="bf16", rows=8192, k=8192, n=8192, add=False),
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
    op = rng.choice(["attention", "attention", "attention", "store", "verify", "i8", "i8"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "i8":
        return dict(op=op, dtype=dtype, rows=_log_int(rng, 1, 8192), k=16 * _log_int(rng, 1, 512), n=_log_int(rng, 1, 30000),
                    add=rng.random() < 0.4)
    if op == "verify":
        tree = rng.random() < 0.5
        c = dict(op=op, dtype=dtype, rows=_log_int(rng, 1, 64), tokens=_log_int(rng, 1, 63 if tree else 16),
                 vocab=_log_int(rng, 2, 131072), tree=tree, sure=rng.random() < 0.3)
        return c if c["rows"] * (c["tokens"] + 1) * c["vocab"] <= 16 * 32 * 131072 else _draw(rng)
    heads, kv_heads, d = rng.choice(HEADS)
    c = dict(op=op, dtype=dtype, i8=rng.random() < 0.6, rows=_log_int(rng, 1, 64), heads=heads, kv_heads=kv_heads, d=d,
             length=_log_int(rng, 1, 132000) - 1, page=rng.choice([16, 16, 32, 48, 64, 128, 256]), ragged=rng.random() < 0.5)
    if op == "store":
        return dict(c, tokens=_log_int(rng, 1, 4096))
    return dict(c, tokens=_log_int(rng, 1, 16), buckets=rng.choice([0, 0, 16, 128, 1000]))


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 4e12, w["flops"] / 1e15)


def work(case):
    e, m = BYTES[case["dtype"]], case["rows"]
    if case["op"] == "i8":
        k, n = case["k"], case["n"]
        return {"bytes": n * (k + 4) + m * (k + (2 if case["add"] else 1) * n) * e, "flops": 2 * m * n * k}
    if case["op"] == "verify":
        T, V = case["tokens"], case["vocab"]
        # the distributions that the last token is drawn from, and each node's own probabilities
        return {"bytes": m * (V * e * (1 if case["sure"] else 2) + T * (2 * e + 12) + 12), "flops": 0}
    G, d = case["kv_heads"], case["d"]
    entry = G * (d + 4 if case["i8"] else d * e)  # of K, or of V
    fresh, lengths = _fresh(case), _lengths(case)
    new = sum(fresh)
    if case["op"] == "store":  # written, and read back
        return {"bytes": 2 * new * (2 * G * d * e + 2 * entry) + 8 * m, "flops": 0}
    H, T = case["heads"], case["tokens"]
    total = sum(n + f for n, f in zip(lengths, fresh) if f > 0)
    return {"bytes": 2 * total * entry + 2 * m * T * H * d * e + 4 * m * T * H + 4 * H * case["buckets"],
            "flops": sum(4 * f * (n + (f + 1) / 2) * H * d for n, f in zip(lengths, fresh))}


def _lengths(case):
    """Entries in use of each sequence: equal, or spread from the whole length down to a seventh of it."""
    L, m = case["length"], case["rows"]
    return [L - (L - L // 7) * b // max(1, m - 1) if case["ragged"] else L for b in range(m)]


def _fresh(case):
    """New tokens of each sequence: all, or in a ragged batch of several each fewer ones by turns, every seventh none."""
    T, m = case["tokens"], case["rows"]
    if not case["ragged"]:
        return [T] * m
    return [0 if b % 7 == 6 else max(1, T - T * (b % 3) // 4) for b in range(m)]


# ---------------------------------------------------------------------------
# Inputs


def _quantised(x):
    """8-bit codes of the last dimension's vectors, and their scales."""
    scale = x.abs().amax(-1).float() * STEP
    return (x.float() / scale[..., None]).round().to(torch.int8), scale


def prepare(case, seed):
    rng = np.random.RandomState(seed & 0x7FFFFFFF)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = TORCH[case["dtype"]]

    def normal(*shape, scale=1.0, to=dt):
        return torch.empty(shape, device=DEV, dtype=to).normal_(0.0, scale, generator=g)

    def ints(v):
        return torch.from_numpy(np.ascontiguousarray(v, dtype=np.int32)).to(DEV)

    s = dict(op=case["op"], dtype=dt)
    m = case["rows"]
    if case["op"] == "i8":
        k, n = case["k"], case["n"]
        # a few channels far above the others, as activations of trained models have
        x = normal(m, k, to=torch.float32) * (1 + 10 * (torch.rand(k, device=DEV, generator=g) < 0.01))
        s.update(x=x.to(dt), add=normal(m, n) if case["add"] else None)
        s["w"], s["w_scale"] = _quantised(normal(n, k, scale=1 / math.sqrt(k), to=torch.float32))
        return s
    if case["op"] == "verify":
        return _prepare_verify(case, s, rng, g, dt)
    G, d, T, page = case["kv_heads"], case["d"], case["tokens"], case["page"]
    lengths, fresh = _lengths(case), _fresh(case)
    need = [-(-(n + T) // page) for n in lengths]
    per_row, pages = max(need) + 1, sum(need) + 3
    table, order, at = np.full((m, per_row), -1), rng.permutation(pages), 0
    for b, n in enumerate(need):  # pages of the pool in no order; no page behind a sequence's last
        table[b, :n], at = order[at:at + n], at + n
    # a page that no sequence has: what the plain form writes for tokens that are not there goes there
    s.update(spare=int(order[-1]), table=ints(table), length=ints(lengths), fresh=ints(fresh) if case["ragged"] else None, k_scale=None, v_scale=None)
    for x in "kv":
        pool = normal(pages, G, page, d)
        if case["i8"]:
            pool, s[x + "_scale"] = _quantised(pool)
        s[x] = pool
    if case["op"] == "store":
        s.update(k_new=normal(m, T, G, d), v_new=normal(m, T, G, d), length_out=torch.zeros_like(s["length"]),
                 k_out=torch.zeros((m, G, T, d), dtype=dt, device=DEV), v_out=torch.zeros((m, G, T, d), dtype=dt, device=DEV))
        return s
    s.update(q=normal(m, T, case["heads"], d, scale=1.5), scale=1 / math.sqrt(d), bias=None)
    if case["buckets"]:
        s["bias"] = normal(case["heads"], case["buckets"], to=torch.float32)
    return s


def _prepare_verify(case, s, rng, g, dt):
    m, T, V = case["rows"], case["tokens"], case["vocab"]
    if case["tree"]:  # half of the nodes extend the newest branch, the others branch anywhere
        parents = [[-1] + [t - 1 if rng.rand() < 0.5 else int(rng.randint(-1, t)) for t in range(1, T)] for _ in range(m)]
    else:
        parents = [list(range(-1, T - 1))] * m
    s["parents"] = torch.tensor(parents, dtype=torch.int32, device=DEV) if case["tree"] else None
    # a draft that is near the target: the same logits and noise on both
    logits = torch.empty((m, T + 1, V), device=DEV).normal_(0.0, 2.5, generator=g)
    target = (logits + torch.empty_like(logits).normal_(0.0, 0.5, generator=g)).softmax(-1)
    draft = logits[:, :T].softmax(-1)
    slot = torch.tensor(parents, device=DEV) + 1
    if case["sure"]:  # drafts that were not drawn: the draft's likeliest, the next for the next child
        tokens = torch.zeros((m, T), dtype=torch.int32, device=DEV)
        for b in range(m):
            seen = {}
            for t, p in enumerate(parents[b]):
                seen.setdefault(p, []).append(t)
            for p, kids in seen.items():
                best = draft[b, p + 1].topk(min(len(kids), V)).indices.to(torch.int32)
                tokens[b, kids] = best[torch.arange(len(kids), device=DEV) % len(best)]
        draft = None
    else:
        rows = draft.gather(1, slot[..., None].expand(m, T, V)).reshape(m * T, V)
        tokens = torch.multinomial(rows, 1, generator=g).view(m, T).to(torch.int32)
        del rows
    s.update(target=target.to(dt), draft=None if draft is None else draft.to(dt), tokens=tokens,
             uniforms=torch.rand((m, T + 1), device=DEV, generator=g))
    return s


# ---------------------------------------------------------------------------
# One pass


def run(s):
    if own:
        return _run_own(s)
    return {"attention": _attention, "store": _store, "verify": _verify, "i8": _i8}[s["op"]](s)


def _run_own(s):
    mrt_df = _package()
    if s["op"] == "i8":
        codes, scale = mrt_df.i8_quantize(s["x"])
        return mrt_df.i8_matmul(codes, scale, s["w"], s["w_scale"], dtype=s["dtype"], add=s["add"])
    if s["op"] == "verify":
        return mrt_df.draft_verify(s["target"], s["draft"], s["tokens"], s["uniforms"], parents=s["parents"])
    cache = mrt_df.PagedCache(s["k"], s["v"], s["table"], s["length"], s["k_scale"], s["v_scale"])
    if s["op"] == "attention":
        return mrt_df.paged_attention(s["q"], cache, fresh=s["fresh"], scale=s["scale"], bias=s["bias"])
    mrt_df.paged_write(cache, s["k_new"], s["v_new"], fresh=s["fresh"], length_out=s["length_out"])
    grown = mrt_df.PagedCache(s["k"], s["v"], s["table"], s["length_out"], s["k_scale"], s["v_scale"])
    mrt_df.paged_read(grown, s["k_out"], s["v_out"], start=s["length"])
    return [s["k_out"], s["v_out"], s["length_out"], s["k_scale"], s["v_scale"]]


def _counts(s, T):
    m = s["length"].shape[0]
    return s["fresh"].long() if s["fresh"] is not None else torch.full((m,), T, dtype=torch.long, device=DEV)


def _gathered(s, x):
    """(rows, kv_heads, capacity, d) fp32 values of each sequence's pages; what absent pages give is masked later."""
    pool, at = s[x], s["table"].clamp_min(0).long()
    got = pool[at].float()
    if s[x + "_scale"] is not None:
        got = got * s[x + "_scale"][at][..., None]
    m, n, G, page, d = got.shape
    return got.transpose(1, 2).reshape(m, G, n * page, d)


def _attention(s):
    q = s["q"].float()
    m, T, H, d = q.shape
    k, v = _gathered(s, "k"), _gathered(s, "v")
    G, C = k.shape[1], k.shape[2]
    q = q.transpose(1, 2).reshape(m, G, H // G * T, d)
    x = (q @ k.transpose(-1, -2).contiguous()).view(m, H, T, C) * s["scale"]
    at = s["length"].long()[:, None] + torch.arange(T, device=DEV)  # the slot of each new token
    slot = torch.arange(C, device=DEV)
    if s["bias"] is not None:
        far = (at[..., None] - slot).clamp(0, s["bias"].shape[1] - 1)
        x = x + s["bias"][:, far].transpose(0, 1)
    seen = (slot <= at[..., None]) & (torch.arange(T, device=DEV) < _counts(s, T)[:, None])[..., None]
    x = x.masked_fill(~seen[:, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp_min(-3e38)
    x = (x - top).exp_()
    total = x.sum(-1, keepdim=True)
    out = (x.view(m, G, H // G * T, C) @ v).view(m, H, T, d) / torch.where(total > 0, total, 1.0)
    lse = torch.where(total > 0, top + total.log(), -math.inf)
    return out.transpose(1, 2).to(s["q"].dtype).contiguous(), lse[..., 0].transpose(1, 2).contiguous()


def _store(s):
    m, T, G, d = s["k_new"].shape
    page, C = s["k"].shape[2], s["table"].shape[1] * s["k"].shape[2]
    count = torch.minimum(_counts(s, T), C - s["length"].long())
    at = s["length"].long()[:, None] + torch.arange(T, device=DEV)
    there = torch.arange(T, device=DEV) < count[:, None]
    row = torch.arange(m, device=DEV)[:, None]
    where = torch.where(there, s["table"][row, (at // page).clamp(max=s["table"].shape[1] - 1)].long(), s["spare"])
    slot, there = at % page, there[..., None, None]
    for x in "kv":
        new = s[x + "_new"]
        if s[x + "_scale"] is not None:
            scale = new.float().abs().amax(-1) * STEP
            codes = torch.where(scale[..., None] > 0, new.float() / scale[..., None], 0.0).round().to(torch.int8)
            s[x][where, :, slot] = torch.where(there, codes, s[x][where, :, slot])
            s[x + "_scale"][where, :, slot] = torch.where(there[..., 0], scale, s[x + "_scale"][where, :, slot])
            back = s[x][where, :, slot].float() * s[x + "_scale"][where, :, slot][..., None]
        else:
            s[x][where, :, slot] = torch.where(there, new, s[x][where, :, slot])
            back = s[x][where, :, slot]
        out = s[x + "_out"].transpose(1, 2)
        out.copy_(torch.where(there, back.to(out.dtype), out))
    s["length_out"].copy_(s["length"] + count)
    return [s["k_out"], s["v_out"], s["length_out"], s["k_scale"], s["v_scale"]]


def _verify(s):
    target, draft, tokens, u = s["target"], s["draft"], s["tokens"].long(), s["uniforms"].double()
    m, T = tokens.shape
    row = torch.arange(m, device=DEV)
    parents = s["parents"].long() if s["parents"] is not None else torch.arange(-1, T - 1, device=DEV).expand(m, T)
    here = torch.zeros(m, dtype=torch.long, device=DEV)  # the slot reached: 0 the root, t + 1 node t
    left, size = target[:, 0].double(), torch.ones(m, dtype=torch.float64, device=DEV)
    accepted = torch.zeros((m, T), dtype=torch.bool, device=DEV)
    for t in range(T):
        mine, x = parents[:, t] + 1 == here, tokens[:, t]
        q = draft[row, here.clamp(max=T - 1)].double() if draft is not None else None
        good = mine & (u[:, t] * size * (q[row, x] if q is not None else 1.0) < left[row, x])
        if q is not None:
            rest = (left - size[:, None] * q).clamp_min(0.0)
            rest_size = rest.sum(-1)
        else:
            rest = left.scatter(1, x[:, None], 0.0)
            rest_size = size - left[row, x]
        bad = mine & ~good
        left = torch.where(good[:, None], target[:, t + 1].double(), torch.where(bad[:, None], rest, left))
        size = torch.where(good, 1.0, torch.where(bad, rest_size, size))
        here = torch.where(good, t + 1, here)
        accepted[:, t] = good
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, target[row, here].double())
    total = left.cumsum(-1)
    token = (total <= u[:, T:] * total[:, -1:]).sum(-1)
    order = torch.where(accepted, torch.arange(T, device=DEV), T).sort(-1).values
    path = torch.where(order < T, order, -1)
    return path.to(torch.int32), accepted.sum(-1).to(torch.int32), token.to(torch.int32)


def _i8(s):
    x = s["x"].float()
    scale = x.abs().amax(-1) * STEP
    codes = torch.where(scale[:, None] > 0, x / scale[:, None], 0.0).round()
    y = (codes @ s["w"].float().t().contiguous()) * scale[:, None] * s["w_scale"]
    if s["add"] is not None:
        y = y + s["add"].float()
    return y.to(s["x"].dtype)


# ---------------------------------------------------------------------------
# 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _attention64, "store": _store64, "verify": _verify64, "i8": _i8_64}[case["op"]](s)


def _entries(s, x, b, g, end):
    """The first `end` entries of sequence b, head g, in 64 bits."""
    page = s[x].shape[2]
    at = s["table"][b, :-(-end // page)].long()
    got = s[x][at, g].double()
    if s[x + "_scale"] is not None:
        got = got * s[x + "_scale"][at, g].double()[..., None]
    return got.reshape(-1, s[x].shape[3])[:end]


def _attention64(s):
    m, T, H, d = s["q"].shape
    G = s["k"].shape[1]
    n = H // G
    out = torch.zeros((m, T, H, d), dtype=torch.float64, device=DEV)
    lse = torch.full((m, T, H), -math.inf, dtype=torch.float64, device=DEV)
    fresh = s["fresh"].tolist() if s["fresh"] is not None else [T] * m
    for b, length in enumerate(s["length"].tolist()):
        new = fresh[b]
        if new == 0:
            continue
        end = length + new
        qpos, kpos = torch.arange(length, end, device=DEV)[:, None], torch.arange(end, device=DEV)
        late = kpos > qpos
        for g in range(G):
            keys, values = _entries(s, "k", b, g, end), _entries(s, "v", b, g, end)
            for h in range(g * n, (g + 1) * n):
                x = s["q"][b, :new, h].double() @ keys.t() * s["scale"]
                if s["bias"] is not None:
                    x = x + s["bias"][h].double()[(qpos - kpos).clamp(0, s["bias"].shape[1] - 1)]
                x = x.masked_fill(late, -math.inf)
                lse[b, :new, h] = torch.logsumexp(x, -1)
                out[b, :new, h] = torch.softmax(x, -1) @ values
    return out, lse


def _store64(s):
    """Scales are fp32 products by definition, codes the fp32 quotients rounded to whole numbers; the values are their products."""
    m, T, G, d = s["k_new"].shape
    page = s["k"].shape[2]
    fresh = s["fresh"].tolist() if s["fresh"] is not None else [T] * m
    lengths = s["length"].tolist()
    table = s["table"].cpu().numpy()
    got = []
    for x in "kv":
        out = s[x + "_out"].double()
        scales = None if s[x + "_scale"] is None else s[x + "_scale"].clone()
        for b in range(m):
            n = fresh[b]
            new = s[x + "_new"][b, :n].double()
            if scales is not None:
                scale = (new.abs().amax(-1) * STEP).float()
                codes = (new / scale.double()[..., None]).float().round().double()
                codes = torch.where(scale[..., None] > 0, codes, 0.0)
                new = codes * scale.double()[..., None]
                at = np.arange(lengths[b], lengths[b] + n)
                where = torch.from_numpy(table[b, at // page]).long().to(DEV)
                scales[where, :, torch.from_numpy(at % page).to(DEV)] = scale
            out[b, :, :n] = new.transpose(0, 1)
        got.append((out, scales))
    length = torch.tensor([n + f for n, f in zip(lengths, fresh)], dtype=torch.int32, device=DEV)
    return [got[0][0], got[1][0], length, got[0][1], got[1][1]]


def _verify64(s):
    m, T = s["tokens"].shape
    tokens, u = s["tokens"].tolist(), s["uniforms"].double().tolist()
    parents = s["parents"].tolist() if s["parents"] is not None else [list(range(-1, T - 1))] * m
    paths, counts, last = [], [], []
    for b in range(m):
        node, path = -1, []
        while True:
            p = s["target"][b, node + 1].double()
            kids = [t for t in range(T) if parents[b][t] == node]
            q = s["draft"][b, node + 1].double() if s["draft"] is not None and kids else None
            rest, size, took = p.clone(), 1.0, None
            for t in kids:
                x = tokens[b][t]
                if u[b][t] * size * (float(q[x]) if q is not None else 1.0) < float(rest[x]):
                    took = t
                    break
                if q is not None:
                    rest = torch.relu(rest - size * q)
                    size = float(rest.sum())
                else:
                    size -= float(rest[x])
                    rest[x] = 0.0
            if took is None:
                break
            node = took
            path.append(took)
        weights = (rest if float(rest.sum()) > 0 else p).cpu().numpy()
        run_sum = np.cumsum(weights)
        last.append(int(np.searchsorted(run_sum, u[b][T] * run_sum[-1], side="right")))
        paths.append(path + [-1] * (T - len(path)))
        counts.append(len(path))
    whole = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return whole(paths), whole(counts), whole(last)


def _i8_64(s):
    x = s["x"].double()
    scale = (x.abs().amax(-1) * STEP).float().double()
    codes = torch.where(scale[:, None] > 0, (x / scale[:, None]).float().round().double(), 0.0)
    y = torch.empty((x.shape[0], s["w"].shape[0]), dtype=torch.float64, device=DEV)
    for lo in range(0, y.shape[1], 4096):
        y[:, lo:lo + 4096] = codes @ s["w"][lo:lo + 4096].double().t().contiguous()
    y = y * scale[:, None] * s["w_scale"].double()
    return y if s["add"] is None else y + s["add"].double()
