"""Attention of a drafted tree over a cache (mrt_tree_attention) against 64 bits.

Tolerances, per output, from the arithmetic: a logit is a sum of d exact products
(16-bit operands) or fp32 products in fp32, scaled, biased and shifted by the running
maximum, each step rounded to 2^-24 of a magnitude of at most `big`; exp2 is good to
2^-22; 16-bit weights are two-part (2^-17 of each for bf16, 2^-22 for fp16).  A weight's
relative error is then `delta`, the quotient's at most 2 delta plus the sums' own, and
the output's rounding is half a step of its type.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import mrt_df
from oracle import drafting_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SPLIT = {"bf16": 2.0 ** -17, "fp16": 2.0 ** -22, "fp32": 0.0}


def random_tree(rng, nodes):
    return [-1] + [t - 1 if rng.random() < 0.4 else int(rng.integers(-1, t)) for t in range(1, nodes)]


def make(seed, dtype, rows, heads, kv_heads, d, nodes, lengths, capacity=None, buckets=0, evicted=False):
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    cap = capacity or max(max(lengths), 1) + 3
    dt = DT[dtype]
    s = dict(q=torch.randn((rows, nodes, heads, d), generator=g).to(dt),
             k_new=torch.randn((rows, nodes, kv_heads, d), generator=g).to(dt),
             v_new=torch.randn((rows, nodes, kv_heads, d), generator=g).to(dt),
             k=torch.randn((rows, kv_heads, cap, d), generator=g).to(dt),
             v=torch.randn((rows, kv_heads, cap, d), generator=g).to(dt),
             length=torch.tensor(lengths, dtype=torch.int32),
             parents=torch.tensor([random_tree(rng, nodes) for _ in range(rows)], dtype=torch.int32),
             scale=1.5 / math.sqrt(d), bias=None, pos=None, next_pos=None)
    if buckets:
        s["bias"] = torch.randn((heads, buckets), generator=g)
    if evicted:
        pos = torch.randint(1, 4, (rows, kv_heads, cap), generator=g).cumsum(-1)
        s["pos"] = pos[:, :, torch.randperm(cap, generator=g)].to(torch.int32)
        s["next_pos"] = (pos.amax((1, 2)) + 1).to(torch.int32)
    return s


def on_gpu(s):
    return {n: x.to(DEV) if isinstance(x, torch.Tensor) else x for n, x in s.items()}


def call(s, **kw):
    d = on_gpu(s)
    cache = mrt_df.KVCache(d["k"], d["v"], d["length"], pos=d["pos"], next_pos=d["next_pos"])
    out, lse = mrt_df.tree_attention(d["q"], d["k_new"], d["v_new"], cache, d["parents"], scale=s["scale"],
                                     bias=d["bias"], **kw)
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


def oracle(s):
    return O.tree_attention(**{n: s[n] for n in ("q", "k_new", "v_new", "k", "v", "length", "parents", "scale", "bias",
                                                 "pos", "next_pos")})


def bounds(s, dtype):
    """(bound of an output beyond its own rounding, bound of lse)."""
    d = s["q"].shape[-1]
    N = s["k"].shape[2] + s["q"].shape[1]
    qn = s["q"].double().norm(dim=-1).max()
    kn = max(s["k"].double().nan_to_num(0, 0, 0).norm(dim=-1).max(), s["k_new"].double().nan_to_num(0, 0, 0).norm(dim=-1).max())
    big = float(s["scale"] * qn * kn) + (float(s["bias"].abs().max()) if s["bias"] is not None else 0.0)
    delta = (d + 8) * 2.0 ** -24 * big + 2.0 ** -21
    vmax = max(float(s["v"].double().nan_to_num(0, 0, 0).abs().max()), float(s["v_new"].double().nan_to_num(0, 0, 0).abs().max()))
    # sums of N terms in fp32, four waves and the splits joined: N 2^-24 of their magnitude
    return vmax * (2 * delta + SPLIT[dtype] + 2 * N * 2.0 ** -24), delta + N * 2.0 ** -24 + 2.0 ** -22 * (big + math.log(N))


def check(s, dtype, got):
    out, lse = got
    ref, rlse = oracle(s)
    tol, ltol = bounds(s, dtype)
    fin = torch.isfinite(ref)
    assert torch.equal(fin, torch.isfinite(out.double()))
    assert torch.equal(torch.isnan(ref), torch.isnan(out))
    err = (out.double() - ref).abs()[fin]
    lim = tol + torch.finfo(out.dtype).eps / 2 * (ref.abs()[fin] + tol)
    assert (err <= lim).all(), float((err / lim).max())
    there = torch.isfinite(rlse)
    assert torch.equal(there, torch.isfinite(lse))
    assert (lse.double() - rlse).abs()[there].max() <= ltol


CASES = [
    # rows heads kv d nodes lengths            what it is for
    (1, 1, 1, 64, 1, [0]),                     # nothing but the node itself
    (1, 1, 1, 64, 1, [1]),
    (2, 16, 16, 64, 1, [49, 50]),              # a decode step of a CFG pair
    (2, 16, 16, 64, 16, [0, 33]),              # one sequence without a cache
    (2, 4, 2, 64, 33, [1006, 31]),             # two node steps, rows in two tiles
    (1, 12, 12, 64, 64, [517]),                # the largest tree, four row tiles
    (3, 8, 1, 64, 64, [65, 64, 63]),           # 512 rows of one KV head
    (2, 8, 2, 128, 5, [2500, 700]),            # split keys, joined
    (2, 28, 4, 128, 9, [1500, 3000]),          # seven heads share a KV head
    (1, 4, 4, 128, 64, [4097]),
    (1, 2, 2, 8, 3, [40]),                     # the narrowest head
    (1, 3, 1, 24, 7, [100]),
    (2, 6, 2, 96, 5, [300, 90]),               # between the padded widths
    (1, 2, 1, 200, 20, [130]),
    (1, 8, 1, 256, 4, [777]),
    (5, 2, 1, 32, 2, [5, 0, 200, 32, 96]),
    (2, 8, 4, 64, 15, [900, 260]),             # 30 rows: two row tiles, four key groups
    (2, 8, 4, 128, 16, [900, 260]),
    (2, 4, 2, 64, 31, [900, 260]),             # 62 rows: four row tiles
    (2, 4, 2, 128, 20, [300, 1100]),
    (1, 16, 4, 64, 30, [513]),                 # 120 rows: eight
    (1, 8, 2, 128, 29, [1025]),
    (1, 12, 2, 64, 50, [333]),                 # 300 rows: two blocks of sixteen
    (2, 9, 1, 128, 33, [100, 640]),
    # work enough that parts are cut by equal shares, across sequences and heads
    # (where the caches have 32768 steps and less, as here, each unit is cut by itself; shared
    # out by all lengths: BIG below and test_gpu_tree_forms.py)
    (4, 16, 8, 64, 9, [7000, 5000, 31, 6200]),
    (3, 32, 16, 128, 17, [6000, 3333, 1]),
    (70, 8, 4, 64, 20, [700 + 13 * b for b in range(70)]),
    (2, 16, 2, 64, 20, [9000, 30000]),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=[f"r{c[0]}h{c[1]}kv{c[2]}d{c[3]}n{c[4]}l{max(c[5])}" for c in CASES])
def test_matches_oracle(case, dtype):
    s = make(3, dtype, *case)
    check(s, dtype, call(s))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("buckets,evicted", [(1, False), (16, False), (128, True), (2000, False), (9000, True)])
def test_bias_by_distance(dtype, buckets, evicted):
    s = make(5, dtype, 2, 6, 2, 64, 11, [300, 37], buckets=buckets, evicted=evicted)
    check(s, dtype, call(s))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_absent_nodes(dtype):
    s = make(7, dtype, 3, 4, 2, 64, 9, [100, 40, 0])
    s["parents"] = torch.tensor([[-1, 0, 5, 2, 1, -2, 5, -1, 9],      # 2 points ahead, 3 hangs on it, 5 is none, 6 on 5
                                 [-7, -1, 1, 2, 3, 4, 5, 6, 7],       # no first node, a chain
                                 [-5, -5, -5, -5, -5, -5, -5, -5, 8]], dtype=torch.int32)  # none at all; 8 its own parent
    out, lse = call(s)
    check(s, dtype, (out, lse))
    for b, t in ((0, 2), (0, 3), (0, 5), (0, 6), (0, 8), (1, 0), (2, 0), (2, 8)):
        assert (out[b, t] == 0).all() and (lse[b, t] == -math.inf).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d", [64, 128, 32])
def test_unseen_values_do_not_matter(dtype, d):
    """NaN and infinities in slots past the length, in absent nodes and in other branches."""
    s = make(11, dtype, 2, 4, 2, d, 40, [45, 3], capacity=70)
    s["parents"][:, 39] = -9
    s["parents"][:, 38] = 36  # keeps node 37 a leaf
    clean = call(s)
    check(s, dtype, clean)
    dirty = {n: x.clone() if isinstance(x, torch.Tensor) else x for n, x in s.items()}
    for b in range(2):
        L = int(s["length"][b])
        for x in (dirty["k"], dirty["v"]):
            x[b, :, L:] = math.nan
            x[b, :, L + 1] = math.inf
        for x in (dirty["k_new"], dirty["v_new"]):
            x[b, 39] = math.nan
            x[b, 37, :, ::2] = math.inf
            x[b, 37, :, 1::4] = -math.inf
            x[b, 37, :, 3] = math.nan
    got = call(dirty)
    others = [t for t in range(40) if t != 37]
    assert torch.equal(got[0][:, others], clean[0][:, others])
    assert torch.equal(got[1][:, others], clean[1][:, others])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_seen_infinities_stay(dtype):
    """An infinite or NaN value of an ancestor reaches its descendants as itself."""
    s = make(13, dtype, 1, 2, 1, 64, 6, [20])
    s["parents"] = torch.tensor([[-1, 0, 0, 1, 2, -1]], dtype=torch.int32)
    s["v_new"][0, 1, 0, 5] = math.inf
    s["v_new"][0, 2, 0, 5] = -math.inf
    s["v_new"][0, 2, 0, 7] = math.nan
    out, lse = call(s)
    check(s, dtype, (out, lse))
    assert (out[0, 3, :, 5] == math.inf).all() and (out[0, 4, :, 5] == -math.inf).all()
    assert torch.isnan(out[0, 4, :, 7]).all() and torch.isfinite(out[0, 5]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strides_and_one_tree(dtype):
    """Operands as views: heads before nodes, slots of a larger cache, one parents row."""
    s = make(17, dtype, 2, 4, 2, 64, 7, [90, 33])
    s["parents"] = s["parents"][:1].expand(2, -1).contiguous()
    ref = call(s)
    check(s, dtype, ref)
    d = on_gpu(s)
    big = torch.zeros((3, 2, 200, 2, 64), dtype=DT[dtype], device=DEV)
    kk, vv = big[:2, :, 10:10 + d["k"].shape[2], 0], big[:2, :, 10:10 + d["k"].shape[2], 1]
    kk.copy_(d["k"]), vv.copy_(d["v"])
    q = d["q"].transpose(1, 2).contiguous().transpose(1, 2)
    kv = torch.stack([d["k_new"], d["v_new"]], 3)
    out = torch.zeros((2, 7, 6, 64), dtype=DT[dtype], device=DEV)[:, :, 1:5]
    got, lse = mrt_df.tree_attention(q, kv[..., 0, :], kv[..., 1, :], mrt_df.KVCache(kk, vv, d["length"]),
                                     d["parents"][0].contiguous(), scale=s["scale"], out=out)
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(got.cpu(), ref[0]) and torch.equal(lse.cpu(), ref[1])


def test_repeats_and_graph_replays():
    """Bit-equal from call to call, on another stream and from a captured graph."""
    s = make(19, "bf16", 3, 8, 2, 128, 12, [5000, 100, 2600])
    want = call(s)
    check(s, "bf16", want)
    d = on_gpu(s)
    cache = mrt_df.KVCache(d["k"], d["v"], d["length"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o, l = mrt_df.tree_attention(d["q"], d["k_new"], d["v_new"], cache, d["parents"], scale=s["scale"])
    side.synchronize()
    assert torch.equal(o.cpu(), want[0]) and torch.equal(l.cpu(), want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, l = mrt_df.tree_attention(d["q"], d["k_new"], d["v_new"], cache, d["parents"], scale=s["scale"])
    for _ in range(3):
        o.zero_(), l.zero_()
        graph.replay()
        eager, _ = mrt_df.tree_attention(d["q"], d["k_new"], d["v_new"], cache, d["parents"], scale=s["scale"])
        torch.cuda.synchronize()
        assert torch.equal(o.cpu(), want[0]) and torch.equal(l.cpu(), want[1]) and torch.equal(eager.cpu(), want[0])


def test_length_changes_under_a_graph():
    """The length is read on the device: a captured step serves the cache as it grows."""
    s = make(23, "bf16", 2, 2, 2, 64, 3, [10, 700], capacity=1500)
    d = on_gpu(s)
    cache = mrt_df.KVCache(d["k"], d["v"], d["length"])
    graph = torch.cuda.CUDAGraph()
    mrt_df.tree_attention(d["q"], d["k_new"], d["v_new"], cache, d["parents"], scale=s["scale"])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        o, l = mrt_df.tree_attention(d["q"], d["k_new"], d["v_new"], cache, d["parents"], scale=s["scale"])
    for lengths in ([10, 700], [1500, 0], [-3, 4000], [64, 1499]):
        d["length"].copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check({**s, "length": torch.tensor(lengths, dtype=torch.int32)}, "bf16", (o.cpu(), l.cpu()))


def test_long_cache_offsets():
    """Slots past 2^31 elements from the start of the cache."""
    rows, cap, d = 3, 3_000_000, 256
    k = torch.zeros((rows, 1, cap, d), dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    lengths = [5, 0, cap]
    g = torch.Generator().manual_seed(1)
    tail = torch.randn((2, 40, d), generator=g).to(torch.bfloat16)
    q = (torch.randn((rows, 2, 2, d), generator=g)).to(torch.bfloat16)
    kn, vn = torch.randn((2, rows, 2, 1, d), generator=g).to(torch.bfloat16)
    k[2, 0, -40:], v[2, 0, -40:] = tail[0].to(DEV), tail[1].to(DEV)
    out, lse = mrt_df.tree_attention(q.to(DEV), kn.to(DEV), vn.to(DEV),
                                     mrt_df.KVCache(k, v, torch.tensor(lengths, dtype=torch.int32, device=DEV)),
                                     torch.tensor([[-1, 0]] * 3, dtype=torch.int32, device=DEV), scale=0.1)
    # row 2: cap - 40 entries with logit 0 and value 0, then the tail
    keys = torch.cat([tail[0], kn[2, :, 0]]).double()
    vals = torch.cat([tail[1], vn[2, :, 0]]).double()
    for t in range(2):
        x = 0.1 * (q[2, t].double() @ keys[:40 + t + 1].T)
        e = x.exp()
        total = e.sum(1) + (cap - 40)
        assert (lse[2, t].cpu().double() - total.log()).abs().max() < 1e-4
        ref = (e @ vals[:40 + t + 1]) / total[:, None]
        assert (out[2, t].cpu().double() - ref).norm() <= 5e-3 * ref.norm()


@pytest.mark.parametrize("masked", [-math.inf, float(torch.finfo(torch.float32).min)], ids=["inf", "lowest"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("nodes,heads,lengths", [(4, 4, [40, 3]), (33, 4, [40, 3]), (9, 8, [3000, 5000]), (40, 8, [9000, 0])])
def test_masks_in_the_bias(nodes, heads, lengths, dtype, masked):
    """Distances of 5 and more are masked for one head, all of them for another: what is
    left is as if the rest were not there, and a row with nothing left is 0, its lse -inf."""
    s = make(41, dtype, 2, heads, 2, 64, nodes, lengths, buckets=8)
    plain = s["bias"].clone()
    s["bias"][0, 5:], s["bias"][1] = -math.inf, -math.inf
    ref, rlse = oracle(s)
    out, lse = call(dict(s, bias=s["bias"].clamp(min=masked)))
    assert (out[:, :, 1] == 0).all() and (lse[:, :, 1] == -math.inf).all()
    tol, ltol = bounds(dict(s, bias=plain), dtype)
    rest = [h for h in range(heads) if h != 1]
    err = (out.double() - ref).abs()[:, :, rest]
    assert (err <= tol + torch.finfo(out.dtype).eps / 2 * (ref.abs()[:, :, rest] + tol)).all()
    assert ((lse.double() - rlse).abs()[:, :, rest] <= ltol).all()


BIG = [
    # rows heads kv d nodes capacity lengths   work that is shared out by all lengths
    (4, 4, 4, 64, 17, 70000, [60000, 0, 100, 9000]),               # cut anywhere, whole sequences in one part
    (4, 4, 4, 64, 17, 70000, [900, 0, 100, 3]),                    # far less than the caches hold
    (17, 8, 1, 64, 9, 63000, [50000, 3, 50000, 1, 50000] + [40 * i for i in range(12)]),  # halves, 72 rows
    (4, 4, 4, 64, 1, 140000, [60000, 0, 100, 9000]),               # few rows
    (4, 4, 4, 64, 1, 140000, [900, 0, 100, 3]),
    (300, 4, 1, 64, 5, 4000, [(37 * i) % 700 for i in range(299)] + [4000]),   # more sequences than blocks at a time
    (300, 1, 1, 64, 1, 4000, [(37 * i) % 700 for i in range(299)] + [4000]),
]


@pytest.mark.parametrize("case", BIG, ids=[f"r{c[0]}h{c[1]}n{c[4]}l{max(c[6])}" for c in BIG])
def test_work_shared_out_by_lengths(case):
    rows, heads, kv, d, nodes, cap, lengths = case
    s = make(43, "bf16", rows, heads, kv, d, nodes, lengths, capacity=cap)
    got = call(s)
    check(s, "bf16", got)
    again = call(s)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
