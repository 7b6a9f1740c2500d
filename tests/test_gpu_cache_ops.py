"""Commit of accepted paths and eviction by attention weight against 64 bits.

What is moved is compared bit for bit, lengths, positions and choices exactly.  A
score's tolerance: each weight exp(logit - lse) carries the logit's error (d + 8
roundings of 2^-24 of its largest magnitude `big`, and lse's own 2^-24 |lse|) and
exp2's 2^-22; a score sums them and the old score in fp32, N terms of 2^-24 each.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import mrt_df
from oracle import drafting_oracle as O
from test_gpu_tree_attention import DEV, DT, make, on_gpu

pytestmark = pytest.mark.gpu


def make_commit(seed, dtype, rows, heads, kv_heads, d, nodes, lengths, accepted, capacity=None, buckets=0, evicted=False,
                old_scores=True):
    s = make(seed, dtype, rows, heads, kv_heads, d, nodes, lengths, capacity or max(lengths) + nodes, buckets, evicted)
    g = torch.Generator().manual_seed(seed + 1)
    width = max(len(a) for a in accepted)
    s["accepted"] = torch.tensor([list(a) + [-1] * (width - len(a)) for a in accepted], dtype=torch.int32)
    s["lse"] = O.tree_attention(**{n: s[n] for n in ("q", "k_new", "v_new", "k", "v", "length", "parents", "scale", "bias",
                                                     "pos", "next_pos")})[1].float()
    slots = s["k"].shape[:3]
    s["score"] = torch.rand(slots, generator=g) * 4 if old_scores else None
    s["score_out"] = torch.full(slots, -7.0)
    return s


def commit(s, weights=True):
    d = on_gpu(s)
    cache = mrt_df.KVCache(d["k"], d["v"], d["length"], pos=d["pos"], next_pos=d["next_pos"], score=d["score"])
    length_out = torch.full_like(d["length"], -1)
    next_out = torch.full_like(d["length"], -1) if d["pos"] is not None else None
    kw = dict(q=d["q"], lse=d["lse"], score_out=d["score_out"], scale=s["scale"], bias=d["bias"]) if weights else {}
    mrt_df.cache_commit(cache, d["k_new"], d["v_new"], d["accepted"], length_out, next_out=next_out, **kw)
    torch.cuda.synchronize()
    back = lambda x: None if x is None else x.cpu()  # noqa: E731
    return dict(k=d["k"].cpu(), v=d["v"].cpu(), pos=back(d["pos"]), length=length_out.cpu(), next_pos=back(next_out),
                score=d["score_out"].cpu())


def check_commit(s, got, weights=True):
    kw = dict(q=s["q"], lse=s["lse"], score=s["score"], score_out=s["score_out"], scale=s["scale"], bias=s["bias"]) if weights else {}
    ref = O.cache_commit(s["k"], s["v"], s["length"], s["k_new"], s["v_new"], s["accepted"], pos=s["pos"],
                         next_pos=s["next_pos"], **kw)
    same = lambda a, b: torch.equal(a.nan_to_num(11), b.nan_to_num(11))  # noqa: E731
    assert same(got["k"], ref["k"]) and same(got["v"], ref["v"])
    assert torch.equal(got["length"], ref["length"])
    if s["pos"] is not None:
        assert torch.equal(got["pos"], ref["pos"]) and torch.equal(got["next_pos"], ref["next_pos"])
    if not weights:
        return
    d = s["q"].shape[-1]
    N = s["accepted"].shape[1] * (s["q"].shape[2] // s["k"].shape[1]) + 1
    fin = lambda x: x.double().nan_to_num(0, 0, 0)  # noqa: E731
    big = float(s["scale"] * fin(s["q"]).norm(dim=-1).max() * max(fin(s["k"]).norm(dim=-1).max(), fin(s["k_new"]).norm(dim=-1).max()))
    big += float(s["bias"].abs().max()) if s["bias"] is not None else 0.0
    top = float(s["lse"][torch.isfinite(s["lse"])].abs().max()) if torch.isfinite(s["lse"]).any() else 0.0
    rel = (d + 8) * 2.0 ** -24 * (big + top) + 2.0 ** -21 + N * 2.0 ** -24
    assert ((got["score"].double() - ref["score"]).abs() <= rel * ref["score"].abs()).all()


COMMITS = [
    # rows heads kv d nodes lengths accepted
    (1, 1, 1, 64, 1, [0], [[0]]),                                    # the first token
    (2, 16, 16, 64, 1, [49, 3], [[0], []]),                          # a step; nothing accepted
    (2, 16, 16, 64, 16, [1006, 70], [[0, 1, 2, 7, 15], [3]]),
    (3, 8, 2, 128, 9, [700, 0, 33], [[1, 4, 8], [0, 1, 2, 3, 4, 5, 6, 7, 8], [-1]]),
    (1, 28, 4, 128, 20, [1500], [list(range(0, 20, 2))]),            # 70 rows a KV head: two turns
    (1, 12, 1, 64, 64, [130], [list(range(64))]),                    # every node, twelve heads on one KV head
    (2, 2, 1, 24, 3, [31, 32], [[0, 2], [1]]),
    (1, 4, 2, 256, 6, [257], [[2, 5]]),
    (1, 3, 3, 32, 4, [5000], [[0, 3]]),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", COMMITS, ids=[f"r{c[0]}h{c[1]}kv{c[2]}d{c[3]}n{c[4]}l{max(c[5])}" for c in COMMITS])
def test_commit(case, dtype):
    s = make_commit(3, dtype, *case)
    check_commit(s, commit(s))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("buckets,evicted", [(16, False), (128, True), (0, True), (2900, True)])
def test_commit_bias_and_positions(dtype, buckets, evicted):
    s = make_commit(5, dtype, 2, 6, 2, 64, 11, [300, 37], [[0, 1, 9], [2, 10]], buckets=buckets, evicted=evicted)
    check_commit(s, commit(s))


def test_commit_without_weights_and_first_scores():
    s = make_commit(7, "bf16", 2, 4, 2, 64, 5, [40, 7], [[0, 2], [4]], evicted=True)
    check_commit(s, commit(s, weights=False), weights=False)
    s = make_commit(7, "bf16", 2, 4, 2, 64, 5, [40, 7], [[0, 2], [4]], old_scores=False)
    check_commit(s, commit(s))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("old_scores", [False, True], ids=["first", "later"])
def test_commit_writes_the_scores_of_sequences_that_accept_nothing(dtype, old_scores):
    """All drafts rejected, a full cache, an empty one: their scores are the old ones, 0 where
    there were none, and not what score_out held."""
    acc = [[], [0, 2], [3], [], [1, 4]]
    s = make_commit(35, dtype, 5, 4, 2, 64, 5, [300, 7, 310, 0, 45], acc, capacity=310, old_scores=old_scores)
    got = commit(s)
    assert got["length"].tolist() == [300, 9, 310, 0, 47]
    check_commit(s, got)
    for b in (0, 2):
        n = int(s["length"][b])
        assert torch.equal(got["score"][b, :, :n], s["score"][b, :, :n] if old_scores else torch.zeros(2, n))
        assert (got["score"][b, :, n:] == -7).all()


def test_commit_stops_where_the_path_does():
    """Descending, repeated and foreign ids end the path, and so does a full cache."""
    acc = [[0, 3, 3, 4], [2, 1, 4, -1], [1, 5, -1, -1], [-1, 0, 1, 2], [1, 2, 4, -1], [0, 1, 2, 3]]
    s = make_commit(9, "bf16", 6, 2, 2, 64, 5, [20, 20, 20, 20, 20, 23], acc, capacity=25)
    got = commit(s)
    assert got["length"].tolist() == [22, 21, 21, 20, 23, 25]
    check_commit(s, got)
    s["length"] = torch.tensor([25, 26, -4, 0, 24, 25], dtype=torch.int32)  # full, out of range, empty
    s["lse"] = s["lse"].clamp_max(50.0)
    got = commit(s)
    assert got["length"].tolist() == [25, 25, 1, 0, 25, 25]
    check_commit(s, got)


def test_commit_of_absent_nodes_gives_no_weight():
    s = make_commit(11, "bf16", 1, 4, 2, 64, 5, [20], [[0, 2, 4]])
    s["lse"][0, 2] = -math.inf
    got = commit(s)
    assert torch.isfinite(got["score"]).all()
    check_commit(s, got)


def test_commit_ignores_unused_slots_and_scores_in_place():
    s = make_commit(13, "bf16", 2, 4, 2, 128, 5, [45, 3], [[0, 3], [1]], capacity=80)
    clean = commit(s)
    check_commit(s, clean)
    for b in range(2):
        for x in (s["k"], s["v"]):
            x[b, :, int(s["length"][b]):] = math.nan
    got = commit(s)
    check_commit(s, got)
    assert torch.equal(got["score"], clean["score"])
    d = on_gpu(s)
    cache = mrt_df.KVCache(d["k"], d["v"], d["length"], score=d["score"])
    mrt_df.cache_commit(cache, d["k_new"], d["v_new"], d["accepted"], torch.empty_like(d["length"]), q=d["q"], lse=d["lse"],
                        score_out=d["score"], scale=s["scale"])
    for b in range(2):
        n = int(clean["length"][b])
        assert torch.equal(d["score"][b, :, :n].cpu(), clean["score"][b, :, :n])


@pytest.mark.parametrize("masked", [-math.inf, float(torch.finfo(torch.float32).min)], ids=["inf", "lowest"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_commit_masks_in_the_bias(dtype, masked):
    """Masked distances add nothing, nor does a head for which nothing is left."""
    s = make_commit(31, dtype, 2, 6, 2, 64, 9, [300, 37], [[0, 1, 5], [2]], buckets=16)
    plain = s["bias"].clone()
    s["bias"][0, 3:], s["bias"][4] = -math.inf, -math.inf
    s["lse"] = O.tree_attention(**{n: s[n] for n in ("q", "k_new", "v_new", "k", "v", "length", "parents", "scale", "bias",
                                                     "pos", "next_pos")})[1].float()
    assert (s["lse"][:, :, 4] == -math.inf).all()
    got = commit(dict(s, bias=s["bias"].clamp(min=masked)))
    ref = O.cache_commit(s["k"], s["v"], s["length"], s["k_new"], s["v_new"], s["accepted"], q=s["q"], lse=s["lse"],
                         score=s["score"], score_out=s["score_out"], scale=s["scale"], bias=s["bias"])
    big = float(s["scale"] * s["q"].double().norm(dim=-1).max() * max(s[n].double().norm(dim=-1).max() for n in ("k", "k_new")))
    big += float(plain.abs().max()) + float(s["lse"][s["lse"] > -math.inf].abs().max())
    rel = (64 + 8) * 2.0 ** -24 * big + 2.0 ** -21 + 10 * 2.0 ** -24
    assert ((got["score"].double() - ref["score"]).abs() <= rel * ref["score"].abs()).all()


@pytest.mark.parametrize("masked", [-math.inf, float(torch.finfo(torch.float32).min)], ids=["inf", "lowest"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("evicted", [False, True], ids=["slots", "pos"])
def test_commit_masked_entries_may_hold_anything(dtype, evicted, masked):
    """Infinities and NaN in the keys of entries that the bias masks for every token: their
    scores are the old ones, and all others as without them."""
    s = make_commit(37, dtype, 2, 6, 2, 64, 9, [300, 37], [[0, 1, 5], [2]], buckets=12, evicted=evicted)
    s["bias"][:, 9:] = -math.inf
    s["lse"] = O.tree_attention(**{n: s[n] for n in ("q", "k_new", "v_new", "k", "v", "length", "parents", "scale", "bias",
                                                     "pos", "next_pos")})[1].float()
    s["bias"] = s["bias"].clamp(min=masked)
    want = commit(s)["score"]
    for b, L in enumerate((300, 37)):
        first = int(s["next_pos"][b]) if evicted else L
        for g in range(2):
            pos = s["pos"][b, g, :L] if evicted else torch.arange(L)
            far = (first - pos >= 9).nonzero()[:, 0]
            for at, bad in zip((far[0], far[len(far) // 2], far[-1]), (math.nan, math.inf, -math.inf)):
                s["k"][b, g, at, int(at) % 64] = bad
                assert want[b, g, at] == s["score"][b, g, at]
    assert torch.equal(commit(s)["score"], want)


def test_commit_lse_that_is_not_a_number():
    """It makes the scores of the entries that its token sees NaN, as the formula says."""
    s = make_commit(33, "bf16", 1, 4, 2, 64, 6, [50], [[1, 2, 4]])
    s["lse"][0, 2, 1] = math.nan
    got = commit(s)["score"][0]
    assert got[0, :52].isnan().all() and not got[0, 52:].isnan().any() and not got[1].isnan().any()


def make_evict(seed, dtype, rows, kv_heads, d, lengths, capacity=None, spread=True):
    g = torch.Generator().manual_seed(seed)
    cap = capacity or max(lengths) + 3
    s = dict(k=torch.randn((rows, kv_heads, cap, d), generator=g).to(DT[dtype]),
             v=torch.randn((rows, kv_heads, cap, d), generator=g).to(DT[dtype]),
             length=torch.tensor(lengths, dtype=torch.int32), score=torch.rand((rows, kv_heads, cap), generator=g),
             pos=torch.full((rows, kv_heads, cap), -5, dtype=torch.int32), next_pos=torch.tensor(lengths, dtype=torch.int32))
    for b, L in enumerate(lengths):
        for h in range(kv_heads):
            s["pos"][b, h, :L] = (torch.randperm(L, generator=g) if spread else torch.arange(L)).to(torch.int32)
    return s


def evict(s, keep, recent=0, sinks=0, in_place=False):
    d = on_gpu(s)
    cache = mrt_df.KVCache(d["k"], d["v"], d["length"], pos=d["pos"], next_pos=d["next_pos"], score=d["score"])
    length_out = torch.full_like(d["length"], -1)
    score_out = d["score"] if in_place else torch.full_like(d["score"], -7)
    pos_out = d["pos"] if in_place else torch.full_like(d["pos"], -7)
    mrt_df.cache_evict(cache, keep, length_out, score_out, pos_out, recent=recent, sinks=sinks)
    torch.cuda.synchronize()
    return dict(k=d["k"].cpu(), v=d["v"].cpu(), length=length_out.cpu(), score=score_out.cpu(), pos=pos_out.cpu())


def check_evict(s, got, keep, recent=0, sinks=0, untouched=True):
    ref = O.cache_evict(s["k"], s["v"], s["length"], s["pos"], s["next_pos"], s["score"], keep, recent, sinks)
    assert torch.equal(got["length"], ref["length"])
    heads = s["k"].shape[1]
    for b in range(s["k"].shape[0]):
        m = int(ref["length"][b])
        for h in range(heads):
            assert torch.equal(got["pos"][b, h, :m], ref["pos"][b * heads + h])
            assert torch.equal(got["score"][b, h, :m].nan_to_num(11), ref["score"][b * heads + h].nan_to_num(11))
            if untouched:
                assert (got["pos"][b, h, m:] == -7).all() and (got["score"][b, h, m:] == -7).all()
    assert torch.equal(got["k"], ref["k"]) and torch.equal(got["v"], ref["v"])


EVICTS = [
    # rows kv d lengths keep recent sinks
    (1, 1, 64, [1], 1, 0, 0),
    (1, 1, 64, [2], 1, 1, 0),
    (2, 3, 64, [40, 17], 16, 4, 2),
    (3, 2, 64, [1056, 0, 1006], 1006, 128, 4),
    (2, 2, 128, [2047, 2048], 900, 100, 0),
    (2, 1, 24, [2100, 5000], 1999, 0, 4),
    (1, 2, 256, [9000], 4000, 4000, 0),          # every entry that stays is recent
    (1, 1, 32, [20000], 15000, 7, 1),
    (1, 1, 8, [75000], 100, 10, 10),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("case", EVICTS, ids=[f"r{c[0]}kv{c[1]}d{c[2]}l{max(c[3])}k{c[4]}" for c in EVICTS])
def test_evict(case, dtype):
    rows, kv, d, lengths, keep, recent, sinks = case
    s = make_evict(3, dtype, rows, kv, d, lengths)
    check_evict(s, evict(s, keep, recent, sinks), keep, recent, sinks)


@pytest.mark.parametrize("capacity", [200, 256, 257, 512, 513, 768, 769, 1024, 1025, 1280, 1281, 1536, 1537, 1792, 1793, 2048, 2049])
def test_evict_at_the_capacities_where_kernels_change(capacity):
    s = make_evict(17, "bf16", 2, 2, 16, [capacity, capacity - 70], capacity=capacity)
    s["score"][1, 1] = torch.randint(0, 5, (capacity,)).float()  # ties
    for keep in (capacity - 40, capacity // 3):
        check_evict(s, evict(s, keep, 9, 4), keep, 9, 4)


def test_evict_ties_and_special_scores():
    """Equal scores go by the lower slot; NaN and -inf last, +inf first, -0 is 0."""
    s = make_evict(5, "bf16", 2, 2, 64, [300, 300], spread=False)
    s["score"][0] = 1.0
    s["score"][1, 0] = torch.randint(0, 3, (303,)).float()
    s["score"][1, 1] = torch.tensor([math.nan, -math.inf, 0.0, -0.0, 1e-42, -1e-42, math.inf, -3.0] * 38)[:303]
    for keep in (1, 37, 150, 299):
        check_evict(s, evict(s, keep), keep)


@pytest.mark.parametrize("length", [2900, 4096, 4097, 20000, 140000])
def test_evict_long_ties_and_special_scores(length):
    """The same where a head's slots go to several blocks: one score everywhere, few
    scores, scores that differ in their last bits alone."""
    s = make_evict(13, "bf16", 2, 2, 16, [length, length // 2 + 1], spread=False)
    c = s["score"].shape[-1]
    s["score"][0, 0] = 0.25
    s["score"][0, 1] = torch.randint(0, 3, (c,)).float()
    s["score"][1, 0] = torch.tensor([math.nan, -math.inf, 0.0, -0.0, 1e-42, -1e-42, math.inf, -3.0]).repeat(c // 8 + 1)[:c]
    s["score"][1, 1] = torch.nextafter(torch.tensor(1.0), torch.tensor(2.0)) * (1 + torch.randint(0, 9, (c,)) * 2.0**-23)
    for keep, recent, sinks in ((1, 0, 0), (length // 3, 5, 4), (length // 2 + 1, 0, 1), (length - 1, 700, 3)):
        check_evict(s, evict(s, keep, recent, sinks), keep, recent, sinks)


def test_evict_in_place_and_repeated():
    s = make_evict(7, "fp16", 2, 4, 128, [4000, 3000])
    for keep in (3500, 1000):
        got = evict(s, keep, 64, 4)
        check_evict(s, got, keep, 64, 4)
        check_evict(s, evict(s, keep, 64, 4, in_place=True), keep, 64, 4, untouched=False)
        again = evict(s, keep, 64, 4)
        assert all(torch.equal(got[n], again[n]) for n in got)


def test_evict_strided_cache_and_out_of_range_lengths():
    s = make_evict(9, "bf16", 3, 2, 64, [90, 90, 90], capacity=100)
    s["length"] = torch.tensor([-1, 500, 60], dtype=torch.int32)
    s["pos"][:, :, 90:] = torch.arange(90, 100, dtype=torch.int32)
    d = on_gpu(s)
    both = torch.zeros((3, 100, 2, 2, 64), dtype=torch.bfloat16, device=DEV)
    kk, vv = both[:, :, :, 0].transpose(1, 2), both[:, :, :, 1].transpose(1, 2)
    kk.copy_(d["k"]), vv.copy_(d["v"])
    d["k"], d["v"] = kk, vv
    cache = mrt_df.KVCache(kk, vv, d["length"], pos=d["pos"], next_pos=d["next_pos"], score=d["score"])
    out = torch.full_like(d["length"], -1), torch.full_like(d["score"], -7), torch.full_like(d["pos"], -7)
    mrt_df.cache_evict(cache, 50, *out, recent=8, sinks=1)
    check_evict(s, dict(k=kk.cpu(), v=vv.cpu(), length=out[0].cpu(), score=out[1].cpu(), pos=out[2].cpu()), 50, 8, 1)


def test_evict_and_commit_replay_from_a_graph():
    s = make_commit(15, "bf16", 2, 8, 2, 128, 6, [9000, 4000], [[0, 2, 5], [1]], evicted=True)
    want = commit(s)
    d = on_gpu(s)
    cache = mrt_df.KVCache(d["k"], d["v"], d["length"], pos=d["pos"], next_pos=d["next_pos"], score=d["score"])
    length_out, next_out = torch.empty_like(d["length"]), torch.empty_like(d["length"])
    score2, pos2, length2 = torch.empty_like(d["score"]), torch.empty_like(d["pos"]), torch.empty_like(d["length"])
    after = mrt_df.KVCache(d["k"], d["v"], length_out, pos=d["pos"], next_pos=next_out, score=d["score_out"])

    def step():
        mrt_df.cache_commit(cache, d["k_new"], d["v_new"], d["accepted"], length_out, next_out=next_out, q=d["q"],
                            lse=d["lse"], score_out=d["score_out"], scale=s["scale"])
        mrt_df.cache_evict(after, 3000, length2, score2, pos2, recent=50, sinks=4)

    ref = {**s, "k": want["k"], "v": want["v"], "length": want["length"], "pos": want["pos"], "next_pos": want["next_pos"],
           "score": want["score"]}
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        d["k"].copy_(s["k"]), d["v"].copy_(s["v"])
        score2.fill_(-7), pos2.fill_(-7), length2.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        check_evict(ref, dict(k=d["k"].cpu(), v=d["v"].cpu(), length=length2.cpu(), score=score2.cpu(), pos=pos2.cpu()),
                    3000, 50, 4)
