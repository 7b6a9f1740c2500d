"""Arguments that the drafting operators refuse, without a GPU: a status code and a
message before any device call, and ValueError from the binding."""

from __future__ import annotations

import ctypes

import pytest
import torch

import mrt_df

INVALID = 1
P = 0x1000  # a pointer that no refused call follows
V = 0x100000  # another, far from it


@pytest.fixture(scope="module")
def lib():
    return mrt_df.load_library()


def cache(k=P, v=P, rs=2048, hs=1024, ss=64, length=P, pos=0, next_pos=0, score=0, rows=2, kv=2, cap=16, d=64, dtype=1):
    return mrt_df._CACHE_STRUCT.pack(k, v, rs, hs, ss, length, pos, next_pos, score, rows, kv, cap, d, dtype)


BAD_CACHES = {
    "null k": dict(k=0), "null v": dict(v=0), "null length": dict(length=0), "misaligned k": dict(k=P + 8),
    "negative rows": dict(rows=-1), "no heads": dict(kv=0), "no slots": dict(cap=0), "odd d": dict(d=60),
    "wide d": dict(d=264), "no d": dict(d=0), "dtype": dict(dtype=3), "stride": dict(ss=68), "negative stride": dict(hs=-1024),
    "overlapping slots": dict(ss=32), "pos alone": dict(pos=P), "too many heads": dict(rows=1 << 12, kv=1 << 9),
    "too long": dict(cap=(1 << 30) + 1),
}


def tree(q=P, k=P, v=P, out=P, qs=(4 * 256, 256, 64), os=(4 * 256, 256, 64), parents=P, ps=4, lse=P, bias=0, buckets=0,
         nodes=4, heads=4, scale=1.0):
    return mrt_df._TREE_STRUCT.pack(q, *qs, k, 512, 128, 64, v, 512, 128, 64, out, *os, parents, ps, lse, bias, buckets,
                                    nodes, heads, scale)


BAD_TREES = {
    "null q": dict(q=0), "null k": dict(k=0), "null v": dict(v=0), "null out": dict(out=0), "null parents": dict(parents=0),
    "misaligned q": dict(q=P + 4), "stride": dict(qs=(1024, 250, 64)), "negative stride": dict(qs=(1024, 256, -64)),
    "no nodes": dict(nodes=0), "many nodes": dict(nodes=65), "heads": dict(heads=3), "no heads": dict(heads=0),
    "bias without buckets": dict(bias=P), "overlapping out": dict(os=(1024, 256, 0)), "parents stride": dict(ps=-4),
    "too many buckets": dict(bias=P, buckets=(1 << 18) + 1),
}


def refused(lib, code):
    assert code == INVALID and lib.mrt_last_error()


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_tree_attention_refuses_caches(lib, bad):
    refused(lib, lib.mrt_tree_attention(cache(**BAD_CACHES[bad]), tree(), P, 1 << 20, 0, None))


@pytest.mark.parametrize("bad", BAD_TREES)
def test_tree_attention_refuses(lib, bad):
    refused(lib, lib.mrt_tree_attention(cache(), tree(**BAD_TREES[bad]), P, 1 << 20, 0, None))


def test_tree_attention_refuses_null_and_small_workspaces(lib):
    refused(lib, lib.mrt_tree_attention(None, tree(), None, 0, 0, None))
    refused(lib, lib.mrt_tree_attention(cache(), None, None, 0, 0, None))
    size = ctypes.c_size_t()
    refused(lib, lib.mrt_tree_attention_workspace(cache(), 4, 4, None))
    refused(lib, lib.mrt_tree_attention_workspace(cache(), 4, 65, ctypes.byref(size)))
    long = cache(cap=100000, hs=6400000, rs=12800000)
    assert lib.mrt_tree_attention_workspace(long, 4, 4, ctypes.byref(size)) == 0 and size.value > 0
    refused(lib, lib.mrt_tree_attention(long, tree(), None, 0, 0, None))
    refused(lib, lib.mrt_tree_attention(long, tree(), P, size.value - 1, 0, None))
    refused(lib, lib.mrt_tree_attention(long, tree(), P + 4, size.value, 0, None))
    assert lib.mrt_tree_attention_workspace(cache(cap=64), 4, 4, ctypes.byref(size)) == 0 and size.value == 0


def test_tree_attention_refuses_more_rows_than_it_counts(lib):
    many = cache(rows=1 << 20, kv=1, rs=0, hs=0)
    refused(lib, lib.mrt_tree_attention(many, tree(nodes=64, heads=64), P, 1 << 40, 0, None))
    size = ctypes.c_size_t()
    refused(lib, lib.mrt_tree_attention_workspace(many, 64, 64, ctypes.byref(size)))


def test_no_rows_is_no_work(lib):
    assert lib.mrt_tree_attention(cache(rows=0), tree(), None, 0, 0, None) == 0
    empty = cache(rows=0, k=0, v=0, length=0)  # as an empty tensor's pointers are
    assert lib.mrt_tree_attention(empty, tree(q=0, k=0, v=0, out=0, parents=0, lse=0), None, 0, 0, None) == 0
    assert lib.mrt_cache_commit(empty, commit(k=0, v=0, q=0, accepted=0, length_out=0), 0, None) == 0
    assert lib.mrt_cache_evict(empty, evict(score_out=0, pos_out=0, length_out=0), None, 0, 0, None) == 0
    assert lib.mrt_q4_matmul(None, 64, 0, None, None, None, 64, 64, 64, 1, None, 64, 0, None) == 0


def test_writes_refuse_caches_that_share_slots(lib):
    full = dict(pos=P, next_pos=P, score=P)
    for bad in (dict(rs=0), dict(hs=0)):
        refused(lib, lib.mrt_cache_commit(cache(**bad), commit(), 0, None))
        refused(lib, lib.mrt_cache_evict(cache(**bad, **full), evict(), P, 1 << 20, 0, None))


def test_outputs_of_their_own(lib):
    positions = dict(pos=P, next_pos=P + 128)
    refused(lib, lib.mrt_cache_commit(cache(**positions), commit(length_out=P + 128, next_out=P + 256), 0, None))
    refused(lib, lib.mrt_cache_commit(cache(**positions), commit(length_out=P + 256, next_out=P + 256), 0, None))
    refused(lib, lib.mrt_cache_commit(cache(**positions), commit(next_out=P), 0, None))
    refused(lib, lib.mrt_cache_evict(cache(score=P, **positions), evict(length_out=P + 128), P, 1 << 20, 0, None))


def test_binding_refuses_cpu_tensors_and_wrong_shapes():
    k = torch.zeros((2, 2, 16, 64))
    n = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        mrt_df.KVCache(k, k.clone(), n)                    # not on a GPU
    with pytest.raises(ValueError):
        mrt_df.KVCache(k.double(), k.double(), n)          # dtype
    with pytest.raises(ValueError):
        mrt_df.KVCache(k[0], k[0], n)                      # three dimensions
    with pytest.raises(ValueError):
        mrt_df.KVCache(k, k[:, :, :8], n)                  # v unlike k
    with pytest.raises(ValueError):
        mrt_df.KVCache(k.transpose(2, 3), k.transpose(2, 3), n)  # d not contiguous


def commit(k=P, v=P, q=P, lse=P, score_out=P, accepted=P, astride=4, length_out=P + 64, next_out=0, accepted_n=4, nodes=4,
           heads=4, bias=0, buckets=0):
    qs = (4 * 256, 256, 64)
    return mrt_df._COMMIT_STRUCT.pack(k, 512, 128, 64, v, 512, 128, 64, q, *qs, accepted, astride, lse, bias, score_out,
                                      length_out, next_out, accepted_n, nodes, heads, buckets, 1.0)


BAD_COMMITS = {
    "null k": dict(k=0), "null v": dict(v=0), "misaligned k": dict(k=P + 2), "null accepted": dict(accepted=0),
    "accepted stride": dict(astride=-1), "null length_out": dict(length_out=0), "length_out in place": dict(length_out=P),
    "no lse": dict(lse=0), "no score_out": dict(score_out=0), "nothing accepted": dict(accepted_n=0),
    "many accepted": dict(accepted_n=65), "no nodes": dict(nodes=0), "many nodes": dict(nodes=65), "heads": dict(heads=5),
    "bias without buckets": dict(bias=P),
}


@pytest.mark.parametrize("bad", BAD_COMMITS)
def test_commit_refuses(lib, bad):
    refused(lib, lib.mrt_cache_commit(cache(), commit(**BAD_COMMITS[bad]), 0, None))


def test_commit_refuses_caches(lib):
    for bad in BAD_CACHES.values():
        refused(lib, lib.mrt_cache_commit(cache(**bad), commit(), 0, None))
    refused(lib, lib.mrt_cache_commit(None, commit(), 0, None))
    refused(lib, lib.mrt_cache_commit(cache(), None, 0, None))
    positions = dict(pos=P, next_pos=P + 128)
    refused(lib, lib.mrt_cache_commit(cache(**positions), commit(), 0, None))                     # no next_out
    refused(lib, lib.mrt_cache_commit(cache(**positions), commit(next_out=P + 128), 0, None))     # in place
    assert lib.mrt_cache_commit(cache(rows=0), commit(), 0, None) == 0


def evict(score_out=P, pos_out=P, length_out=P + 64, keep=8, recent=0, sinks=0):
    return mrt_df._EVICT_STRUCT.pack(score_out, pos_out, length_out, keep, recent, sinks)


BAD_EVICTS = {
    "null score_out": dict(score_out=0), "null pos_out": dict(pos_out=0), "null length_out": dict(length_out=0),
    "length_out in place": dict(length_out=P), "keep": dict(keep=0), "recent": dict(recent=-1), "sinks": dict(sinks=-1),
    "more fixed than kept": dict(recent=5, sinks=4), "overflow": dict(recent=2 ** 31 - 1, sinks=2 ** 31 - 1),
}


@pytest.mark.parametrize("bad", BAD_EVICTS)
def test_evict_refuses(lib, bad):
    full = cache(pos=P, next_pos=P, score=P)
    refused(lib, lib.mrt_cache_evict(full, evict(**BAD_EVICTS[bad]), P, 1 << 20, 0, None))


def test_evict_refuses_caches_and_workspaces(lib):
    for bad in BAD_CACHES.values():
        refused(lib, lib.mrt_cache_evict(cache(**{**dict(pos=P, next_pos=P, score=P), **bad, **({"next_pos": 0} if "pos" in bad else {})}),
                                         evict(), P, 1 << 20, 0, None))
    refused(lib, lib.mrt_cache_evict(cache(score=P), evict(), P, 1 << 20, 0, None))
    refused(lib, lib.mrt_cache_evict(cache(pos=P, next_pos=P), evict(), P, 1 << 20, 0, None))
    refused(lib, lib.mrt_cache_evict(None, evict(), P, 1 << 20, 0, None))
    refused(lib, lib.mrt_cache_evict(cache(pos=P, next_pos=P, score=P), None, P, 1 << 20, 0, None))
    size = ctypes.c_size_t()
    refused(lib, lib.mrt_cache_evict_workspace(cache(), 0, ctypes.byref(size)))
    refused(lib, lib.mrt_cache_evict_workspace(cache(), 4, None))
    long = cache(pos=P, next_pos=P, score=P, cap=100000, hs=6400000, rs=12800000)
    assert lib.mrt_cache_evict_workspace(long, 50000, ctypes.byref(size)) == 0 and size.value > 0
    refused(lib, lib.mrt_cache_evict(long, evict(keep=50000), None, 0, 0, None))
    refused(lib, lib.mrt_cache_evict(long, evict(keep=50000), P, size.value - 1, 0, None))
    assert lib.mrt_cache_evict(cache(rows=0, pos=P, next_pos=P, score=P), evict(), None, 0, 0, None) == 0


Q4 = dict(x=P, ldx=128, rows=2, w=P, scales=P, biases=P, n=16, k=128, group=64, dtype=1, out=P, ldo=16)
BAD_Q4 = {
    "null x": dict(x=None), "null w": dict(w=None), "null scales": dict(scales=None), "null biases": dict(biases=None),
    "null out": dict(out=None), "misaligned x": dict(x=P + 8), "misaligned w": dict(w=P + 4), "rows": dict(rows=-1),
    "n": dict(n=0), "k": dict(k=0), "k and group": dict(k=96), "group": dict(group=16), "dtype": dict(dtype=7),
    "narrow ldx": dict(ldx=64), "odd ldx": dict(ldx=132), "narrow ldo": dict(ldo=8),
}


@pytest.mark.parametrize("bad", BAD_Q4)
def test_q4_matmul_refuses(lib, bad):
    a = {**Q4, **BAD_Q4[bad]}
    refused(lib, lib.mrt_q4_matmul(a["x"], a["ldx"], a["rows"], a["w"], a["scales"], a["biases"], a["n"], a["k"], a["group"],
                                   a["dtype"], a["out"], a["ldo"], 0, None))


def test_q4_no_rows_and_quantize_refusals(lib):
    assert lib.mrt_q4_matmul(P, 128, 0, P, P, P, 16, 128, 64, 1, P, 16, 0, None) == 0
    for a in ((None, 128, 16, 128, 64, 1, P, P, P), (P, 128, 16, 128, 48, 1, P, P, P), (P, 64, 16, 128, 64, 1, P, P, P),
              (P, 128, 0, 128, 64, 1, P, P, P), (P, 128, 16, 128, 64, 9, P, P, P), (P, 128, 16, 128, 64, 1, None, P, P),
              (P, 128, 16, 128, 64, 1, P, None, P), (P, 128, 16, 128, 64, 1, P, P, None)):
        refused(lib, lib.mrt_q4_quantize(*a, 0, None))
    with pytest.raises(ValueError):
        mrt_df.q4_matmul(torch.zeros(2, 64), torch.zeros(4, 8, dtype=torch.int32), torch.zeros(4, 1), torch.zeros(4, 1))
    with pytest.raises(ValueError):
        mrt_df.q4_quantize(torch.zeros(4, 64), 64)


@pytest.mark.parametrize("name", ["length", "pos", "next_pos", "score"])
def test_refuses_misaligned_arrays_of_caches(lib, name):
    full = dict(pos=P, next_pos=P, score=P)
    bad = cache(**{**full, name: P + 2})
    refused(lib, lib.mrt_tree_attention(bad, tree(), P, 1 << 20, 0, None))
    refused(lib, lib.mrt_cache_commit(bad, commit(next_out=P + 256), 0, None))
    refused(lib, lib.mrt_cache_evict(bad, evict(), P, 1 << 20, 0, None))


@pytest.mark.parametrize("bad", [dict(parents=P + 2), dict(lse=P + 1), dict(bias=P + 2, buckets=4)], ids=["parents", "lse", "bias"])
def test_tree_attention_refuses_misaligned_arrays(lib, bad):
    refused(lib, lib.mrt_tree_attention(cache(), tree(**bad), P, 1 << 20, 0, None))


@pytest.mark.parametrize("name", ["accepted", "lse", "score_out", "length_out", "next_out"])
def test_commit_refuses_misaligned_arrays(lib, name):
    args = dict(length_out=P + 64, next_out=P + 256)
    refused(lib, lib.mrt_cache_commit(cache(pos=P, next_pos=P), commit(**{**args, name: P + 514}), 0, None))


@pytest.mark.parametrize("name", ["score_out", "pos_out", "length_out"])
def test_evict_refuses_misaligned_arrays(lib, name):
    refused(lib, lib.mrt_cache_evict(cache(pos=P, next_pos=P, score=P), evict(**{name: P + 66}), P, 1 << 20, 0, None))


@pytest.mark.parametrize("dtype,off", [(0, 2), (1, 1), (2, 1)], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("name", ["scales", "biases", "out"])
def test_q4_matmul_refuses_misaligned_arrays(lib, name, dtype, off):
    a = {**Q4, "dtype": dtype, name: P + off}
    refused(lib, lib.mrt_q4_matmul(a["x"], a["ldx"], a["rows"], a["w"], a["scales"], a["biases"], a["n"], a["k"], a["group"],
                                   a["dtype"], a["out"], a["ldo"], 0, None))


@pytest.mark.parametrize("at", [0, 6, 7, 8], ids=["src", "w", "scales", "biases"])
def test_q4_quantize_refuses_misaligned_arrays(lib, at):
    a = [P, 128, 16, 128, 64, 1, P, P, P]
    a[at] = P + 1
    refused(lib, lib.mrt_q4_quantize(*a, 0, None))


OVERLAPS = {
    "sequences share slots": dict(rs=0), "heads share slots": dict(hs=0), "sequences reach into heads": dict(rs=1024, hs=1024),
    "sequences reach into slots": dict(rs=64, hs=1024), "heads reach into slots": dict(hs=1016), "heads among slots": dict(hs=64),
    "sequences a slot short": dict(rs=1984), "slots reach into each other": dict(hs=64, ss=120, rs=2048),
    "v is k": dict(v=P), "v a slot behind k": dict(v=P + 128), "v a sequence behind k": dict(v=P + 4096),
    "v before k": dict(k=V + 1024, v=V), "v half a slot behind k": dict(v=P + 64),
}


@pytest.mark.parametrize("bad", OVERLAPS)
def test_writes_refuse_caches_that_overlap(lib, bad):
    c = cache(**{"v": V, "pos": P, "next_pos": P, "score": P, **OVERLAPS[bad]})
    refused(lib, lib.mrt_cache_commit(c, commit(next_out=P + 256), 0, None))
    assert b"overlap" in lib.mrt_last_error()
    refused(lib, lib.mrt_cache_evict(c, evict(), P, 1 << 20, 0, None))
    assert b"overlap" in lib.mrt_last_error()


@pytest.mark.parametrize("strides", [(1024, 64, 64), (1024, 256, 256), (256, 256, 64), (1024, 256, 56), (1016, 256, 64), (0, 256, 64)])
def test_tree_attention_refuses_out_that_overlaps(lib, strides):
    refused(lib, lib.mrt_tree_attention(cache(), tree(os=strides), P, 1 << 20, 0, None))
    assert b"out overlaps" in lib.mrt_last_error()


NOWHERE = 1 << 20  # a device that there is not: a call that passes the checks ends there


def test_tree_attention_takes_out_with_sequences_innermost(lib):
    code = lib.mrt_tree_attention(cache(), tree(os=(64, 1024, 256)), P, 1 << 20, NOWHERE, None)
    assert code not in (0, INVALID)


@pytest.mark.parametrize("layout", [
    dict(rs=2048, hs=1024, ss=64, v=P + 8192),                  # one array after the other
    dict(rs=4096, hs=128, ss=256, k=P, v=P + 128),              # slots of k and v in turn: (rows, capacity, heads, 2, d)
    dict(rs=4096, hs=64, ss=256, v=P + 256),                    # (rows, capacity, 2, heads, d)
    dict(rs=1024, hs=8192, ss=64, v=P + (1 << 20)),               # heads outermost
    dict(rs=64, hs=4096, ss=128, v=P + 2048 * 2),               # sequences innermost; v behind k's head
    dict(rs=7, hs=1024, ss=64, rows=1, v=P + 4096),             # a single sequence's stride is not used
    dict(rs=1 << 60, hs=1 << 59, ss=1 << 40, cap=1 << 18, v=V),  # extents past 64 bits
])
def test_writes_take_caches_whose_slots_lie_apart(lib, layout):
    c = cache(**{"pos": P, "next_pos": P, **layout})
    assert lib.mrt_cache_commit(c, commit(next_out=P + 256), NOWHERE, None) not in (0, INVALID)


def test_refuses_what_a_launch_has_no_threads_for(lib):
    size = ctypes.c_size_t()
    for rows, heads, nodes, ok in ((1 << 20, 1, 64, True), (1 << 20, 16, 64, False), (1 << 16, 1024, 16, False), (1, 4096, 64, True),
                                   (1 << 14, 64, 64, True)):
        c = cache(rows=rows, kv=1, rs=0, hs=0)
        assert (lib.mrt_tree_attention_workspace(c, heads, nodes, ctypes.byref(size)) == 0) == ok, (rows, heads, nodes)
        if not ok:
            wide = (heads * nodes * 64, heads * 64, 64)
            refused(lib, lib.mrt_tree_attention(c, tree(nodes=nodes, heads=heads, os=wide), P, 1 << 60, NOWHERE, None))
            assert b"too many" in lib.mrt_last_error()
    a = {**Q4, "n": (1 << 28) - 63, "ldo": 1 << 28, "rows": 40}
    refused(lib, lib.mrt_q4_matmul(a["x"], a["ldx"], a["rows"], a["w"], a["scales"], a["biases"], a["n"], a["k"], a["group"],
                                   a["dtype"], a["out"], a["ldo"], NOWHERE, None))
    refused(lib, lib.mrt_q4_quantize(P, 1 << 20, 1 << 15, 1 << 20, 64, 1, P, P, P, NOWHERE, None))
    assert lib.mrt_q4_quantize(P, 1 << 20, (1 << 15) - 1, 1 << 20, 64, 1, P, P, P, NOWHERE, None) not in (0, INVALID)
