"""Arguments that the drafting operators refuse, without a GPU: a status code and a
message before any device call, and ValueError from the binding."""

from __future__ import annotations

import ctypes

import pytest
import torch

import mrt_df

INVALID = 1
P = 0x1000  # a pointer that no refused call follows


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


def test_no_rows_is_no_work(lib):
    assert lib.mrt_tree_attention(cache(rows=0), tree(), None, 0, 0, None) == 0


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
