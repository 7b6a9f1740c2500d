"""Forms of tree attention and of the commit that the other tests' sizes do not reach: every
row tile with a bias and both head sizes of the kernel for many rows, and work that is
shared out by all lengths in each type, with positions and with a bias in LDS or too large
for it.  Which form a call takes depends on the cache's capacity, so caches here are larger
than what is in use, and NaN beyond it.
"""

from __future__ import annotations

import math

import pytest
import torch

import mrt_df
from test_gpu_cache_ops import check_commit, commit, make_commit
from test_gpu_tree_attention import DEV, bounds, call, check, make, on_gpu, oracle

pytestmark = pytest.mark.gpu


BIASED = [
    # heads kv d nodes lengths    rows of a K/V head: 16-row tiles 2, 4, 8, 16, two blocks of 16
    (8, 4, 64, 11, [900, 40]),
    (8, 4, 128, 11, [900, 40]),
    (8, 4, 128, 16, [33]),
    (8, 2, 128, 15, [2100, 0]),
    (8, 1, 128, 15, [700, 64]),
    (8, 1, 128, 31, [1300]),
    (16, 1, 128, 31, [95, 400]),
    (8, 1, 64, 31, [1300]),
    (12, 1, 64, 50, [95, 400]),
]


@pytest.mark.parametrize("buckets,evicted", [(16, False), (128, True), (3000, True)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("f", BIASED, ids=[f"h{f[0]}kv{f[1]}d{f[2]}n{f[3]}" for f in BIASED])
def test_bias_with_many_rows(f, dtype, buckets, evicted):
    heads, kv, d, nodes, lengths = f
    s = make(71, dtype, len(lengths), heads, kv, d, nodes, lengths, buckets=buckets, evicted=evicted)
    check(s, dtype, call(s))


SHARED = [
    # rows heads kv d nodes capacity lengths buckets evicted
    (3, 32, 8, 128, 15, 45000, [9000, 0, 333], 0, False),           # 60 rows; parts of a length
    (3, 32, 8, 128, 15, 45000, [20000, 0, 333], 0, False),          # ... and teams that pass through units
    (4, 32, 4, 128, 64, 34000, [3000, 17, 0, 900], 0, False),       # 512 rows: two blocks of sixteen tiles
    (4, 32, 4, 128, 64, 34000, [17000, 17, 0, 900], 0, False),
    (5, 8, 4, 64, 9, 54000, [50, 0, 2000, 31, 700], 128, True),     # a bias in LDS, another for each head
    (5, 8, 4, 64, 9, 54000, [50, 0, 34000, 31, 700], 128, True),
    (5, 8, 4, 64, 9, 54000, [50, 0, 34000, 31, 700], 16, False),
    (5, 8, 4, 128, 20, 54000, [50, 0, 34000, 31, 700], 3000, True),  # a bias too large for it
    (3, 8, 4, 128, 30, 88000, [900, 44000, 5], 128, True),          # 60 rows
    (2, 16, 4, 128, 30, 132000, [35000, 77], 128, True),            # 120 rows: halves
    (4, 16, 2, 128, 30, 132000, [70000, 40, 1, 77], 100, False),    # 240 rows
    (4, 4, 4, 64, 1, 70000, [30000, 0, 100, 9000], 128, True),      # one node
    (4, 6, 2, 96, 5, 140000, [30000, 0, 100, 9000], 64, True),      # 15 rows, d 96
    (4, 4, 4, 256, 3, 70000, [5000, 0, 100, 70], 0, False),
]


def widen(x, capacity, fill):
    out = torch.full((*x.shape[:2], capacity, *x.shape[3:]), fill, dtype=x.dtype, device=DEV)
    out[:, :, :x.shape[2]] = x.to(DEV)
    return out


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("f", SHARED, ids=[f"r{f[0]}h{f[1]}kv{f[2]}d{f[3]}n{f[4]}l{max(f[6])}b{f[7]}" for f in SHARED])
def test_work_shared_out_by_lengths(f, dtype):
    rows, heads, kv, d, nodes, capacity, lengths, buckets, evicted = f
    s = make(73, dtype, rows, heads, kv, d, nodes, lengths, buckets=buckets, evicted=evicted)
    g = on_gpu(s)
    pos = None if s["pos"] is None else widen(s["pos"], capacity, -(2 ** 31))
    cache = mrt_df.KVCache(widen(s["k"], capacity, math.nan), widen(s["v"], capacity, math.nan), g["length"], pos=pos,
                           next_pos=g["next_pos"])
    got = [mrt_df.tree_attention(g["q"], g["k_new"], g["v_new"], cache, g["parents"], scale=s["scale"], bias=g["bias"])
           for _ in range(2)]
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    check(s, dtype, tuple(x.cpu() for x in got[0]))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("buckets", [0, 30])
def test_commit_of_many_rows_with_wide_heads(dtype, buckets):
    """d 256, 24 rows of a K/V head: two row tiles a turn; 136: five turns."""
    for heads, kv, accepted in ((8, 2, [[0, 1, 2, 4, 7, 8], [3]]), (8, 1, [list(range(17)), [2, 16]])):
        s = make_commit(75, dtype, 2, heads, kv, 256, 17, [333, 50], accepted, buckets=buckets, evicted=buckets > 0)
        check_commit(s, commit(s))
