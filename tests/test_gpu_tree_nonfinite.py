"""Infinities, NaN and masks of tree attention, in every form of its kernels.

What an output is follows from the definition, out = sum of w v over the entries that are
not masked, each w > 0 however small: an infinite v makes it that infinity, two opposite
ones or a NaN make it NaN, and what is masked has no part in it, whatever it holds.
Finite outputs have the tolerances of test_gpu_tree_attention.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle import drafting_oracle as O
from test_gpu_cache_ops import check_commit, commit, make_commit
from test_gpu_tree_attention import bounds, call, make, oracle

pytestmark = pytest.mark.gpu

FORMS = [
    # heads kv d nodes lengths capacity   which kernel, and how its work is cut
    (4, 4, 64, 1, [40], None),          # few rows, one block a unit
    (4, 4, 64, 3, [3000], None),        # ... cut
    (3, 1, 24, 7, [300], None),         # ... other head sizes
    (2, 1, 128, 20, [700], None),       # two, four and eight row tiles (16-bit), d 128
    (2, 1, 256, 9, [700], None),
    (2, 2, 64, 25, [40], None),         # d 64: two, four, eight, sixteen row tiles; whole and cut
    (2, 2, 64, 25, [3000], None),
    (2, 1, 64, 25, [900], None),
    (4, 1, 64, 25, [900], None),
    (8, 1, 64, 25, [40], None),
    (8, 1, 128, 25, [2000], None),
    (8, 2, 128, 25, [900], None),
    (4, 4, 64, 17, [9000, 0, 400], 70000),   # shared out by all lengths
    (4, 4, 64, 1, [9000, 0, 400], 140000),
]
IDS = [f"h{f[0]}kv{f[1]}d{f[2]}n{f[3]}l{f[4][0]}c{f[5] or 0}" for f in FORMS]


def form(seed, dtype, f, **kw):
    heads, kv, d, nodes, lengths, cap = f
    return make(seed, dtype, len(lengths), heads, kv, d, nodes, lengths, capacity=cap, **kw)


def finite_check(s, dtype, out, ref, where):
    tol, _ = bounds(s, dtype)
    lim = tol + torch.finfo(out.dtype).eps / 2 * (ref.abs() + tol)
    assert ((out.double() - ref).abs() <= lim)[where].all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("f", FORMS, ids=IDS)
def test_infinite_nodes_stay_beside_a_dominating_entry(f, dtype):
    """An ancestor's infinite value stays, though a cached key outweighs it by some 150 powers
    of e, so that its weight beside the key's is far below what fp32 holds."""
    s = form(51, dtype, f)
    s["v_new"][0, 0, :, 3] = math.inf
    s["v_new"][0, 0, :, 5] = -math.inf
    s["parents"][0] = torch.arange(-1, f[3] - 1, dtype=torch.int32)  # a chain: all see node 0
    s["q"][0] = s["q"][0].abs() * 0.5 + 0.5
    big = 150 / (s["scale"] * f[2] * 0.5)  # every q is at least 0.5 in every dimension
    s["k"][0, :, s["length"][0] - 1] = big
    assert (s["scale"] * (s["q"][0].double().sum(-1) * big)).min() > 150
    out, lse = call(s)
    ref, rlse = oracle(s)
    assert (out[0, :, :, 3] == math.inf).all() and (out[0, :, :, 5] == -math.inf).all()
    fin = torch.ones(out.shape[-1], dtype=torch.bool)
    fin[3], fin[5] = False, False
    assert torch.isfinite(out[0][..., fin]).all() and torch.isfinite(lse[0]).all()
    # the dominating entry's values, to the type's last digit and the logits' own
    want = s["v"][0, :, s["length"][0] - 1].double().repeat_interleave(f[0] // f[1], 0)[None].expand_as(out[0])
    err = (out[0].double() - want).abs()[..., fin]
    assert (err <= (torch.finfo(out.dtype).eps / 2 + 2.0 ** -16) * want.abs()[..., fin]).all()


def seen_values(s, j):
    """Infinities and a NaN in cached entries of sequence 0, the columns that they reach."""
    s["v"][0, :, j[0], 1] = math.inf
    s["v"][0, :, j[1], 2] = -math.inf
    s["v"][0, :, j[2], 3] = math.nan
    s["v"][0, :, j[0], 4], s["v"][0, :, j[2], 4] = math.inf, -math.inf
    s["v"][0, :, j[1], 6] = math.inf
    s["v_new"][0, 0, :, 6] = math.inf
    s["parents"][0] = torch.arange(-1, s["parents"].shape[1] - 1, dtype=torch.int32)
    return {1: math.inf, 2: -math.inf, 3: math.nan, 4: math.nan, 6: math.inf}


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("f", FORMS, ids=IDS)
@pytest.mark.parametrize("buckets", [0, 16])
def test_infinities_of_the_cache_stay(f, dtype, buckets):
    """In its first, its last and another entry; other columns and sequences as without them."""
    s = form(53, dtype, f, buckets=buckets)
    ref, rlse = oracle(s)
    L = int(s["length"][0])
    s2 = {n: x.clone() if isinstance(x, torch.Tensor) else x for n, x in s.items()}
    want = seen_values(s2, (0, L // 2 + 1, L - 1))
    s["parents"][0] = s2["parents"][0]
    ref, rlse = oracle(s)
    out, lse = call(s2)
    for col, v in want.items():
        got = out[0, :, :, col]
        assert (got.isnan() if math.isnan(v) else got == v).all(), (col, got)
        ref[0, :, :, col], out[0, :, :, col] = 0, 0
    finite_check(s, dtype, out, ref, torch.ones(out.shape, dtype=torch.bool))
    assert (lse.double() - rlse).abs().max() <= bounds(s, dtype)[1]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("f", FORMS, ids=IDS)
def test_infinities_of_the_cache_stay_beside_a_dominating_entry(f, dtype):
    s = form(55, dtype, f)
    L = int(s["length"][0])
    want = seen_values(s, (0, L // 2 + 1, L - 2))
    s["q"][0] = s["q"][0].abs() * 0.5 + 0.5
    s["k"][0, :, L - 1] = 150 / (s["scale"] * f[2] * 0.5)
    out, _ = call(s)
    for col, v in want.items():
        got = out[0, :, :, col]
        assert (got.isnan() if math.isnan(v) else got == v).all(), (col, got)
    rest = [c for c in range(f[2]) if c not in want]
    assert torch.isfinite(out[0][..., rest]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("f", FORMS, ids=IDS)
def test_infinite_keys(f, dtype):
    """A key with a logit of -inf is masked, of +inf or NaN makes its row NaN, and no other."""
    s = form(57, dtype, f)
    heads, kv, d, nodes = f[:4]
    s["q"][0, :, :, 0] = 1.0
    s["q"][0, 0, 0, 0] = -1.0       # one row for which the infinite key is +inf
    s["k"][0, 0, 5, 0] = -math.inf
    s["v"][0, 0, 5] = math.nan      # and whose value nobody else reads
    clean = {n: x.clone() if isinstance(x, torch.Tensor) else x for n, x in s.items()}
    clean["k"][0, 0, 5] = 0
    clean["v"][0, 0, 5] = 0
    ref, rlse = oracle(clean)
    # without entry 5: its weight e^0 and value 0 taken out again
    n = heads // kv
    for h in range(n):
        w = (-rlse[0, :, h]).exp()
        ref[0, :, h] /= (1 - w)[:, None]
        rlse[0, :, h] += torch.log1p(-w)
    out, lse = call(s)
    assert out[0, 0, 0].isnan().all() and lse[0, 0, 0].isnan()
    out[0, 0, 0], lse[0, 0, 0], ref[0, 0, 0], rlse[0, 0, 0] = 0, 0, 0, 0
    finite_check(clean, dtype, out, ref, torch.ones(out.shape, dtype=torch.bool))
    assert (lse.double() - rlse).abs().max() <= bounds(clean, dtype)[1]


@pytest.mark.parametrize("lowest", [False, True], ids=["inf", "lowest"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("evicted", [False, True], ids=["slots", "pos"])
@pytest.mark.parametrize("f", FORMS, ids=IDS)
def test_masked_entries_may_hold_anything(f, evicted, dtype, lowest):
    """Distances of 9 and more masked by the bias: infinities and NaN in the keys and values of
    such entries change nothing."""
    s = form(59, dtype, f, buckets=12, evicted=evicted)
    heads, kv, d, nodes = f[:4]
    plain = s["bias"].clone()
    s["bias"][:, 9:] = -math.inf
    ref, rlse = oracle(s)
    run = dict(s, bias=s["bias"].clamp(min=float(torch.finfo(torch.float32).min))) if lowest else s
    L, first = int(s["length"][0]), int(s["next_pos"][0]) if evicted else int(s["length"][0])
    pos = s["pos"][0, :, :L] if evicted else torch.arange(L).expand(kv, L)
    dirty = dict(run, k=s["k"].clone(), v=s["v"].clone())
    for g in range(kv):
        far = (first - pos[g] >= 9).nonzero()[:, 0]  # of every node: a node's position is first or later
        for at, bad in zip((0, len(far) // 3, len(far) // 2, len(far) - 2, len(far) - 1),
                           (math.nan, math.inf, -math.inf, math.nan, math.inf)):
            dirty["k"][0, g, far[at], at % d] = bad
            dirty["v"][0, g, far[at], (at + 1) % d] = bad
            dirty["v"][0, g, far[at], d - 1] = -bad
    out, lse = call(dirty)
    finite_check(dict(s, bias=plain), dtype, out, ref, torch.ones(out.shape, dtype=torch.bool))
    assert (lse.double() - rlse).abs().max() <= bounds(dict(s, bias=plain), dtype)[1]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("nodes", [3, 20, 60])
def test_masked_nodes_may_hold_anything(nodes, dtype):
    """The same of drafted nodes: ancestors from distance 2 on are masked."""
    s = make(61, dtype, 2, 4, 2, 64, nodes, [30, 0], buckets=3)
    s["parents"][:] = torch.arange(-1, nodes - 1, dtype=torch.int32)
    plain = s["bias"].clone()
    s["bias"][:, 2:] = -math.inf
    ref, rlse = oracle(s)
    dirty = dict(s, k_new=s["k_new"].clone(), v_new=s["v_new"].clone())
    dirty["k_new"][:, 0], dirty["v_new"][:, 0] = math.nan, math.inf  # masked for nodes 2 and on
    out, lse = call(dirty)
    where = torch.zeros(out.shape, dtype=torch.bool)
    where[:, 2:] = True
    finite_check(dict(s, bias=plain), dtype, out, ref, where)
    assert (lse.double() - rlse).abs()[:, 2:].max() <= bounds(dict(s, bias=plain), dtype)[1]
    assert out[:, :2].isnan().all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("nodes", [1, 10, 25, 60])
@pytest.mark.parametrize("buckets", [0, 16])
def test_scales_of_every_kind(nodes, buckets, dtype):
    """0, tiny and negative scales as the formula says; one that is NaN makes every row that is
    there NaN, in every kernel, and an absent node's 0."""
    s = make(63, dtype, 2, 4, 2, 64, nodes, [300, 0], buckets=buckets)
    if nodes > 1:
        s["parents"][:, 1:] = 0
        s["parents"][:, nodes - 1] = -3
    for scale in (0.0, 1e-42, -0.11):
        run = dict(s, scale=scale)
        out, lse = call(run)
        ref, rlse = oracle(run)
        tol, ltol = bounds(dict(s, scale=abs(scale)), dtype)
        assert ((out.double() - ref).abs() <= tol + torch.finfo(out.dtype).eps / 2 * (ref.abs() + tol)).all()
        there = torch.isfinite(rlse)
        assert (lse.double() - rlse).abs()[there].max() <= ltol and torch.equal(there, torch.isfinite(lse))
    out, lse = call(dict(s, scale=math.nan))
    there = nodes - 1 if nodes > 1 else 1
    assert out[:, :there].isnan().all() and lse[:, :there].isnan().all()
    assert (out[:, there:] == 0).all() and (lse[:, there:] == -math.inf).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("f", FORMS, ids=IDS)
def test_absent_nodes_may_hold_anything(f, dtype):
    """Padding: q, k_new and v_new of absent nodes that nobody wrote.  No bit of the others
    depends on them."""
    s = form(65, dtype, f)
    nodes = f[3]
    s["parents"][:, (nodes + 1) // 2:] = -9
    for n in ("q", "k_new", "v_new"):
        s[n][:, (nodes + 1) // 2:] = 0
    ref, rlse = oracle(s)
    there = torch.isfinite(rlse)
    clean = call(s)
    for bad in ((math.nan, math.inf, -math.inf), (60.0, -60.0, 1e4)):
        dirty = dict(s)
        for n, x in zip(("q", "k_new", "v_new"), bad):
            dirty[n] = s[n].clone()
            dirty[n][:, (nodes + 1) // 2:] = x
        out, lse = call(dirty)
        finite_check(s, dtype, out, ref, torch.ones(out.shape, dtype=torch.bool))
        assert torch.equal(there, torch.isfinite(lse)) and (lse.double() - rlse).abs()[there].max() <= bounds(s, dtype)[1]
        assert torch.equal(out, clean[0]) and torch.equal(lse, clean[1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("f", FORMS, ids=IDS)
def test_rows_do_not_depend_on_each_other(f, dtype):
    """Other queries for one node, NaN too: the other nodes' bits stay."""
    s = form(69, dtype, f)
    clean = call(s)
    for q in (s["q"][:, -1] * 7 + 1, math.nan):
        run = dict(s, q=s["q"].clone())
        run["q"][:, -1] = q
        got = call(run)
        assert torch.equal(got[0][:, :-1], clean[0][:, :-1]) and torch.equal(got[1][:, :-1], clean[1][:, :-1])
    assert got[0][:, -1].isnan().all() and got[1][:, -1].isnan().all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("nodes", [1, 25])
def test_positions_at_the_ends_of_their_type(nodes, dtype):
    """Distances beyond 31 bits count as far, or where they are negative as 0."""
    s = make(67, dtype, 2, 4, 2, 64, nodes, [90, 40], buckets=7, evicted=True)
    s["pos"][:, :, ::3] = -(2 ** 31)
    s["pos"][:, :, 1::3] = 2 ** 31 - 1
    s["next_pos"] = torch.tensor([2 ** 31 - 100, -(2 ** 31) + 5], dtype=torch.int32)
    ref, rlse = oracle(s)
    out, lse = call(s)
    finite_check(s, dtype, out, ref, torch.ones(out.shape, dtype=torch.bool))
    there = torch.isfinite(rlse)
    assert (lse.double() - rlse).abs()[there].max() <= bounds(s, dtype)[1]
    c = make_commit(67, dtype, 2, 4, 2, 64, nodes, [90, 40], [[0], [nodes - 1]], buckets=7, evicted=True)
    c["pos"][:, :, ::3] = -(2 ** 31)
    c["pos"][:, :, 1::3] = 2 ** 31 - 1
    c["next_pos"] = s["next_pos"].clone()
    c["lse"] = O.tree_attention(**{n: c[n] for n in ("q", "k_new", "v_new", "k", "v", "length", "parents", "scale", "bias",
                                                     "pos", "next_pos")})[1].float()
    check_commit(c, commit(c))
