"""Caches in pages: entries written, read back and attended (mrt_paged_*) against 64 bits.

Writing and reading are exact: scales are fp32 products, codes fp32 quotients rounded to
whole numbers, values fp32 products rounded once.

Attention, per output, from the arithmetic.  Pages of the operands' type: a logit is a sum
of d products in fp32, scaled, biased and shifted by the running maximum, each step rounded
to 2^-24 of a magnitude of at most `big`; exp2 is good to 2^-22; 16-bit weights are two-part
(2^-17 of each for bf16, 2^-22 for fp16).  8-bit pages: q is within 2^-22 of its row's
largest magnitude, so a logit within scale 2^-22 max|q| |k|_1; the sum is exact, six
roundings follow; weights times scales are within 2^-22 of the largest of 64 entries, whose
sum over the steps is at most the sum of the weights: 64 2^-22 of the largest value.  The
quotient's error is at most twice a weight's plus the sums' own, and the output's rounding
half a step of its type.
"""

from __future__ import annotations

import math

import pytest
import torch

import mrt_df
from oracle import serving_oracle as O
from test_gpu_i8 import near_ties

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SPLIT = {"bf16": 2.0 ** -17, "fp16": 2.0 ** -22, "fp32": 0.0}
STORES = ["bf16", "fp16", "fp32", "i8-bf16", "i8-fp16", "i8-fp32"]


def types(store):
    return store.startswith("i8"), DT[store.split("-")[-1]]


def make(seed, store, rows, heads, kv_heads, d, tokens, lengths, page=16, buckets=0, fresh=None, spare=2, slots_first=False):
    """A cache whose pages lie in no order; what no entry is in holds infinities and NaN."""
    codes, dt = types(store)
    g = torch.Generator().manual_seed(seed)
    need = [-(-(n + tokens) // page) for n in lengths]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g)
    table = torch.full((rows, max(need) + 1), 2 ** 31 - 1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].to(torch.int32)
        table[b, n + 1:] = -1
        at += n
    c = dict(table=table, length=torch.tensor(lengths, dtype=torch.int32), k_scale=None, v_scale=None)
    used = torch.zeros((pages, page), dtype=torch.bool)
    for b, n in enumerate(lengths):
        end = n + (tokens if fresh is None else fresh[b])
        for e in range(end):
            used[table[b, e // page], e % page] = True
    for x in "kv":
        pool = torch.randn((pages, kv_heads, page, d), generator=g).to(dt)
        if codes:
            pool, scale = O.quantise(pool)
            c[x + "_scale"] = torch.where(used[:, None], scale, torch.tensor(math.nan))
        else:
            pool = torch.where(used[:, None, :, None], pool, torch.tensor(math.nan if x == "k" else math.inf, dtype=dt))
        c[x] = pool.transpose(1, 2).contiguous().transpose(1, 2) if slots_first else pool
    s = dict(q=torch.randn((rows, tokens, heads, d), generator=g).to(dt), scale=1.5 / math.sqrt(d), bias=None,
             fresh=None if fresh is None else torch.tensor(fresh, dtype=torch.int32))
    if buckets:
        s["bias"] = torch.randn((heads, buckets), generator=g)
    return c, s


def on_gpu(x):
    if isinstance(x, dict):
        return {n: on_gpu(y) for n, y in x.items()}
    if not isinstance(x, torch.Tensor):
        return x
    return torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=DEV).copy_(x)


def pages(c):
    return mrt_df.PagedCache(c["k"], c["v"], c["table"], c["length"], c["k_scale"], c["v_scale"])


def call(c, s, **kw):
    c, s = on_gpu(c), on_gpu(s)
    out, lse = mrt_df.paged_attention(s["q"], pages(c), fresh=s["fresh"], scale=s["scale"], bias=s["bias"], **kw)
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


def workspace(c, s):
    """Bytes; none where a block takes whole sequences' heads."""
    n, kv, page, d = c["k"].shape
    return mrt_df._paged_workspace(*c["table"].shape, n, kv, page, d, mrt_df._KIND[c["k"].dtype], s["q"].shape[2], s["q"].shape[1])


def size_of(c, x, norm):
    """The largest norm of an entry's finite values."""
    v = c[x].double()
    if c[x + "_scale"] is not None:
        v = v * c[x + "_scale"].double()[..., None]
    return float(v.nan_to_num(0, 0, 0).norm(p=norm, dim=-1).max())


def bounds(c, s, store):
    codes, dt = types(store)
    N, d = int(c["length"].max()) + s["q"].shape[1], s["q"].shape[3]
    q = s["q"].double().nan_to_num(0, 0, 0)
    big = float(abs(s["scale"]) * q.norm(dim=-1).max()) * size_of(c, "k", 2)
    if s["bias"] is not None:
        by = s["bias"][s["bias"] > -1e29]
        big += float(by.abs().max()) if len(by) else 0.0
    top = size_of(c, "v", math.inf)
    delta = (d + 8) * 2.0 ** -24 * big + 2.0 ** -21
    parts = SPLIT.get(store, 0.0)
    if codes:
        delta = 8 * 2.0 ** -24 * big + 2.0 ** -21 + float(abs(s["scale"]) * q.abs().max()) * 2.0 ** -22 * size_of(c, "k", 1)
        parts = 64 * 2.0 ** -22
    return top * (2 * delta + parts + 2 * N * 2.0 ** -24), delta + N * 2.0 ** -24 + 2.0 ** -22 * (big + math.log(max(N, 2)))


def check(c, s, store, got):
    out, lse = got
    ref, rlse = O.paged_attention(s["q"], c, s["fresh"], s["scale"], s["bias"])
    tol, ltol = bounds(c, s, store)
    fin = torch.isfinite(ref)
    assert torch.equal(fin, torch.isfinite(out.double()))
    assert torch.equal(torch.isnan(ref), torch.isnan(out))
    assert torch.equal(ref[~fin & ~torch.isnan(ref)], out.double()[~fin & ~torch.isnan(ref)])
    err = (out.double() - ref).abs()[fin]
    lim = tol + torch.finfo(out.dtype).eps / 2 * (ref.abs()[fin] + tol) + (2.0 ** -25 if out.dtype == torch.float16 else 0)
    assert (err <= lim).all(), float((err / lim).max())
    there = torch.isfinite(rlse)
    assert torch.equal(there, torch.isfinite(lse)) and torch.equal(torch.isnan(rlse), torch.isnan(lse))
    assert torch.equal(rlse == -math.inf, lse == -math.inf)
    assert not there.any() or (lse.double() - rlse).abs()[there].max() <= ltol


CASES = [
    # rows heads kv d tokens lengths page         what it is for
    (1, 1, 1, 64, 1, [0], 16),                    # nothing but the token itself
    (1, 2, 1, 64, 3, [0], 16),
    (2, 16, 16, 64, 1, [49, 15], 16),             # a decode step of a CFG pair; a page that is just full
    (2, 16, 16, 64, 1, [1005, 47], 64),
    (3, 4, 2, 64, 5, [62, 63, 64], 48),           # new tokens across a page's and a step's end
    (2, 12, 12, 64, 3, [300, 17], 32),
    (2, 8, 2, 128, 1, [2500, 700], 128),          # cut and joined
    (1, 28, 4, 128, 9, [1500], 16),               # seven heads share a K/V head: 63 rows, two row blocks
    (1, 8, 1, 256, 4, [777], 256),
    (1, 2, 1, 256, 1, [4100], 16),                # the widest head, cut
    (2, 6, 2, 96, 5, [300, 90], 16),              # between the padded widths
    (1, 3, 1, 16, 7, [100], 16),                  # the narrowest head
    (1, 2, 1, 208, 20, [130], 32),
    (5, 2, 1, 32, 2, [5, 0, 200, 32, 96], 16),
    (2, 8, 4, 64, 15, [900, 260], 80),            # 30 rows: two row tiles
    (2, 8, 4, 128, 16, [900, 260], 16),
    (1, 8, 1, 64, 64, [65], 16),                  # 512 rows of one K/V head
    (1, 2, 2, 64, 1, [9000], 16),                 # several lookups of pages a wave
    (1, 4, 1, 128, 2, [20001], 512),
    (70, 2, 1, 64, 1, [13 * b for b in range(70)], 16),  # more sequences than lanes
]
IDS = [f"r{c[0]}h{c[1]}kv{c[2]}d{c[3]}t{c[4]}l{max(c[5])}p{c[6]}" for c in CASES]


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_attention_matches_oracle(case, store):
    c, s = make(3, store, *case)
    check(c, s, store, call(c, s))


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("buckets", [1, 16, 128, 2000, 9000])
def test_bias_by_distance(buckets, store):
    c, s = make(5, store, 2, 6, 2, 64, 4, [300, 37], buckets=buckets)
    check(c, s, store, call(c, s))


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("fresh", [[4, 0, 1], [0, 0, 0], [2, 3, 4]])
def test_padded_batches(fresh, store):
    """Tokens that are not there: outputs 0, lse -inf; what their slots hold is seen by nobody."""
    c, s = make(7, store, 3, 4, 2, 64, 4, [100, 33, 47], fresh=fresh, page=48)
    check(c, s, store, call(c, s))


@pytest.mark.parametrize("store", STORES)
def test_lengths_and_counts_out_of_range(store):
    c, s = make(8, store, 3, 2, 1, 64, 2, [30, 12, 40], fresh=[2, 2, 2])
    c["length"][1] = -5
    s["fresh"][2] = 9
    check(c, s, store, call(c, s))
    c["length"][0] = 2 ** 31 - 1  # every entry that the table has room for, and no new one
    c["table"][0] = c["table"][0, 0]
    s["fresh"][0] = -1
    check(c, s, store, call(c, s))


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("gone", [[0], [1, 2], [0, 1, 2, 3, 4, 5, 6]], ids=["first", "middle", "all"])
def test_pages_that_are_not_there(gone, store):
    """Freed pages (a window, a dropped prefix): their entries have no part."""
    c, s = make(9, store, 2, 4, 2, 64, 1, [100, 70], buckets=64)
    for x in gone:
        c["table"][0, x] = -1 if x % 2 else c["k"].shape[0]
    check(c, s, store, call(c, s))


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min], ids=["inf", "lowest"])
def test_masks_in_the_bias(low, store):
    """A window, one that leaves nothing, and infinities and NaN in what they mask."""
    c, s = make(10, store, 2, 4, 2, 64, 3, [200, 40], buckets=300)
    s["bias"][0, 50:] = low
    s["bias"][1, :2] = low   # not even the token itself
    s["bias"][2] = low
    s["bias"][3, 100:] = low
    for b, e in ((0, 60), (0, 3), (0, 95)):  # seen by no head of the second K/V head
        at = O.entry_place(c, b, e)
        for x in "kv":
            if c[x + "_scale"] is not None:
                c[x + "_scale"][at[0], 1, at[1]] = math.nan
            else:
                c[x][at[0], 1, at[1]] = math.inf if e == 60 else math.nan
    check(c, s, store, call(c, s))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("entry", [0, 31, 62, 63, 64])
def test_infinite_values_reach_those_who_see_them(entry, dtype):
    """Entries 62 .. 64 are new: token t sees those up to 62 + t and no later ones."""
    c, s = make(11, dtype, 1, 4, 2, 64, 3, [62])
    at = O.entry_place(c, 0, entry)
    c["v"][at[0], 0, at[1], 5] = math.inf
    c["v"][at[0], 0, at[1], 6] = -math.inf
    c["v"][at[0], 1, at[1], 7] = math.nan
    check(c, s, dtype, call(c, s))
    c["v"][at[0], 0, at[1], 6] = 1.0
    s["q"][0, 2] *= 40  # weights that underflow
    out, _ = call(c, s)
    ref, _ = O.paged_attention(s["q"], c, None, s["scale"], None)
    assert torch.equal(torch.isinf(out), torch.isinf(ref) | (out == math.inf) & (ref != ref))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_codes_that_stand_for_nan(dtype):
    """An entry with scale NaN makes NaN of the rows that see it, of its head alone."""
    store = "i8-" + dtype
    c, s = make(12, store, 2, 4, 2, 64, 3, [80, 30])
    at = O.entry_place(c, 0, 81)  # the second new token's
    c["v_scale"][at[0], 1, at[1]] = math.nan
    check(c, s, store, call(c, s))
    c["k_scale"][at[0], 0, at[1]] = math.nan
    out, lse = call(c, s)
    assert torch.isnan(out[0, 1:, :2]).all() and torch.isnan(lse[0, 1:, :2]).all()
    assert torch.isfinite(out[0, 0]).all() and torch.isfinite(out[1]).all()
    s["q"][1, 2, 3, 9] = math.inf
    out, _ = call(c, s)
    assert torch.isnan(out[1, 2, 3]).all() and torch.isfinite(out[1, :2]).all() and torch.isfinite(out[1, 2, :3]).all()


@pytest.mark.parametrize("store", ["i8-bf16", "i8-fp32"])
def test_scales_of_any_size(store):
    """Entries far apart in size, empty ones, and weights far below the largest."""
    c, s = make(13, store, 2, 4, 2, 64, 2, [200, 130])
    c["v_scale"] *= torch.exp2(torch.randint(-30, 30, c["v_scale"].shape, generator=torch.Generator().manual_seed(1)).float())
    c["k_scale"][:, :, ::7] = torch.where(torch.isnan(c["k_scale"][:, :, ::7]), c["k_scale"][:, :, ::7], 0.0)
    c["k_scale"] *= 3
    check(c, s, store, call(c, s))
    s["q"][:] = 0
    check(c, s, store, call(c, s))


@pytest.mark.parametrize("store", STORES)
def test_strides(store):
    """Pages with their heads side by side, shared pages, operands inside wider rows."""
    c, s = make(14, store, 2, 6, 2, 64, 3, [130, 130], slots_first=True)
    c["table"][1, :4] = c["table"][0, :4]  # a prefix in common
    wide = torch.randn((2, 3, 10, 96)).to(s["q"].dtype)
    wide[:, :, 2:8, 16:80] = s["q"]
    q = wide.to(DEV)[:, :, 2:8, 16:80]
    out = torch.full((3, 2, 6, 72), 7.0, dtype=q.dtype, device=DEV)
    d = on_gpu(c)
    got, lse = mrt_df.paged_attention(q, pages(d), scale=s["scale"], out=out.transpose(0, 1)[..., 8:])
    torch.cuda.synchronize()
    assert (out[..., :8] == 7).all()
    check(c, s, store, (got.cpu(), lse.cpu()))


@pytest.mark.parametrize("store", ["bf16", "i8-fp16", "fp32"])
def test_rows_do_not_depend_on_their_batch(store):
    """The parts of a sequence depend on the batch, but not on time: the same bits every time."""
    c, s = make(15, store, 3, 8, 2, 128, 4, [5000, 1300, 2049])
    first = call(c, s)
    for _ in range(3):
        again = call(c, s)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_offsets_past_31_bits():
    """A pool of more than 2^32 elements, its last page in use."""
    d, kv, page, n = 256, 8, 4096, 513
    for store in ("i8-bf16", "bf16"):
        codes, dt = types(store)
        pool = [torch.empty((n, kv, page, d), dtype=torch.int8 if codes else dt, device=DEV) for _ in range(2)]
        scale = [torch.empty((n, kv, page), device=DEV) for _ in range(2)] if codes else [None, None]
        c, s = make(16, store, 1, 16, 8, 256, 2, [20], page=4096, spare=0)
        for x, p, sc in zip("kv", pool, scale):
            p[n - 1] = c[x][0].to(DEV)
            if codes:
                sc[n - 1] = c[x + "_scale"][0].to(DEV)
        table = torch.tensor([[n - 1]], dtype=torch.int32, device=DEV)
        cache = mrt_df.PagedCache(*pool, table, c["length"].to(DEV), *scale)
        got = mrt_df.paged_attention(s["q"].to(DEV), cache, scale=s["scale"])
        torch.cuda.synchronize()
        c["table"] = c["table"][:, :1]
        check(c, s, store, [x.cpu() for x in got])
        new = torch.randn((1, 3, kv, d)).to(dt)
        c["table"] = torch.zeros((1, 1), dtype=torch.int32)
        mrt_df.paged_write(cache, new.to(DEV), new.to(DEV))
        torch.cuda.synchronize()
        want = O.paged_write(c, new, new)
        assert torch.equal(pool[0][n - 1, :, 20:23].cpu(), want["k"][0, :, 20:23])


# ---- writing and reading


def store_case(seed, store, rows, kv, d, tokens, lengths, page, fresh=None, slots_first=False):
    c, _ = make(seed, store, rows, kv, kv, d, tokens, lengths, page=page, fresh=fresh, slots_first=slots_first)
    g = torch.Generator().manual_seed(seed + 1)
    new = [(torch.randn((rows, tokens, kv, d), generator=g) * torch.exp2(torch.randint(-9, 9, (rows, tokens, kv, 1), generator=g)))
           .to(types(store)[1]) for _ in range(2)]
    return c, new, None if fresh is None else torch.tensor(fresh, dtype=torch.int32)


def same(a, b):
    return torch.equal(a.nan_to_num(1234.5), b.nan_to_num(1234.5)) and torch.equal(torch.isnan(a), torch.isnan(b))


def check_write(c, new, fresh, kn=None, vn=None):
    d = on_gpu(c)
    length = torch.full_like(d["length"], -9)
    mrt_df.paged_write(pages(d), new[0].to(DEV) if kn is None else kn, new[1].to(DEV) if vn is None else vn,
                       fresh=on_gpu(fresh), length_out=length)
    torch.cuda.synchronize()
    want = O.paged_write(c, *new, fresh)
    for n in ("k", "v", "k_scale", "v_scale"):
        if c[n] is not None:
            assert same(d[n].cpu().float(), want[n].float()), n
    assert torch.equal(length.cpu(), want["length_out"])
    return d, length


WRITES = [
    # rows kv d tokens lengths page
    (1, 1, 64, 1, [0], 16),
    (5, 8, 128, 1, [0, 15, 16, 200, 31], 16),
    (2, 3, 96, 7, [10, 0], 48),
    (2, 2, 256, 33, [100, 1], 16),
    (1, 5, 16, 130, [3], 64),
    (3, 4, 64, 50, [0, 50, 100], 32),
    (2, 2, 208, 5, [14, 15], 16),
]


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("slots_first", [False, True], ids=["heads", "slots"])
@pytest.mark.parametrize("case", WRITES, ids=[f"r{c[0]}kv{c[1]}d{c[2]}t{c[3]}p{c[5]}" for c in WRITES])
def test_write_and_read(case, slots_first, store):
    c, new, fresh = store_case(21, store, *case, slots_first=slots_first)
    d, length = check_write(c, new, fresh)
    rows, kv, dim, tokens = case[:4]
    grown = dict(d, length=length)
    for start in (None, c["length"], c["length"] - 3):
        out = [torch.full((rows, kv, tokens + 4, dim), 3.0, dtype=types(store)[1], device=DEV) for _ in range(2)]
        mrt_df.paged_read(pages(grown), *out, start=on_gpu(start))
        torch.cuda.synchronize()
        host = {n: x.cpu() if isinstance(x, torch.Tensor) else x for n, x in grown.items()}
        want = O.paged_read(host, *[torch.full_like(o, 3.0).cpu() for o in out], start)
        assert same(out[0].cpu(), want[0]) and same(out[1].cpu(), want[1])


@pytest.mark.parametrize("store", STORES)
def test_write_what_there_is_room_for(store):
    """Counts out of range, sequences that are full, pages that are not there."""
    c, new, fresh = store_case(22, store, 4, 2, 64, 20, [40, 5, 30, 10], 16, fresh=[20, 20, 20, 20])
    c["length"] = torch.tensor([c["table"].shape[1] * 16 - 4, -7, 30, 10], dtype=torch.int32)
    c["table"][0] = torch.where((c["table"][0] < 0) | (c["table"][0] >= c["k"].shape[0]), c["k"].shape[0] - 1, c["table"][0])
    c["table"][2, 2] = -3
    check_write(c, new, torch.tensor([20, 99, 20, -1], dtype=torch.int32))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_codes_of_odd_entries(dtype):
    """Zeros, infinities, NaN, the type's smallest and largest values, ties."""
    store = "i8-" + dtype
    c, new, _ = store_case(23, store, 1, 2, 64, 9, [0], 16)
    k, fi = new[0], torch.finfo(DT[dtype])
    k[0, 0] = 0
    k[0, 1, 0, 3], k[0, 1, 1, 3] = math.inf, -math.inf
    k[0, 2, 0, 7] = math.nan
    k[0, 3] = fi.max * torch.linspace(-1, 1, 64)
    k[0, 4] = fi.tiny * torch.linspace(-3, 3, 64)
    k[0, 5] = fi.smallest_normal * 2.0 ** -5 * torch.linspace(-1, 1, 64)
    k[0, 6] = (torch.arange(64) - 31.5)   # ties where the scale is 1/2
    k[0, 6, :, 0] = 63.5
    k[0, 7, :, 1:] = 0
    check_write(c, new, None)


def test_codes_near_ties():
    c, new, _ = store_case(26, "i8-fp32", 2, 3, 128, 200, [0, 7], 64)
    new = [near_ties(1200, 128, seed).view(new[0].shape) for seed in (1, 2)]
    check_write(c, new, None)


@pytest.mark.parametrize("store", ["bf16", "i8-bf16", "i8-fp32"])
def test_write_from_wider_rows(store):
    """k and v as they come out of one product, heads inside its rows."""
    c, new, _ = store_case(24, store, 2, 2, 64, 3, [5, 17], 16)
    wide = torch.zeros((2, 3, 8 * 64), dtype=new[0].dtype)
    wide[..., 256:384], wide[..., 384:] = new[0].flatten(2), new[1].flatten(2)
    g = wide.to(DEV)
    check_write(c, new, None, g[..., 256:384].unflatten(-1, (2, 64)), g[..., 384:].unflatten(-1, (2, 64)))


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("rows", [30, 150])
def test_sequences_without_new_tokens_among_long_ones(rows, store):
    """Wherever a share of the keys ends among them, their outputs are zeros."""
    lengths = [(4000 if b % 37 == 0 else 60 * (b % 5)) for b in range(rows)]
    fresh = [1 if b % 37 == 0 or b % 11 == 0 else 0 for b in range(rows)]
    c, s = make(17, store, rows, 2, 1, 64, 1, lengths, fresh=fresh)
    assert workspace(c, s) > 0  # shared out by length
    g, h = on_gpu(c), on_gpu(s)
    out = torch.full(s["q"].shape, 9.0, dtype=s["q"].dtype, device=DEV)
    lse = torch.full(s["q"].shape[:3], 9.0, device=DEV)
    mrt_df.paged_attention(h["q"], pages(g), fresh=h["fresh"], scale=s["scale"], out=out, lse=lse)
    torch.cuda.synchronize()
    check(c, s, store, (out.cpu(), lse.cpu()))


SHARED = [
    # rows heads kv d tokens lengths page                           shares end
    (70, 2, 1, 64, 1, [(37 * b * b) % 2900 for b in range(70)], 16),  # inside and between more sequences than lanes
    (3, 4, 2, 64, 2, [2700, 1, 900], 32),                           # across a sequence that is one step
    (2, 8, 1, 64, 9, [3000, 1700], 16),                             # for several row blocks alike
    (1, 14, 2, 128, 11, [5500], 64),
    (2, 2, 1, 256, 33, [2900, 2700], 128),
    (3, 2, 2, 32, 5, [5000, 17, 1300], 16),
]


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("case", SHARED, ids=[f"r{c[0]}h{c[1]}kv{c[2]}d{c[3]}t{c[4]}" for c in SHARED])
def test_keys_shared_out(case, store):
    c, s = make(18, store, *case)
    assert workspace(c, s) > 0
    check(c, s, store, call(c, s))


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("tokens", [1, 3])
def test_several_heads_a_block(tokens, store):
    """More sequences and heads than blocks: a block takes them in turn, the bias of each."""
    fresh = [b % (tokens + 1) for b in range(160)]
    c, s = make(19, store, 160, 8, 8, 64, tokens, [(7 * b) % 40 for b in range(160)], buckets=20, fresh=fresh)
    assert workspace(c, s) == 0
    check(c, s, store, call(c, s))
