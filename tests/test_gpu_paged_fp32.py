"""Attention of fp32 operands over 8-bit pages (mrt_paged_attention): as accurate as fp32 pages, whatever
one channel of q or one entry of the cache holds.

Per output, from the arithmetic: codes are exact, and so are the parts that q, scaled by a power of two,
and the weights are multiplied in (three of 8 bits).  A logit is a sum of d products in fp32, each partial
sum rounded to 2^-24 of at most the sum of the terms' magnitudes, and one of 2 d small ones, each rounded to
2^-8 of that, which is d + 2 roundings at most for d up to 256; then it is scaled twice, biased and
shifted by the running maximum: delta = (d + 8) 2^-24 of the largest such sum (and bias) and 2^-21 for exp2.
A weight is off by 2 delta of itself at most, the quotient's sum likewise; weights times scales, and the sums
over N entries of weights, of values and of small parts, add (3 N + 8) 2^-24 of the sum of the magnitudes
weighted the same way, which the oracle gives for a cache of magnitudes.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle import serving_oracle as O
from test_gpu_paged import call, make

pytestmark = pytest.mark.gpu
STORE = "i8-fp32"


def terms(c, s):
    """The largest sum of the magnitudes of a logit's terms, over the entries that have a value."""
    n = s["q"].shape[2] // c["k"].shape[1]
    most = 0.0
    for g in range(c["k"].shape[1]):
        k = (c["k"][:, g].double().abs() * c["k_scale"][:, g].double().nan_to_num(0)[..., None]).flatten(0, 1)
        q = s["q"][:, :, g * n:(g + 1) * n].double().abs().flatten(0, 2)
        most = max(most, float((q @ k.T).max()))
    return abs(s["scale"]) * most + (0.0 if s["bias"] is None else float(s["bias"][s["bias"] > -1e29].abs().max()))


def check(c, s):
    out, lse = call(c, s)
    ref, rlse = O.paged_attention(s["q"], c, s["fresh"], s["scale"], s["bias"])
    size, _ = O.paged_attention(s["q"], dict(c, v=c["v"].abs()), s["fresh"], s["scale"], s["bias"])
    N, d, big = int(c["length"].max()) + s["q"].shape[1], s["q"].shape[3], terms(c, s)
    delta = (d + 8) * 2.0 ** -24 * big + 2.0 ** -21
    err = (out.double() - ref).abs()
    lim = (4 * delta + (3 * N + 8) * 2.0 ** -24) * size
    assert torch.isfinite(out).all() and (err <= lim).all(), float((err / lim).nan_to_num(0).max())
    there = torch.isfinite(rlse)
    assert torch.equal(there, torch.isfinite(lse))
    ltol = delta + N * 2.0 ** -24 + 2.0 ** -22 * (big + math.log(max(N, 2)))
    assert not there.any() or (lse.double() - rlse).abs()[there].max() <= ltol


CASES = [
    # rows heads kv d tokens lengths page
    (2, 16, 16, 64, 1, [49, 15], 16),
    (2, 12, 12, 64, 3, [300, 17], 32),
    (2, 8, 2, 128, 1, [2500, 700], 128),
    (1, 8, 1, 256, 4, [777], 256),
    (2, 6, 2, 96, 5, [300, 90], 16),
    (1, 3, 1, 16, 7, [100], 16),
    (2, 8, 4, 64, 15, [900, 260], 80),
]
IDS = [f"h{c[1]}kv{c[2]}d{c[3]}t{c[4]}l{max(c[5])}" for c in CASES]


@pytest.mark.parametrize("ratio", [1.0, 2.0 ** 10, 2.0 ** 20, 2.0 ** 40])
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_channels_far_above_the_others(case, ratio):
    """One channel of q, where keys have nothing: the others count as if it were not there."""
    c, s = make(41, STORE, *case, buckets=32)
    s["q"][..., 5] *= ratio
    c["k"][..., 5] = 0
    check(c, s)


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_entries_far_above_the_others(case):
    """One entry with a large scale and few values: the dimensions that it has nothing in keep theirs."""
    c, s = make(42, STORE, *case)
    for b, length in enumerate(case[5]):
        at = O.entry_place(c, b, length // 2)
        c["v_scale"][at[0], :, at[1]] *= 2.0 ** 20
        c["v"][at[0], :, at[1], 4:] = 0
    check(c, s)


def test_queries_of_any_size():
    """Rows of q from 2^-100 to 2^100 beside keys that make logits of them, an empty row, one of one value."""
    c, s = make(43, STORE, 2, 4, 2, 64, 3, [200, 40])
    up = torch.exp2(torch.tensor([-100.0, 0.0, 100.0]))
    for t in range(3):
        one = dict(s, q=s["q"] * up[t])
        few = dict(c, k_scale=c["k_scale"] / up[t])
        check(few, one)
    s["q"][0, 1] = 0
    s["q"][1, 2, 3] = 0
    s["q"][1, 2, 3, 63] = -3.0
    check(c, s)


def test_rows_that_are_not_finite():
    """They are NaN, also where every logit would be minus infinity; no other row changes a bit."""
    c, s = make(44, STORE, 2, 4, 2, 64, 3, [200, 40])
    c["k"].abs_()  # an infinity times these is never opposite
    want, wlse = call(c, s)
    s["q"][0, 1, 2, 9], s["q"][1, 0, 0, 63], s["q"][1, 2, 3, 0] = -math.inf, math.nan, math.inf
    bad = ~torch.isfinite(s["q"]).all(-1)
    out, lse = call(c, s)
    assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
    assert torch.equal(out[~bad], want[~bad]) and torch.equal(lse[~bad], wlse[~bad])
