"""Products with 4-bit weights (mrt_q4_matmul) against 64 bits.

Tolerance of an output: codes times activations are exact; sums are fp32 of k terms
of at most 31 |scale x| + (|bias| + 16 |scale|) |x| each, in blocks, so an error of
`steps` 2^-24 of their total with steps = 32 per instruction and group chains, k / 32
groups and 8 waves (no chain is longer than 64 + k / 32 + 8 additions); then half a
step of the type.
"""

from __future__ import annotations

import pytest
import torch

import mrt_df
from oracle import drafting_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make(seed, dtype, rows, k, n, group):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), generator=g, dtype=torch.int64).to(torch.int32)
    scales = (torch.rand((n, k // group), generator=g) + 0.5) / 16
    return (torch.randn((rows, k), generator=g).to(DT[dtype]), w, scales.to(DT[dtype]),
            (scales * (torch.randn((n, k // group), generator=g) - 7)).to(DT[dtype]))


def check(x, w, scales, biases, got):
    wd = O.q4_weights(w, scales, biases)
    ref = x.double() @ wd.T
    group = x.shape[1] // scales.shape[1]
    size = (31 * scales.double().abs() + biases.double().abs() + 16 * scales.double().abs()).repeat_interleave(group, 1)
    total = x.double().abs() @ size.T
    tol = (64 + x.shape[1] / 32 + 8) * 2.0 ** -24 * total
    lim = tol + torch.finfo(got.dtype).eps / 2 * (ref.abs() + tol) + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    err = (got.double() - ref).abs()
    assert (err <= lim).all(), float((err / lim).max())


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,k,n", [(1, 128, 16), (2, 1024, 5632), (3, 128, 1), (1, 384, 17), (16, 2816, 100), (17, 768, 50),
                                      (33, 1152, 129), (64, 256, 333), (5, 8192, 70)])
def test_matches_oracle(dtype, group, rows, k, n):
    x, w, s, b = make(3, dtype, rows, k, n, group)
    got = mrt_df.q4_matmul(x.to(DEV), w.to(DEV), s.to(DEV), b.to(DEV))
    check(x, w, s, b, got.cpu())


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,k,n,group", [(1, 32, 5, 32), (2, 96, 40, 32), (130, 320, 37, 64), (65, 160, 16, 32), (1, 64, 1, 64)])
def test_ragged(dtype, rows, k, n, group):
    x, w, s, b = make(5, dtype, rows, k, n, group)
    got = mrt_df.q4_matmul(x.to(DEV), w.to(DEV), s.to(DEV), b.to(DEV))
    check(x, w, s, b, got.cpu())


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_strides_leave_the_rest(dtype):
    """x as a column range, out into a wider array at an odd column."""
    x, w, s, b = make(7, dtype, 6, 256, 61, 64)
    want = mrt_df.q4_matmul(x.to(DEV), w.to(DEV), s.to(DEV), b.to(DEV))
    check(x, w, s, b, want.cpu())
    wide = torch.full((6, 400), 7.0, dtype=DT[dtype], device=DEV)
    wide[:, 64:320] = x.to(DEV)
    out = torch.full((8, 71), 9.0, dtype=DT[dtype], device=DEV)
    got = mrt_df.q4_matmul(wide[:, 64:320], w.to(DEV), s.to(DEV), b.to(DEV), out=out[1:7, 3:64])
    assert torch.equal(got, want)
    rest = out.clone()
    rest[1:7, 3:64] = 9.0
    assert (rest == 9.0).all()


def test_rows_do_not_depend_on_each_other():
    """A row's outputs are the same bits whatever other rows are in the call."""
    x, w, s, b = (t.to(DEV) for t in make(9, "bf16", 64, 1024, 200, 64))
    whole = mrt_df.q4_matmul(x, w, s, b)
    for lo, hi in ((0, 1), (3, 20), (5, 64)):
        assert torch.equal(mrt_df.q4_matmul(x[lo:hi], w, s, b), whole[lo:hi])
    x[7, 100] = float("nan")
    x[9, 5] = float("inf")
    dirty = mrt_df.q4_matmul(x, w, s, b)
    keep = [r for r in range(64) if r not in (7, 9)]
    assert torch.equal(dirty[keep], whole[keep]) and not torch.isfinite(dirty[[7, 9]].float()).any()


def test_graph_replays():
    x, w, s, b = (t.to(DEV) for t in make(11, "bf16", 2, 1024, 5632, 64))
    want = mrt_df.q4_matmul(x, w, s, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = mrt_df.q4_matmul(x, w, s, b)
    for _ in range(3):
        got.zero_()
        graph.replay()
        assert torch.equal(mrt_df.q4_matmul(x, w, s, b), want)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize(dtype, group):
    """Every weight within half a code step (and the roundings of scale, bias and
    range to the type) of its 4-bit value; a flat group exactly its bias."""
    g = torch.Generator().manual_seed(13)
    w = torch.randn((70, 640), generator=g)
    w[3, :group] = 0.75
    w[4, :group] = torch.linspace(-1, 2, group)
    w = w.to(DT[dtype])
    big = torch.zeros((70, 704), dtype=DT[dtype], device=DEV)
    big[:, :640] = w.to(DEV)
    codes, scales, biases = (t.cpu() for t in mrt_df.q4_quantize(big[:, :640], group))
    back = O.q4_weights(codes, scales, biases)
    span = w.double().view(70, -1, group)
    step = ((span.amax(-1) - span.amin(-1)) / 15).repeat_interleave(group, 1)
    eps = torch.finfo(DT[dtype]).eps / 2
    # the scale's rounding moves code 15 by 15 steps' worth of it; the quotient is fp32
    lim = step * (0.5 + 16 * eps + 2.0 ** -20)
    assert ((back - w.double()).abs() <= lim).all()
    assert (back[3, :group] == 0.75).all()
    assert int(codes[3, 0]) == 0


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("mean", [0.0, 1.0, 30.0])
@pytest.mark.parametrize("rows,k,n", [(4, 2048, 64), (5, 1024, 520), (3, 8192, 40)])
def test_fp32_rows_with_a_mean(rows, k, n, mean, group):
    """Codes count from their middle, so that a mean of x does not make large sums that cancel.
    Per instruction (32 products of one of x's parts) two roundings or truncations, at most
    2^-23 each, of the accumulator, whose values are computed here, and the 32 products;
    then per group three roundings of its terms, and of the running sum: 2^-24 each."""
    g = torch.Generator().manual_seed(17)
    w, scales, biases = (t.cpu() for t in mrt_df.q4_quantize(torch.randn((n, k), generator=g).to(DEV), group))
    x = torch.randn((rows, k), generator=g) + mean
    got = mrt_df.q4_matmul(x.to(DEV), w.to(DEV), scales.to(DEV), biases.to(DEV)).cpu().double()
    wd = O.q4_weights(w, scales, biases)
    ref = x.double() @ wd.T
    s = scales.double().repeat_interleave(group, 1)
    b = biases.double().repeat_interleave(group, 1)
    code = (wd - b) / s - 7.5
    xs = x.double()[:, None, :] * (s * code)[None]                       # (rows, n, k)
    step = xs.view(rows, n, k // group, group // 32, 32)
    acc = step.sum(-1).cumsum(-1).abs()
    inside = (acc + step.abs().sum(-1)).sum((-1, -2))
    off = (b + 7.5 * s)[:, ::group][None] * x.double().view(rows, 1, k // group, group).sum(-1)
    terms = acc[..., -1] + off.abs()
    running = (step.sum((-1, -2)) + off).abs().cumsum(-1)
    size = (x.double().abs()[:, None, :] * (b + 7.5 * s).abs()[None]).sum(-1)  # the sums of x, by the same instructions
    tol = 2 * 2.0 ** -23 * (inside + size) + 2.0 ** -24 * (3 * terms.sum(-1) + running.sum(-1) / 8 + 8 * running[..., -1])
    err = (got - ref).abs()
    assert (err <= tol + 2.0 ** -24 * ref.abs()).all(), float((err / tol).max())
    # As a whole, with roundings that do not depend on each other: 6 k / 32 of them (three parts),
    # of sums of at most 128 + 32 products where the result is one of k, so
    # sqrt(6 / 32 160) 2^-23 = 6.6e-7 of it.
    assert err.norm() <= 1e-6 * ref.norm()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_large_rows(dtype, group):
    """Finite x up to the type's largest values: a result within the type's range is right."""
    x, w, s, b = make(19, dtype, 4, 512, 40, group)
    big = torch.finfo(DT[dtype]).max
    x[0] = torch.where(x[0].double() > 0, 1.0, -1.0).to(DT[dtype]) * big
    x[1] = big
    x[2] = (x[2].double() / x[2].double().abs().max() * big).to(DT[dtype])
    s, b = s / 256, b / 256         # outputs stay in range
    got = mrt_df.q4_matmul(x.to(DEV), w.to(DEV), s.to(DEV), b.to(DEV)).cpu()
    ref = x.double() @ O.q4_weights(w, s, b).T
    assert ref.abs().max() < big
    assert torch.isfinite(got.double()).all()
    group_size = (31 * s.double().abs() + b.double().abs() + 16 * s.double().abs()).repeat_interleave(group, 1)
    tol = (64 + 512 / 32 + 8) * 2.0 ** -24 * (x.double().abs() @ group_size.T)
    lim = tol + torch.finfo(got.dtype).eps / 2 * (ref.abs() + tol) + 2.0 ** -25
    assert ((got.double() - ref).abs() <= lim).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_quantize_keeps_what_is_not_a_number(dtype, group, bad):
    """A group with an infinite or NaN weight becomes NaN as a whole, the others as without it."""
    g = torch.Generator().manual_seed(23)
    w = torch.randn((6, 384), generator=g).to(DT[dtype])
    clean = [t.cpu() for t in mrt_df.q4_quantize(w.to(DEV), group)]
    w[1, 5], w[1, group - 1], w[4, 383] = bad, bad, bad
    got = [t.cpu() for t in mrt_df.q4_quantize(w.to(DEV), group)]
    hit = torch.zeros(got[1].shape, dtype=torch.bool)
    hit[1, 0], hit[4, -1] = True, True
    for t, c in zip(got[1:], clean[1:]):
        assert t[hit].isnan().all() and torch.equal(t[~hit], c[~hit])
    words = ~hit.repeat_interleave(group // 8, 1)
    assert torch.equal(got[0][words], clean[0][words])
    y = mrt_df.q4_matmul(torch.ones((2, 384), dtype=DT[dtype], device=DEV), *(t.to(DEV) for t in got)).cpu()
    rows = torch.tensor([False, True, False, False, True, False])
    assert y[:, rows].isnan().all() and torch.isfinite(y[:, ~rows]).all()


WIDE = [
    # rows k n     column tiles of a block: two from n 8177 on, four for up to 16 rows from 16369 on
    (1, 256, 8177), (16, 1152, 8200), (17, 1152, 8177), (32, 256, 8200), (33, 1152, 8177), (64, 1152, 8200),
    (5, 1152, 16385), (16, 256, 16400), (1, 2304, 16385), (9, 128, 29824),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,k,n", WIDE)
def test_many_columns(rows, k, n, group, dtype):
    k -= 128 - group if k > 1024 else 0  # no whole chunk of 128 at the end
    x, w, s, b = make(29, dtype, rows, k, n, group)
    got = mrt_df.q4_matmul(x.to(DEV), w.to(DEV), s.to(DEV), b.to(DEV))
    check(x, w, s, b, got.cpu())
