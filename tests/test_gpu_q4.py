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
