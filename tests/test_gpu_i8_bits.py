"""Products in 8-bit integers, bit for bit: the sum rounded to fp32, times the row's scale, times the
column's, plus what is added, each step rounded to fp32, then to the type.  torch does these steps one
by one, so that a row has the same bits whichever kernel its batch and columns lead to.
"""

from __future__ import annotations

import pytest
import torch

import mrt_df
from test_gpu_i8 import DEV, DT, make

pytestmark = pytest.mark.gpu


def steps(sums, xs, ws, add, dtype):
    y = sums.float() * xs[:, None] * ws
    return (y if add is None else y + add.float()).to(DT[dtype])


SIZES = [
    # rows k n
    (1, 1024, 5632), (16, 1024, 1001), (9, 64, 12288),               # few rows
    (17, 1024, 1001), (32, 48, 6143),
    (33, 1024, 1001), (64, 2816, 1024), (40, 1024, 100),             # cut along k
    (300, 640, 500), (512, 2816, 1024),                              # tiles of 32 x 64
    (40, 128, 8198), (130, 400, 16384), (70, 128, 16385), (257, 128, 13060), (520, 144, 13057), (16, 256, 20001),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_every_step_is_rounded(rows, k, n, dtype):
    x, xs, w, ws = (t.to(DEV) for t in make(21, rows, k, n))
    add = torch.randn((rows, n), generator=torch.Generator().manual_seed(22)).to(DEV, DT[dtype])
    sums = x.double() @ w.double().T.contiguous()  # whole numbers below 2^53: exact
    for a in (None, add):
        got = mrt_df.i8_matmul(x, xs, w, ws, dtype=DT[dtype], add=a)
        want = steps(sums, xs, ws, a, dtype)
        assert torch.equal(got, want), int((got != want).sum())


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_a_row_does_not_depend_on_its_batch(dtype):
    """Alone, with 16 and 32 rows, and in batches that tiles of every size take; all columns and a few."""
    x, xs, w, ws = (t.to(DEV) for t in make(23, 1100, 512, 13060))
    add = torch.randn((1100, 13060), generator=torch.Generator().manual_seed(24)).to(DEV, DT[dtype])
    whole = mrt_df.i8_matmul(x, xs, w, ws, add=add)
    for rows in (1, 16, 17, 32, 33, 64, 300, 1099):
        for n in (33, 1000, 6144, 12288, 13059):
            got = mrt_df.i8_matmul(x[:rows], xs[:rows], w[:n], ws[:n], add=add[:rows, :n])
            assert torch.equal(got, whole[:rows, :n]), (rows, n)


@pytest.mark.parametrize("rows,k,n", [(1, 64, 40), (5, 64, 40), (64, 512, 500), (300, 640, 500), (520, 144, 13056)])
def test_residuals_beside_the_output(rows, k, n):
    """What is added lies between the output's rows, before it, or is the output itself."""
    x, xs, w, ws = (t.to(DEV) for t in make(25, rows, k, n))
    add = torch.randn((rows, n), generator=torch.Generator().manual_seed(26)).to(DEV)
    want = mrt_df.i8_matmul(x, xs, w, ws, add=add)
    both = torch.zeros((rows, 2 * n), device=DEV)
    both[:, :n] = add
    mrt_df.i8_matmul(x, xs, w, ws, add=both[:, :n], out=both[:, n:])
    assert torch.equal(both[:, n:], want) and torch.equal(both[:, :n], add)
    line = torch.zeros((2 * rows, n), device=DEV)
    line[:rows] = add
    mrt_df.i8_matmul(x, xs, w, ws, add=line[:rows], out=line[rows:])
    assert torch.equal(line[rows:], want) and torch.equal(line[:rows], add)
    mrt_df.i8_matmul(x, xs, w, ws, add=line[:rows], out=line[:rows])
    assert torch.equal(line[:rows], want)
