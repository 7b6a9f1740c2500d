"""Products in 8-bit integers (mrt_i8_*) against 64 bits.

The sums are exact.  An output is the sum rounded to fp32, two products and a sum of fp32:
four roundings of 2^-24 of at most |y| + |add| each, then half a step of the type.
"""

from __future__ import annotations

import math

import pytest
import torch

import mrt_df
from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make(seed, rows, k, n):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-128, 128, (rows, k), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    return x, (torch.rand(rows, generator=g) + 0.5) / 128, w, (torch.rand(n, generator=g) + 0.5) / 128 / math.sqrt(k)


def check(got, want, add=None):
    size = want.abs() + (0 if add is None else 2 * add.double().abs())
    lim = 4 * 2.0 ** -24 * size + torch.finfo(got.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -20) + (
        2.0 ** -25 if got.dtype == torch.float16 else 0)
    err = (got.double() - want).abs()
    assert (err <= lim).all(), float((err / lim).max())


SIZES = [
    # rows k n
    (1, 16, 1), (1, 1024, 5632), (2, 1024, 100), (3, 128, 17), (16, 2816, 64), (17, 48, 50), (32, 768, 2000), (33, 1040, 31),
    (64, 4096, 33), (5, 512, 20000), (65, 64, 64), (100, 1024, 1000), (127, 208, 129), (256, 128, 256), (300, 2816, 1024),
    (1000, 144, 777), (513, 512, 4097), (2048, 1024, 2048), (1025, 272, 16385), (4099, 640, 4100), (70, 16, 3),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_matches_oracle(rows, k, n, dtype):
    x, xs, w, ws = make(1, rows, k, n)
    got = mrt_df.i8_matmul(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV), dtype=DT[dtype])
    # whole numbers below 2^53: the product in fp64 on the GPU is exact
    sums = (x.to(DEV).double() @ w.to(DEV).double().T.contiguous()).cpu()
    check(got.cpu(), sums * xs.double()[:, None] * ws.double())


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,k,n", [(1, 64, 5), (9, 256, 70), (40, 512, 130), (200, 320, 257), (700, 128, 1000), (3000, 96, 2055)])
def test_add_and_strides(rows, k, n, dtype):
    """Operands inside wider arrays, a residual of its own, one row for all, and in place."""
    x, xs, w, ws = make(2, rows, k, n)
    dt = DT[dtype]
    g = torch.Generator().manual_seed(3)
    add = torch.randn((rows, n), generator=g).to(dt)
    wx, ww = torch.full((rows, k + 32), 99, dtype=torch.int8), torch.full((n, k + 16), 99, dtype=torch.int8)
    wx[:, 16:k + 16], ww[:, :k] = x, w
    gx, gw, ga = wx.to(DEV)[:, 16:k + 16], ww.to(DEV)[:, :k], add.to(DEV)
    want = O.i8_matmul(x, xs, w, ws, add)
    check(mrt_df.i8_matmul(gx, xs.to(DEV), gw, ws.to(DEV), add=ga).cpu(), want, add)
    out = torch.full((rows, n + 3), 5.0, dtype=dt, device=DEV)
    mrt_df.i8_matmul(gx, xs.to(DEV), gw, ws.to(DEV), add=ga, out=out[:, 1:n + 1])
    check(out[:, 1:n + 1].cpu(), want, add)
    assert (out[:, 0] == 5).all() and (out[:, n + 1:] == 5).all()
    row = ga[:1].expand(rows, n)
    check(mrt_df.i8_matmul(gx, xs.to(DEV), gw, ws.to(DEV), add=row).cpu(), O.i8_matmul(x, xs, w, ws, add[:1]), add[:1])
    mrt_df.i8_matmul(gx, xs.to(DEV), gw, ws.to(DEV), add=ga, out=ga)
    check(ga.cpu(), want, add)


def test_largest_sums():
    """k 2^17 of -128 times -128: 2^31 - the sum that 32 bits just do not hold is refused by k, 2^31 - 2^14 fits."""
    k = 2 ** 17 - 16
    for rows in (2, 80):
        x = torch.full((rows, k), -128, dtype=torch.int8, device=DEV)
        w = torch.full((70, k), -128, dtype=torch.int8, device=DEV)
        w[1] = 127
        one = torch.ones(80, device=DEV)
        y = mrt_df.i8_matmul(x, one[:rows], w, one[:70], dtype=torch.float32).cpu()
        assert (y[:, 0] == float(k * 2 ** 14)).all() and (y[:, 1] == float(torch.tensor(-128 * 127 * k, dtype=torch.float32))).all()


@pytest.mark.parametrize("rows", [3, 40, 200])
def test_scales_that_are_not_finite(rows):
    """A row or channel with scale NaN is NaN, and no other."""
    x, xs, w, ws = make(4, rows, 64, 90)
    xs[1], ws[5], ws[6] = math.nan, math.nan, 0
    y = mrt_df.i8_matmul(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV), dtype=torch.float32).cpu()
    bad = torch.isnan(xs)[:, None] | torch.isnan(ws)
    assert torch.equal(torch.isnan(y), bad) and (y[:, 6][~torch.isnan(xs)] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,k", [(1, 16), (5, 64), (3, 1024), (2, 1040), (7, 4096), (2, 4112), (3, 16384), (2, 20000), (513, 256)])
def test_quantize(rows, k, dtype):
    g = torch.Generator().manual_seed(5)
    x = (torch.randn((rows, k), generator=g) * torch.exp2(torch.randint(-8, 8, (rows, 1), generator=g))).to(DT[dtype])
    if rows > 2:
        x[1] = 0
        x[2, k - 1] = math.nan
    if rows > 4:
        x[3, 5], x[4, 0] = math.inf, -math.inf
    wide = torch.zeros((rows, k + 16), dtype=x.dtype)
    wide[:, 8:k + 8] = x
    codes, scale = mrt_df.i8_quantize(wide.to(DEV)[:, 8:k + 8])
    want, ws = O.quantise(x)
    assert torch.equal(torch.isnan(scale.cpu()), torch.isnan(ws)) and torch.equal(scale.cpu().nan_to_num(), ws.nan_to_num())
    assert torch.equal(codes.cpu(), want)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_products_of_quantised_operands(dtype):
    """Near the product in 64 bits: each operand off by half a step, 1 / 254 of its row's largest."""
    g = torch.Generator().manual_seed(6)
    x, w = torch.randn((130, 512), generator=g).to(DT[dtype]), torch.randn((90, 512), generator=g).to(DT[dtype])
    cx, sx = mrt_df.i8_quantize(x.to(DEV))
    cw, sw = mrt_df.i8_quantize(w.to(DEV))
    y = mrt_df.i8_matmul(cx, sx, cw, sw, dtype=torch.float32).cpu().double()
    ax, aw = x.double().abs(), w.double().abs()
    hx, hw = ax.amax(1, keepdim=True) / 254 * 1.0001, aw.amax(1, keepdim=True) / 254 * 1.0001
    lim = hx * aw.sum(1) + ax.sum(1, keepdim=True) * hw.T + 512 * hx * hw.T
    assert ((y - x.double() @ w.double().T).abs() <= lim).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("aligned", [True, False], ids=["whole", "odd"])
@pytest.mark.parametrize("rows,k,n", [
    (520, 144, 13057), (520, 128, 13056), (4100, 128, 5891), (4100, 32, 5888),  # tiles of 256 x 256, one a block and several
    (257, 128, 13060), (1030, 160, 13056), (1024, 256, 13056),                  # 128 x 256
    (70, 128, 16385), (4100, 48, 1794), (4096, 384, 1792),                      # 128 x 128
    (4100, 128, 133), (130, 400, 16384), (128, 256, 16384),                     # 64 x 128
    (40, 128, 8198), (40, 1040, 8200), (40, 128, 102), (300, 640, 500),         # 32 rows
    (40, 1024, 100), (33, 4096, 999), (256, 2832, 1000), (64, 16384, 2000),     # 32 x 32, cut along k
])
def test_one_and_several_tiles_a_block(rows, k, n, aligned, dtype):
    """With and without a residual; results in 16-byte stores or one by one; nothing past the edges."""
    x, xs, w, ws = (t.to(DEV) for t in make(7, rows, k, n))
    sums = x.double() @ w.double().T.contiguous()
    want = sums * xs.double()[:, None] * ws.double()
    pad = 8 if aligned else 3
    out = torch.full((rows + 1, -(-n // 8) * 8 + pad), 7.0, dtype=DT[dtype], device=DEV)
    got = mrt_df.i8_matmul(x, xs, w, ws, dtype=DT[dtype], out=out[:rows, :n])
    check(got, want)
    assert (out[rows] == 7).all() and (out[:, n:] == 7).all()
    add = torch.randn((rows, out.shape[1]), generator=torch.Generator().manual_seed(8)).to(DEV, DT[dtype])[:, :n]
    check(mrt_df.i8_matmul(x, xs, w, ws, add=add, out=out[:rows, :n]), want + add.double(), add)
    assert (out[rows] == 7).all() and (out[:, n:] == 7).all()


def near_ties(rows, k, seed=9):
    """Rows of fp32 whose values are within four steps of a half of their row's scale, of all sizes."""
    g = torch.Generator().manual_seed(seed)
    most = (torch.rand(rows, generator=g) + 1) * torch.exp2(torch.randint(-118, 120, (rows,), generator=g).float())
    scale = most * (torch.tensor(1.0) / 127)
    half = torch.randint(-126, 126, (rows, k), generator=g).float() + 0.5
    x = (scale.double()[:, None] * half.double()).float().contiguous()
    x = (x.view(torch.int32) + torch.randint(-4, 5, (rows, k), generator=g, dtype=torch.int32)).view(torch.float32)
    x[:, 5] = most
    return x


def test_codes_near_ties():
    """The quotient's rounding decides: equal to the definition in every code."""
    x = near_ties(20000, 128)
    want, ws = O.quantise(x)
    codes, scale = mrt_df.i8_quantize(x.to(DEV))
    assert torch.equal(scale.cpu(), ws) and torch.equal(codes.cpu(), want)
