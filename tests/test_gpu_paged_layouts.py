"""Operands of the operators over pages that lie between each other in one buffer."""

from __future__ import annotations

import pytest
import torch

import mrt_df
from test_gpu_paged import DEV, call, check, make, on_gpu, pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("store", ["bf16", "i8-fp32"])
def test_read_side_by_side(store):
    """k and v of an entry next to each other, and in two layouts behind each other."""
    c, s = make(31, store, 2, 2, 2, 64, 3, [40, 21])
    d = on_gpu(c)
    ref = [torch.full((2, 2, 40, 64), 3.0, dtype=s["q"].dtype, device=DEV) for _ in range(2)]
    mrt_df.paged_read(pages(d), *ref)
    both = torch.full((2, 2, 40, 128), 3.0, dtype=s["q"].dtype, device=DEV)
    mrt_df.paged_read(pages(d), both[..., :64], both[..., 64:])
    assert torch.equal(both[..., :64], ref[0]) and torch.equal(both[..., 64:], ref[1])
    one = torch.full((2 * 2 * 2 * 40 * 64,), 3.0, dtype=s["q"].dtype, device=DEV)
    k, v = one[:one.numel() // 2].view(2, 2, 40, 64), one[one.numel() // 2:].view(2, 40, 2, 64).transpose(1, 2)
    mrt_df.paged_read(pages(d), k, v)
    assert torch.equal(k, ref[0]) and torch.equal(v, ref[1])


@pytest.mark.parametrize("store", ["bf16", "fp32", "i8-fp16"])
def test_attention_into_the_rows_of_q(store):
    """q and the output are columns of the same rows."""
    c, s = make(32, store, 2, 6, 2, 64, 3, [130, 70])
    wide = torch.full((2, 3, 14, 64), 5.0, dtype=s["q"].dtype)
    wide[:, :, 1:7] = s["q"]
    g, d = wide.to(DEV), on_gpu(c)
    out, lse = mrt_df.paged_attention(g[:, :, 1:7], pages(d), scale=s["scale"], out=g[:, :, 8:])
    torch.cuda.synchronize()
    check(c, s, store, (out.cpu(), lse.cpu()))
    assert torch.equal(g[:, :, 1:7].cpu(), s["q"]) and (g[:, :, [0, 7]] == 5).all()
    want = call(c, s)
    assert torch.equal(out.cpu(), want[0]) and torch.equal(lse.cpu(), want[1])
