"""A PagedCache names its tensors for good: what they hold may change, which they are may not."""

from __future__ import annotations

import pytest
import torch

import mrt_df

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make():
    k, v = (torch.randn((5, 2, 16, 64), device=DEV).bfloat16() for _ in range(2))
    table = torch.tensor([[0, 3], [1, 2]], dtype=torch.int32, device=DEV)
    return k, v, table, torch.tensor([3, 17], dtype=torch.int32, device=DEV)


def test_names_are_fixed():
    k, v, table, length = make()
    cache = mrt_df.PagedCache(k, v, table, length)
    assert cache.k is k and cache.v is v and cache.table is table and cache.length is length
    assert cache.k_scale is None and cache.v_scale is None
    assert cache.rows == 2 and cache.row_pages == 2 and tuple(cache.shape) == (5, 2, 16, 64) and cache.index == 0
    for name in ("k", "v", "table", "length", "k_scale", "v_scale", "rows", "row_pages", "shape", "index", "kind", "grown"):
        with pytest.raises(AttributeError):
            setattr(cache, name, length)


def test_contents_may_change():
    """Lengths that grow in place are seen, as those of a new object are."""
    k, v, table, length = make()
    cache = mrt_df.PagedCache(k, v, table, length)
    q = torch.randn((2, 1, 4, 64), device=DEV).bfloat16()
    length += 5
    got = mrt_df.paged_attention(q, cache)[0]
    want = mrt_df.paged_attention(q, mrt_df.PagedCache(k, v, table, length.clone()))[0]
    length -= 5
    other = mrt_df.paged_attention(q, cache)[0]
    assert torch.equal(got, want) and not torch.equal(got, other)
