"""Outputs of a server's operators that overlap in part, at an offset: refused without a GPU, each with
its own message; operands that only lie between each other's rows are not."""

from __future__ import annotations

import pytest

import mrt_df
from test_serving_abi import INVALID, P, V, attention, pages, product, verify

pytestmark = pytest.mark.filterwarnings("ignore")


@pytest.fixture(scope="module")
def lib():
    return mrt_df.load_library()


def says(lib, code, text):
    return code == INVALID and text in lib.mrt_last_error().decode()


# q (2, 4, 4, 64) bf16 at P, rows of 4 x 1024 elements
OUTS = {
    "a head on": dict(out=P + 128), "a token on": dict(out=P + 2048), "a row on": dict(out=P + 8192),
    "a token before": dict(out=P + 65536 - 2048, q=P + 65536),
    "the last vector": dict(out=P + 2 * (4096 + 3 * 1024 + 3 * 64)),
    "another layout": dict(out=P + 2048, os=(1024, 256, 64)),
    "heads first": dict(out=P + 16, os=(1024, 64, 256)),
    "one q for all": dict(out=P + 64, qs=(0, 0, 64)),
}
APART = {
    "behind it": dict(out=P + 2 * 8192), "right before it": dict(q=P + 16384, out=P),
    "heads side by side": dict(qs=(4096, 1024, 128), os=(4096, 1024, 128), out=P + 128),
    "in one product's rows": dict(out=P + 512),
    "another layout behind it": dict(out=P + 2 * 8192, os=(1024, 64, 256)),
}


def paged(lib, **kw):
    return lib.mrt_paged_attention(pages(), attention(**dict(dict(lse=0), **kw)), None, 0, 0, None)


@pytest.mark.parametrize("case", OUTS)
def test_attention_out_of_q(lib, case):
    assert says(lib, paged(lib, **OUTS[case]), "memory of its own")


@pytest.mark.parametrize("case", APART)
def test_attention_beside_q(lib, case):
    """Gets past the checks of q and out, to the last of all: a bias with no table."""
    assert says(lib, paged(lib, fresh=P + 2, **APART[case]), "fresh and lse must be 4-byte aligned")


def test_attention_lse(lib):
    assert says(lib, paged(lib, lse=V + 4), "lse overlaps out")
    assert says(lib, paged(lib, lse=V - 4), "lse overlaps out")


# k and v (2, 2, 2, 64) bf16 of paged_read: rows of 1024, tokens of 512, heads of 128 elements

def store_of(k=P, v=V, kst=(1024, 512, 128), vst=(1024, 512, 128), start=0):
    return mrt_df._STORE_STRUCT.pack(k, *kst, v, *vst, 0, start, 0, 2, 1)


def test_read_into_rows_laid_out_otherwise(lib):
    for kw in (dict(v=P + 256, vst=(1024, 256, 512)), dict(v=P + 1024, vst=(512, 256, 64)), dict(k=P + 2048, v=P, vst=(2048, 1024, 64))):
        assert says(lib, lib.mrt_paged_read(pages(), store_of(**kw), 0, None), "overlaps itself or the other")


def test_written_lengths(lib):
    """length_out (2) int32 against the lengths and counts that other blocks read."""
    def write(length=P, fresh=0, out=0):
        return lib.mrt_paged_write(pages(length=length), store_of(k=V, v=V + (1 << 20))[:64] +
                                   mrt_df.struct.pack("PPPii", fresh, 0, out, 2, 1), 0, None)
    for kw in (dict(out=P + 4), dict(out=P - 4), dict(out=P), dict(out=V + 4, fresh=V), dict(out=V - 4, fresh=V)):
        assert says(lib, write(**kw), "array of its own")


def test_written_scales(lib):
    """(8, 2, 16) fp32 each."""
    for vs in (P + 16, P - 16, P + 1024 - 16):
        c = pages(dtype=3, ks=P, vs=vs, k=V, v=V + (1 << 20))
        assert says(lib, lib.mrt_paged_write(c, store_of(), 0, None), "k_scale and v_scale overlap")


def test_outputs_of_the_verification(lib):
    """accepted (2, 2), count (2) and token (2) int32."""
    for kw in (dict(accepted=P, count=P + 12, token=V), dict(accepted=P + 4, count=P, token=V), dict(accepted=P, count=V, token=P + 8),
               dict(accepted=P, count=V, token=V + 4), dict(accepted=P, count=V + 4, token=V)):
        assert says(lib, lib.mrt_draft_verify(verify(target=V << 4, draft=V << 5, **kw), None, 0, 0, None), "arrays of their own")


def test_residuals(lib):
    """add and out (4, 32) bf16, out at V: the very same, or apart."""
    for kw in (dict(add=V + 8), dict(add=V + 64), dict(add=V - 2), dict(add=V + 64, ld=(64, 64, 0, 32)),
               dict(add=V + 16, ld=(64, 64, 64, 64)), dict(add=V + 2, rows=1), dict(add=V + 128, ld=(64, 64, 64, 32))):
        assert says(lib, lib.mrt_i8_matmul(product(**kw), 0, None), "add overlaps out")
