"""Arguments that the operators over pages, 8-bit products and the verification refuse, without a
GPU: a status code and a message before any device call, and ValueError from the binding."""

from __future__ import annotations

import ctypes

import pytest
import torch

import mrt_df

INVALID = 1
P = 0x1000  # a pointer that no refused call follows
V = 0x10000000  # another, far from it


@pytest.fixture(scope="module")
def lib():
    return mrt_df.load_library()


def refused(lib, code):
    assert code == INVALID and lib.mrt_last_error()


def pages(k=P, v=V, ks=0, vs=0, table=P, length=P, ps=2048, hs=1024, ss=64, ts=4, n=8, rows=2, rp=4, kv=2, size=16, d=64,
          dtype=1):
    return mrt_df._PAGES_STRUCT.pack(k, v, ks, vs, table, length, ps, hs, ss, ts, n, rows, rp, kv, size, d, dtype)


I8 = dict(dtype=3, ks=P, vs=V)
BAD_PAGES = {
    "null k": dict(k=0), "null v": dict(v=0), "null table": dict(table=0), "null length": dict(length=0),
    "misaligned k": dict(k=P + 8), "misaligned v": dict(v=V + 4), "misaligned table": dict(table=P + 2),
    "misaligned length": dict(length=P + 1), "negative rows": dict(rows=-1), "no heads": dict(kv=0), "no pages": dict(n=0),
    "no pages of a row": dict(rp=0), "page size": dict(size=24), "no page size": dict(size=0),
    "large page size": dict(size=(1 << 16) + 16), "odd d": dict(d=60), "wide d": dict(d=264), "no d": dict(d=0),
    "dtype": dict(dtype=4), "stride": dict(ss=68), "negative stride": dict(hs=-1024), "table stride": dict(ts=-1),
    "too long": dict(rp=1 << 20, size=1 << 11), "too many heads": dict(rows=1 << 12, kv=1 << 9),
    "wide slots": dict(ss=(1 << 24) + 64), "codes without scales": dict(dtype=3), "codes with one scale": dict(dtype=3, ks=P), "misaligned scales": dict(I8, ks=P + 4),
    "d of codes": dict(I8, d=72), "stride of codes": dict(I8, ss=72),
}


def store(k=P, v=V, st=(1024, 512, 128), fresh=0, start=0, length=0, tokens=2, dtype=1):
    return mrt_df._STORE_STRUCT.pack(k, *st, v, *st, fresh, start, length, tokens, dtype)


BAD_STORES = {
    "null k": dict(k=0), "null v": dict(v=0), "misaligned k": dict(k=P + 8), "stride": dict(st=(1024, 512, 68)),
    "negative stride": dict(st=(-1024, 512, 128)), "no tokens": dict(tokens=0), "many tokens": dict(tokens=1 << 26),
    "dtype": dict(dtype=3), "another dtype": dict(dtype=2), "misaligned fresh": dict(fresh=P + 2),
    "misaligned start": dict(start=P + 2), "misaligned length": dict(length=P + 2),
}


def attention(q=P, out=V, qs=(4096, 1024, 64), os=(4096, 1024, 64), fresh=0, lse=P, bias=0, buckets=0, tokens=4, heads=4,
              dtype=1, scale=1.0):
    return mrt_df._PAGED_STRUCT.pack(q, *qs, out, *os, fresh, lse, bias, buckets, tokens, heads, dtype, scale)


BAD_ATTENTION = {
    "null q": dict(q=0), "null out": dict(out=0), "misaligned q": dict(q=P + 4), "stride": dict(qs=(4096, 1020, 64)),
    "negative stride": dict(os=(4096, 1024, -64)), "out in place": dict(out=P), "overlapping out": dict(os=(4096, 0, 64)), "no tokens": dict(tokens=0),
    "many tokens": dict(tokens=65), "heads": dict(heads=3), "no heads": dict(heads=0), "bias without buckets": dict(bias=P),
    "too many buckets": dict(bias=P, buckets=(1 << 18) + 1), "misaligned bias": dict(bias=P + 2, buckets=4),
    "large bias": dict(bias=P, heads=1 << 14, buckets=1 << 17), "another dtype": dict(dtype=0), "dtype": dict(dtype=3), "misaligned lse": dict(lse=P + 1), "misaligned fresh": dict(fresh=P + 2),
}


def verify(target=P, draft=P, strides=(300, 100, 200, 100), tokens=P, parents=0, ps=0, u=P, accepted=P, count=V, token=V + 64,
           rows=2, nodes=2, vocab=100, dtype=0):
    return mrt_df._VERIFY_STRUCT.pack(target, draft, *strides, tokens, parents, ps, u, accepted, count, token, rows, nodes,
                                      vocab, dtype)


BAD_VERIFY = {
    "null target": dict(target=0), "null tokens": dict(tokens=0), "null uniforms": dict(u=0), "null accepted": dict(accepted=0),
    "null count": dict(count=0), "null token": dict(token=0), "misaligned target": dict(target=P + 2),
    "misaligned draft": dict(draft=P + 1), "misaligned tokens": dict(tokens=P + 2), "misaligned parents": dict(parents=P + 1),
    "negative stride": dict(strides=(300, -100, 200, 100)), "parents stride": dict(ps=-1), "negative rows": dict(rows=-1),
    "many rows": dict(rows=(1 << 20) + 1), "no nodes": dict(nodes=0), "many nodes": dict(nodes=65), "no vocab": dict(vocab=0),
    "large vocab": dict(vocab=(1 << 24) + 1), "dtype": dict(dtype=3), "outputs alike": dict(count=P),
    "outputs alike too": dict(token=V),
}


def product(x=P, xs=P, w=P, ws=P, add=0, out=V, ld=(64, 64, 32, 32), rows=4, n=32, k=64, dtype=1):
    return mrt_df._I8_STRUCT.pack(x, xs, w, ws, add, out, *ld, rows, n, k, dtype)


BAD_PRODUCTS = {
    "null x": dict(x=0), "null x_scale": dict(xs=0), "null w": dict(w=0), "null w_scale": dict(ws=0), "null out": dict(out=0),
    "misaligned x": dict(x=P + 8), "misaligned w": dict(w=P + 8), "misaligned scale": dict(xs=P + 2), "misaligned out": dict(out=V + 1),
    "misaligned add": dict(add=P + 1), "negative rows": dict(rows=-1), "many rows": dict(rows=1 << 24), "no n": dict(n=0),
    "large n": dict(n=(1 << 26) + 1), "odd k": dict(k=24), "no k": dict(k=0), "large k": dict(k=1 << 17, ld=(1 << 17, 1 << 17, 32, 32)),
    "short ldx": dict(ld=(48, 64, 32, 32)), "odd ldx": dict(ld=(72, 64, 32, 32)), "short ldw": dict(ld=(64, 48, 32, 32)),
    "odd ldw": dict(ld=(64, 72, 32, 32)), "short ldo": dict(ld=(64, 64, 32, 31)), "negative lda": dict(add=P, ld=(64, 64, -32, 32)),
    "long ldx": dict(ld=(1 << 24, 64, 32, 32)), "long ldw": dict(ld=(64, 1 << 24, 32, 32)),
    "in place with another stride": dict(add=V, ld=(64, 64, 0, 32)), "dtype": dict(dtype=3),
    "too many tiles": dict(rows=(1 << 24) - 1, n=1 << 26, ld=(64, 64, 1 << 26, 1 << 26)),
}


@pytest.mark.parametrize("bad", BAD_PAGES)
def test_pages(lib, bad):
    c = pages(**BAD_PAGES[bad])
    refused(lib, lib.mrt_paged_write(c, store(), 0, None))
    refused(lib, lib.mrt_paged_read(c, store(), 0, None))
    refused(lib, lib.mrt_paged_attention(c, attention(), P, 1 << 30, 0, None))


@pytest.mark.parametrize("bad", BAD_STORES)
def test_stores(lib, bad):
    refused(lib, lib.mrt_paged_write(pages(), store(**BAD_STORES[bad]), 0, None))
    refused(lib, lib.mrt_paged_read(pages(), store(**BAD_STORES[bad]), 0, None))


def test_what_is_written_overlaps(lib):
    for bad in (dict(ps=1024), dict(hs=512), dict(hs=0), dict(ss=32), dict(v=P), dict(v=P + 2048), dict(I8, ks=P, vs=P)):
        refused(lib, lib.mrt_paged_write(pages(**bad), store(), 0, None))
    for bad in (dict(st=(1024, 512, 0)), dict(st=(0, 512, 128)), dict(v=P), dict(v=P + 64)):
        refused(lib, lib.mrt_paged_read(pages(), store(**bad), 0, None))
    refused(lib, lib.mrt_paged_write(pages(length=P + 64), store(length=P + 64), 0, None))
    refused(lib, lib.mrt_paged_write(pages(), store(length=V, fresh=V), 0, None))


@pytest.mark.parametrize("bad", BAD_ATTENTION)
def test_attention(lib, bad):
    refused(lib, lib.mrt_paged_attention(pages(), attention(**BAD_ATTENTION[bad]), P, 1 << 30, 0, None))


def test_workspaces_and_null_arguments(lib):
    refused(lib, lib.mrt_paged_attention(None, attention(), None, 0, 0, None))
    refused(lib, lib.mrt_paged_attention(pages(), None, None, 0, 0, None))
    refused(lib, lib.mrt_paged_write(pages(), None, 0, None))
    refused(lib, lib.mrt_paged_read(None, store(), 0, None))
    refused(lib, lib.mrt_draft_verify(None, P, 1 << 30, 0, None))
    refused(lib, lib.mrt_i8_matmul(None, 0, None))
    size = ctypes.c_size_t()
    refused(lib, lib.mrt_paged_attention_workspace(pages(), 4, 4, None))
    refused(lib, lib.mrt_paged_attention_workspace(pages(), 4, 65, ctypes.byref(size)))
    refused(lib, lib.mrt_paged_attention_workspace(pages(dtype=5), 4, 4, ctypes.byref(size)))
    long = pages(rp=10000, ts=10000)
    assert lib.mrt_paged_attention_workspace(long, 4, 4, ctypes.byref(size)) == 0 and size.value > 0
    refused(lib, lib.mrt_paged_attention(long, attention(), None, 0, 0, None))
    refused(lib, lib.mrt_paged_attention(long, attention(), P, size.value - 1, 0, None))
    refused(lib, lib.mrt_paged_attention(long, attention(), P + 4, size.value, 0, None))
    assert lib.mrt_paged_attention_workspace(pages(), 4, 4, ctypes.byref(size)) == 0 and size.value == 0
    many = pages(rows=1 << 20, kv=1)
    refused(lib, lib.mrt_paged_attention_workspace(many, 64, 64, ctypes.byref(size)))
    refused(lib, lib.mrt_paged_attention(many, attention(tokens=64, heads=64), P, 1 << 40, 0, None))


@pytest.mark.parametrize("bad", BAD_VERIFY)
def test_verify(lib, bad):
    refused(lib, lib.mrt_draft_verify(verify(**BAD_VERIFY[bad]), P, 1 << 30, 0, None))


def test_verify_workspace(lib):
    size = ctypes.c_size_t()
    refused(lib, lib.mrt_draft_verify_workspace(None, ctypes.byref(size)))
    refused(lib, lib.mrt_draft_verify_workspace(verify(), None))
    refused(lib, lib.mrt_draft_verify_workspace(verify(nodes=65), ctypes.byref(size)))
    assert lib.mrt_draft_verify_workspace(verify(), ctypes.byref(size)) == 0 and size.value == 0
    large = verify(vocab=100000, parents=P)
    assert lib.mrt_draft_verify_workspace(large, ctypes.byref(size)) == 0 and size.value > 0
    refused(lib, lib.mrt_draft_verify(large, None, 0, 0, None))
    refused(lib, lib.mrt_draft_verify(large, P, size.value - 1, 0, None))
    refused(lib, lib.mrt_draft_verify(large, P + 8, size.value, 0, None))


@pytest.mark.parametrize("bad", BAD_PRODUCTS)
def test_products(lib, bad):
    refused(lib, lib.mrt_i8_matmul(product(**BAD_PRODUCTS[bad]), 0, None))


def test_quantize(lib):
    good = dict(src=P, ld=64, rows=4, k=64, dtype=1, codes=V, ldc=64, scales=P)
    for bad in (dict(src=0), dict(codes=0), dict(scales=0), dict(src=P + 8), dict(codes=V + 8), dict(scales=P + 2), dict(ld=56),
                dict(ld=68), dict(ldc=48), dict(ldc=72), dict(k=24), dict(k=0), dict(k=1 << 17), dict(rows=-1), dict(rows=1 << 24), dict(dtype=7)):
        refused(lib, lib.mrt_i8_quantize(*dict(good, **bad).values(), 0, None))


def test_no_rows_is_no_work(lib):
    empty = pages(rows=0, k=0, v=0, table=0, length=0)
    assert lib.mrt_paged_write(empty, store(k=0, v=0), 0, None) == 0
    assert lib.mrt_paged_read(empty, store(k=0, v=0), 0, None) == 0
    assert lib.mrt_paged_attention(empty, attention(q=0, out=0, lse=0), None, 0, 0, None) == 0
    assert lib.mrt_draft_verify(verify(rows=0, target=0, tokens=0, u=0, accepted=0, count=0, token=0), None, 0, 0, None) == 0
    assert lib.mrt_i8_matmul(product(rows=0, x=0, xs=0, out=0), 0, None) == 0
    assert lib.mrt_i8_quantize(None, 64, 0, 64, 1, None, 64, None, 0, None) == 0


def test_binding_refuses_cpu_tensors_and_wrong_shapes():
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    table, length = torch.zeros((1, 4), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        mrt_df.PagedCache(k, k.clone(), table, length)
    with pytest.raises(ValueError):
        mrt_df.PagedCache(k.double(), k.double(), table, length)
    with pytest.raises(ValueError):
        mrt_df.PagedCache(k[0], k[0], table, length)
    x = torch.zeros((2, 64), dtype=torch.int8)
    with pytest.raises(ValueError):
        mrt_df.i8_matmul(x, torch.zeros(2), x, torch.zeros(2))
    with pytest.raises(ValueError):
        mrt_df.i8_matmul(x, torch.zeros(2), x[:, :32], torch.zeros(2))
    with pytest.raises(ValueError):
        mrt_df.i8_quantize(x.float())
    with pytest.raises(ValueError):
        mrt_df.draft_verify(torch.zeros((1, 3, 9)), None, torch.zeros((1, 2), dtype=torch.int32), torch.zeros((1, 3)))
