"""Verification of drafted tokens (mrt_draft_verify) against 64 bits: whole numbers, equal.

Both sides compare sums over the vocabulary in 64 bits whose order differs, so that a random
number would have to lie within some 2^-45 of a border for them to differ; those here are
multiples of 2^-24.  Where inputs put one right on a border, all sums are exact.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import mrt_df
from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def random_tree(rng, nodes):
    return [-1] + [t - 1 if rng.random() < 0.4 else int(rng.integers(-1, t)) for t in range(1, nodes)]


def make(seed, dtype, rows, nodes, vocab, tree, sure, near=0.5):
    rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    logits = torch.randn((rows, nodes + 1, vocab), generator=g) * 2
    target = (logits + near * torch.randn(logits.shape, generator=g)).softmax(-1).to(DT[dtype])
    draft = logits[:, :nodes].softmax(-1).to(DT[dtype])
    parents = torch.tensor([random_tree(rng, nodes) if tree else list(range(-1, nodes - 1)) for _ in range(rows)],
                           dtype=torch.int32)
    rows_of = draft.float().gather(1, (parents.long() + 1)[..., None].expand(rows, nodes, vocab)).reshape(-1, vocab)
    tokens = torch.multinomial(rows_of.clamp_min(1e-9), 1, generator=g).view(rows, nodes).to(torch.int32)
    return dict(target=target, draft=None if sure else draft, tokens=tokens,
                uniforms=torch.rand((rows, nodes + 1), generator=g), parents=parents if tree else None)


def check(s):
    d = {n: x.to(DEV) if isinstance(x, torch.Tensor) else x for n, x in s.items()}
    got = [x.cpu() for x in mrt_df.draft_verify(d["target"], d["draft"], d["tokens"], d["uniforms"], parents=d["parents"])]
    paths, last = O.draft_verify(**s)
    nodes = s["tokens"].shape[1]
    assert got[0].tolist() == [p + [-1] * (nodes - len(p)) for p in paths]
    assert got[1].tolist() == [len(p) for p in paths]
    assert got[2].tolist() == last
    return paths, last


SIZES = [(1, 1, 1), (1, 1, 2), (3, 2, 7), (4, 16, 1024), (2, 5, 1000), (7, 64, 333), (2, 16, 29824), (2, 3, 100003), (40, 8, 64)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("sure", [False, True], ids=["drawn", "sure"])
@pytest.mark.parametrize("tree", [False, True], ids=["chain", "tree"])
@pytest.mark.parametrize("rows,nodes,vocab", SIZES)
def test_matches_oracle(rows, nodes, vocab, tree, sure, dtype):
    for seed in range(3):
        check(make(seed, dtype, rows, nodes, vocab, tree, sure, near=(0.05, 0.5, 2.0)[seed]))


def test_random_numbers_at_their_ends():
    for u in (0.0, 1.0 - 2.0 ** -24, 1.0):
        for sure in (False, True):
            s = make(5, "fp32", 4, 6, 300, True, sure)
            s["uniforms"][:] = u
            check(s)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_borders(dtype):
    """Dyadic probabilities: sums are exact, and a random number on a border belongs to the next token."""
    p = torch.zeros((8, 3, 520), dtype=DT[dtype])
    p[:, :, [3, 5, 259, 519]] = torch.tensor([0.25, 0.25, 0.125, 0.375], dtype=DT[dtype])
    u = torch.zeros((8, 3))
    u[:, 2] = torch.tensor([0.0, 0.25, 0.5, 0.625, 0.2499, 0.4999, 0.6249, 0.9999])
    tokens = torch.full((8, 2), 4, dtype=torch.int32)  # nothing there: rejected
    s = dict(target=p, draft=None, tokens=tokens, uniforms=u, parents=None)
    assert check(s)[1] == [3, 5, 259, 519, 3, 5, 259, 519]
    s = dict(s, draft=p[:, :2].flip(-1).contiguous())
    check(s)


def test_equal_distributions_accept_everything():
    s = make(6, "fp32", 5, 20, 500, False, False, near=0.0)
    paths, _ = check(s)
    assert paths == [list(range(20))] * 5


def test_nothing_left():
    """A draft that covers the target and is rejected, a target without weight, NaN and infinities."""
    s = make(7, "fp32", 6, 3, 400, True, False)
    s["parents"][:] = -1
    s["draft"][0] = s["target"][0, :3]
    s["tokens"][0] = 9
    s["uniforms"][0, :3] = 1.0  # not below 1: rejects what it should accept
    s["target"][1] = 0
    s["target"][2, :, ::3], s["draft"][2, :, ::5] = math.nan, math.inf
    s["target"][3, :, 7], s["target"][3, :, 8] = -1.0, math.inf
    s["target"][4, 0, 1:] = 0
    paths, last = check(s)
    assert last[1] == -1 and paths[1] == [] and last[4] == 0


def test_absent_nodes_and_tokens():
    """Parents that are not earlier nodes, tokens outside the vocabulary: never accepted, nothing drawn for them."""
    s = make(8, "fp32", 4, 10, 200, True, False, near=0.0)
    s["uniforms"][:, :10] = 0
    s["parents"][0] = torch.tensor([0, 5, -2, -1, 3, 4, 99, 5, 2 ** 31 - 1, 7])
    s["parents"][1] = torch.arange(-1, 9)
    s["tokens"][1, 4] = 200
    s["tokens"][2, 0] = -1
    s["tokens"][3] = -2 ** 31
    paths, _ = check(s)
    assert paths[0] == [3, 4, 5, 7, 9] and paths[1] == [0, 1, 2, 3] and paths[3] == []


def test_strides_and_one_tree_for_all():
    s = make(9, "bf16", 3, 9, 333, True, False)
    s["parents"] = s["parents"][1].contiguous()
    wide = torch.zeros((3, 12, 340), dtype=torch.bfloat16)
    wide[:, 1:11, 5:338] = s["target"]
    paths, last = O.draft_verify(**s)
    d = {n: x.to(DEV) for n, x in s.items()}
    got = mrt_df.draft_verify(wide.to(DEV)[:, 1:11, 5:338], d["draft"].transpose(0, 1).contiguous().transpose(0, 1), d["tokens"],
                              d["uniforms"], parents=d["parents"])
    assert got[1].tolist() == [len(p) for p in paths] and got[2].tolist() == last


def test_draws_follow_the_target():
    """Accepted or drawn, the first token has the target's distribution: chi-square over 4000 trees."""
    rows, vocab = 4000, 12
    g = torch.Generator().manual_seed(3)
    p = torch.randn(vocab, generator=g).softmax(-1)
    q = torch.randn(vocab, generator=g).softmax(-1)
    tokens = torch.multinomial(q.expand(rows, vocab), 3, replacement=True, generator=g).to(torch.int32)
    u = torch.rand((rows, 4), generator=g)
    parents = torch.tensor([-1, -1, -1], dtype=torch.int32)
    path, count, last = (x.cpu() for x in mrt_df.draft_verify(
        p.expand(rows, 4, vocab).contiguous().to(DEV), q.expand(rows, 3, vocab).contiguous().to(DEV), tokens.to(DEV), u.to(DEV),
        parents=parents.to(DEV)))
    first = torch.where(count > 0, tokens.gather(1, path[:, :1].clamp_min(0).long())[:, 0], last)
    seen = torch.bincount(first.long(), minlength=vocab).double()
    want = p.double() * rows
    chi = float(((seen - want) ** 2 / want).sum())
    assert chi < 31.3  # 11 degrees of freedom: 1 in 1000
    assert (count > 0).float().mean() > 0.5


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("sure", [False, True], ids=["drawn", "sure"])
def test_many_rejections_over_a_large_vocabulary(sure, dtype):
    """Up to 20 children of one slot rejected, then some of the next: more passes than are
    made ahead of the last launch, beside sequences that end at once."""
    s = make(11, dtype, 5, 30, 50001, True, sure, near=2.0)
    s["parents"][:] = torch.tensor([-1] * 20 + [19] * 10)
    s["uniforms"][:, :30] = 1.0 - 2.0 ** -24
    s["uniforms"][0, 0] = 0  # its first child, which has none
    s["uniforms"][1, 19] = 0
    s["uniforms"][2, 4] = 0.3
    paths, _ = check(s)
    assert paths[0] == [0] and any(not p or p[0] > 6 for p in paths)


def test_many_sequences_over_a_large_vocabulary():
    """As many as there are CUs: a block each, whatever the vocabulary."""
    s = make(12, "bf16", 257, 1, 40009, False, False)
    check(s)


def test_passes_do_not_depend_on_how_many_blocks_make_them():
    """The same sequence among few, many blocks each, and among so many that one block makes all."""
    s = make(13, "fp32", 2, 9, 40960, True, False, near=2.0)
    few = mrt_df.draft_verify(*(s[n].to(DEV) for n in ("target", "draft", "tokens", "uniforms")), parents=s["parents"].to(DEV))
    many = {n: x.to(DEV).repeat(128, *[1] * (x.dim() - 1)) for n, x in s.items()}
    got = mrt_df.draft_verify(many["target"], many["draft"], many["tokens"], many["uniforms"], parents=many["parents"])
    for x, y in zip(few, got):
        assert torch.equal(x.repeat(128, *[1] * (x.dim() - 1)), y)
