"""The last draw of mrt_draft_verify where the vocabulary ends in tokens without weight.

Sums of segments that hold nothing add nothing, whatever lane has them: a random number of 1, or one
next to it, draws the last token that has any weight, and never none.
"""

from __future__ import annotations

import pytest
import torch

import mrt_df
from test_gpu_verify import DEV, DT, check

pytestmark = pytest.mark.gpu


def ends(seed, dtype, rows, vocab, weighted, kind):
    """Sequences of one node that is not accepted; the tokens from `weighted` on have no weight."""
    g = torch.Generator().manual_seed(seed)
    target = torch.rand((rows, 2, vocab), generator=g)
    if kind == "holes":  # whole stretches without weight between others
        target *= (torch.rand((rows, 2, -(-vocab // 700)), generator=g) < 0.5).repeat_interleave(700, -1)[..., :vocab]
    target[..., weighted:] = 0
    target = (target / target.sum(-1, keepdim=True)).to(DT[dtype])
    draft = None
    if kind == "drawn":  # what is left of the target has holes of its own
        draft = torch.rand((rows, 1, vocab), generator=g)
        draft[..., weighted:] = 0
        draft = (draft / draft.sum(-1, keepdim=True)).to(DT[dtype])
    return dict(target=target, draft=draft, tokens=torch.full((rows, 1), vocab - 1, dtype=torch.int32),
                uniforms=torch.ones((rows, 2)), parents=None)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("kind", ["sure", "drawn", "holes"])
@pytest.mark.parametrize("vocab,weighted", [(20000, 9000), (20000, 19001), (23999, 301), (50001, 23000), (50001, 49000), (131072, 70003)])
def test_tokens_without_weight_at_the_end(vocab, weighted, kind, dtype):
    for seed in range(2):
        s = ends(seed, dtype, 48, vocab, weighted, kind)
        some = (s["target"][:, 0] > 0).any(-1).tolist()
        assert [x >= 0 for x in check(s)[1]] == some
        s["uniforms"][:, 1] = 1.0 - 2.0 ** -24
        check(s)


@pytest.mark.parametrize("vocab", [20000, 50001])
def test_many_sequences_draw_their_last(vocab):
    """Without a node's test in the way, few tokens with weight, anywhere."""
    rows = 250
    g = torch.Generator().manual_seed(5)
    target = torch.rand((rows, 2, vocab), generator=g) * (torch.rand((rows, 2, vocab), generator=g) < 0.002)
    target[..., vocab // 2:] = 0
    target /= target.sum(-1, keepdim=True)
    tokens = torch.full((rows, 1), -1, dtype=torch.int32)
    _, _, token = mrt_df.draft_verify(target.to(DEV), None, tokens.to(DEV), torch.ones((rows, 2), device=DEV))
    last = (target[:, 0] > 0).long().mul(torch.arange(1, vocab + 1)).amax(-1) - 1
    assert token.cpu().long().tolist() == last.tolist()
