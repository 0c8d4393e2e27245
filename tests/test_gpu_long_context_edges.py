"""Calls over long contexts at the edges of what the documentation allows, and just past it."""
from __future__ import annotations

import pytest
import torch

import long_context_reference as ref
from conftest import PKG
from test_gpu_shared_prefix import Batch, _gen, _i32

pytestmark = pytest.mark.gpu


FALLING = [  # cu_seqlens_q of one group's sequences, new tokens at most
    ([4, 0, 2, 8], 6),             # rows before the group's first
    ([0, 9, 2, 6], 9),             # and behind its last
    ([150, 0, 60, 200], 140),
    ([0, 180, 20, 100], 180),
    ([0, 200] * 40 + [0], 200),    # every other sequence is all rows
]


@pytest.mark.parametrize("heads", [4, 32])
@pytest.mark.parametrize("case", FALLING, ids=[str(i) for i in range(len(FALLING))])
def test_new_tokens_that_fall(case, heads, dev):
    """cu_seqlens_q that falls: rows come from parts that were written, or are zero; a workspace of NaN would show."""
    cu, most = case
    gen = _gen(30)
    n = len(cu) - 1
    batch = Batch([(4, [210] * n)], 64, 2, gen)
    tokens = max(cu)
    q = torch.randn((tokens, heads, 128), generator=gen).to(torch.bfloat16).to(dev)
    need = PKG.shared_prefix_workspace_bytes(n, 1, tokens, heads, 2, batch.table.shape[1], 64, max_seqlen_q=most)
    room = torch.full((need,), 255, dtype=torch.uint8, device=dev)
    out = PKG.shared_prefix_attention(q, *batch.args(dev), _i32(cu, dev), max_seqlen_q=most, scale=0.09, workspace=room)
    assert torch.isfinite(out).all()


def test_rows_that_do_not_fall_beside(dev):
    """The group whose rows are in order keeps its result where another group's fall."""
    gen = _gen(31)
    batch = Batch([(3, [40, 30]), (2, [50, 60])], 64, 2, gen)
    new = [5, 7, 4, 3]
    q = torch.randn((19, 8, 128), generator=gen).to(torch.bfloat16)
    want, tol = ref.shared(q, batch.cache, batch.table, batch.lengths, new, 0.09)
    got = PKG.shared_prefix_attention(q.to(dev), *batch.args(dev), _i32([0, 5, 12, 16, 19], dev), max_seqlen_q=7, scale=0.09)
    assert ((got.cpu().double() - want).abs() <= tol).all()
    # the second group: rows 12 .. 18, then a sequence that ends before it starts
    got = PKG.shared_prefix_attention(q.to(dev), *batch.args(dev), _i32([0, 5, 12, 19, 12], dev), max_seqlen_q=7, scale=0.09)
    assert ((got.cpu().double() - want).abs() <= tol)[:12].all() and torch.isfinite(got).all()
