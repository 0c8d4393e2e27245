"""Calls over long contexts at the edges of what the documentation allows, and just past it."""
from __future__ import annotations

import pytest
import torch

import long_context_reference as ref
from conftest import PKG
from test_gpu_block_sparse import _random_selection
from test_gpu_shared_prefix import Batch, _check, _gen, _i32

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


# ---------------------------------------------------------------------------
# forms of the kernels that few shapes take
# ---------------------------------------------------------------------------
CAPPED = [  # groups (own tokens, the new included), new tokens (None: one each), page, heads, kv heads
    ([(4, [100, 7, 30])], None, 64, 80, 4),              # 20 heads a kv head
    ([(4, [100, 7, 30])], [3, 1, 30], 64, 80, 4),        # ... and 256-row tiles, pages of whole tiles
    ([(9, [90, 70])], [64, 33], 64, 32, 8),
    ([(12, [300, 70])], [290, 1], 16, 8, 4),             # pages of a wave's rows
    ([(12, [300, 70])], [290, 1], 20, 8, 4),             # pages found lane by lane
    ([(12, [30, 70, 1])], None, 20, 8, 4),               # ... and one new token each: chunks of their own
    ([(12, [30, 70, 1])], None, 20, 80, 4),
    ([(12, [30, 70])], None, 48, 8, 4),
]


@pytest.mark.parametrize("case", CAPPED, ids=[str(i) for i in range(len(CAPPED))])
def test_soft_cap_of_every_kernel(case, dev, monkeypatch):
    monkeypatch.setattr(PKG.shared_prefix, "shared_prefix_pays", lambda *a: True)
    groups, new, page, heads, kv = case
    gen = _gen(32)
    for zero_q in (True, False):
        _check(Batch(groups, page, kv, gen), heads, dev, gen, new=new, cap=5.0, zero_q=zero_q)


UNEVEN = [  # new tokens behind pages of any size, rows of a sequence on either side of a 256-row tile
    ([(12, [300, 70, 2])], [290, 1, 0], 20, 8, 4),
    ([(9, [40, 70])], [31, 32], 20, 32, 4),
    ([(7, [40, 70])], [32, 33], 24, 32, 4),
    ([(130, [5, 5, 9])], [1, 5, 2], 1, 8, 8),            # pages of one token
    ([(3, [100, 130])], [40, 130], 100, 6, 6),
]


@pytest.mark.parametrize("zero_q", [True, False])
@pytest.mark.parametrize("case", UNEVEN, ids=[str(i) for i in range(len(UNEVEN))])
def test_new_tokens_in_pages_of_any_size(case, zero_q, dev):
    groups, new, page, heads, kv = case
    gen = _gen(33)
    _check(Batch(groups, page, kv, gen), heads, dev, gen, new=new, zero_q=zero_q)


def test_routes_of_a_decode_step(dev, monkeypatch):
    """Narrow tables by the plain decode, wide ones by the shared kernels: the one that is taken, not its result alone."""
    gen = _gen(34)
    batch = Batch([(6, [50, 200, 3, None])], 64, 4, gen)
    q = torch.randn((4, 16, 128), generator=gen).to(torch.bfloat16)
    cache, table, lens, prefixes = batch.args(dev)
    wide = torch.full((4, 4000), -1, dtype=torch.int32, device=dev)
    wide[:, :table.shape[1]] = table
    want, tol = ref.shared(q, batch.cache, batch.table, batch.lengths, [1] * 4, 0.09)
    calls = []
    call = PKG._lib.call
    monkeypatch.setattr(PKG._lib, "call", lambda name, *a: calls.append(name) or call(name, *a))
    for t, name in ((table, "pa_decode"), (wide, "pa_shared_prefix")):
        got = PKG.shared_prefix_attention(q.to(dev), cache, t, lens, prefixes, scale=0.09)
        assert calls == [name] and ((got.cpu().double() - want).abs() <= tol).all()
        calls.clear()


@pytest.mark.parametrize("dim,heads,kv", [(64, 40, 2), (128, 40, 2), (64, 8, 8)])
def test_sparse_decode_with_a_soft_cap(dim, heads, kv, dev):
    gen = _gen(35)
    lengths, block, num = [999, 64, 0, 17], 32, 20
    table, nb = ref.tables(lengths, 64, gen)
    cache = ref.pool(nb, 64, kv, dim, gen)
    q = 3 * torch.randn((4, heads, dim), generator=gen).to(torch.bfloat16)
    sel = _random_selection(lengths, kv, num, block, gen)
    want, tol = ref.sparse_decode(q, cache, table, lengths, sel, block, dim ** -0.5, 20.0)
    got = PKG.block_sparse_decode_attention(q.to(dev), cache.to(dev), table.to(dev), _i32(lengths, dev), sel.to(dev),
                                            block=block, scale=dim ** -0.5, attn_logits_soft_cap=20.0)
    assert ((got.cpu().double() - want).abs() <= tol).all()


def test_routes_of_a_prefill_step(dev, monkeypatch):
    """attention() of a step with groups: few rows a sequence behind wide tables by the shared kernels, many by the plain
    prefill, with its bits."""
    gen = _gen(36)
    calls = []
    call = PKG._lib.call
    monkeypatch.setattr(PKG._lib, "call", lambda name, *a: calls.append(name) or call(name, *a))
    for new, name in (([3, 150, 16], "pa_shared_prefix"), ([199, 100, 86], "pa_prefill")):
        batch = Batch([(4, [250, 200, 130])], 64, 2, gen)
        cache, table, _, shared = batch.args(dev)
        wide = torch.full((3, 1400), -1, dtype=torch.int32, device=dev)
        wide[:, :table.shape[1]] = table
        n = sum(new)
        q = torch.randn((n, 32, 128), generator=gen).to(torch.bfloat16).to(dev)
        pos = [t for c, t0 in zip(new, batch.lengths) for t in range(t0 - c, t0)]
        cu = lambda x: _i32([0, *torch.tensor(x).cumsum(0).tolist()], dev)  # noqa: E731
        args = (_i32(pos, dev), _i32([-1] * n, dev), wide, cu(new), cu(batch.lengths), None, 0, max(new))
        plain = PKG.attention_stored(cache, q, PKG.PrefillAttentionMetadata(*args))
        calls.clear()
        got = PKG.attention_stored(cache, q, PKG.SharedPrefillAttentionMetadata(*args, shared=shared))
        assert calls == [name]
        assert torch.equal(got, plain) == (name == "pa_prefill")
        want, tol = ref.shared(q.cpu(), batch.cache, batch.table, batch.lengths, new, 0.08837890625,
                               scaled_q=name == "pa_prefill")
        assert ((got.cpu().double() - want).abs() <= tol).all()
