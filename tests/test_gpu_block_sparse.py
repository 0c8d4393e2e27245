"""Decode over selected blocks against plain 64-bit forms: the bounds of the blocks' keys, the scores, the selection, the
attention, and the layer seam that runs them together."""
from __future__ import annotations

import math

import pytest
import torch

import long_context_reference as ref
from conftest import PKG

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(x, dev=None):
    return torch.as_tensor(x, dtype=torch.int32, device=dev)


# ---------------------------------------------------------------------------
# bounds
# ---------------------------------------------------------------------------
BOUNDS = [  # lengths, new tokens (None: one each), page, block, kv heads, head size
    ([1, 16, 17, 33, 0, 64], None, 16, 16, 2, 128),
    ([1, 300, 256, 257, 40], [1, 300, 20, 2, 0], 256, 32, 8, 128),
    ([130, 64, 5], [130, 1, 3], 64, 16, 1, 64),
    ([500, 77], [123, 77], 32, 32, 3, 256),
    ([100, 99], [64, 50], 96, 48, 4, 128),
    ([700], [700], 256, 256, 5, 64),
]


@pytest.mark.parametrize("case", BOUNDS, ids=[str(i) for i in range(len(BOUNDS))])
def test_bounds(case, dev):
    lengths, new, page, block, kv, dim = case
    gen = _gen(1)
    table, nb = ref.tables(lengths, page, gen, extra=3)
    cache = ref.pool(nb, page, kv, dim, gen)
    before = torch.randn((nb, page // block, kv, 2, dim), generator=gen).to(torch.bfloat16)
    want = ref.bounds(cache, table, lengths, new or [1] * len(lengths), block, before)
    got = before.to(dev)
    cu = None if new is None else _i32([0, *torch.tensor(new).cumsum(0).tolist()], dev)
    out = PKG.update_block_bounds(got, cache.to(dev), table.to(dev), _i32(lengths, dev), cu,
                                  max_seqlen_q=max(new or [1]))
    assert out is got
    assert torch.equal(got.cpu(), want)


def test_bounds_of_more_new_tokens_than_said(dev):
    """max_seqlen_q sizes the launch alone: longer sequences are done all the same."""
    gen = _gen(2)
    table, nb = ref.tables([900, 40], 64, gen)
    cache = ref.pool(nb, 64, 2, 128, gen)
    before = torch.zeros((nb, 4, 2, 2, 128), dtype=torch.bfloat16)
    for most in (0, 1, 900, 1 << 30):
        got = PKG.update_block_bounds(before.to(dev), cache.to(dev), table.to(dev), _i32([900, 40], dev),
                                      _i32([0, 900, 940], dev), max_seqlen_q=most)
        assert torch.equal(got.cpu(), ref.bounds(cache, table, [900, 40], [900, 40], 16, before))


def test_bounds_leave_other_pages(dev):
    """Table entries outside the pool write nothing, rows behind the length (NaN here) take no part, and pools with
    strides of their own are addressed by them."""
    gen = _gen(3)
    cache = ref.pool(5, 32, 4, 64, gen)
    cache[:, 2, 10:] = float("nan")
    wide = torch.zeros((2, 5, 40, 6, 64), dtype=torch.bfloat16)
    wide[:, :, :32, 1:5] = cache
    view = wide.to(dev)[:, :, :32, 1:5]
    big = torch.zeros((5, 3, 7, 2, 64), dtype=torch.bfloat16).to(dev)
    bounds = big[:, :2, 2:6]
    table = _i32([[2, -1], [7, 1], [-3, 4]])
    PKG.update_block_bounds(bounds, view, table.to(dev), _i32([10, 40, 33], dev), _i32([0, 10, 50, 60], dev),
                            max_seqlen_q=40)
    want = torch.zeros((5, 2, 4, 2, 64), dtype=torch.bfloat16)
    want[2, 0, :, 0], want[2, 0, :, 1] = cache[0, 2, :10].amin(0), cache[0, 2, :10].amax(0)
    want[1, 0, :, 0], want[1, 0, :, 1] = cache[0, 1, :8].amin(0), cache[0, 1, :8].amax(0)
    want[4, 0, :, 0], want[4, 0, :, 1] = cache[0, 4, :1].amin(0), cache[0, 4, :1].amax(0)
    assert torch.equal(bounds.cpu(), want)
    rest = big.clone()
    rest[:, :2, 2:6] = 0
    assert not rest.any()


def test_bounds_follow_copied_pages(dev):
    gen = _gen(4)
    bounds = torch.randn((6, 4, 2, 2, 128), generator=gen).to(torch.bfloat16).to(dev)
    want = bounds.clone()
    want[[4, 5]] = want[[0, 2]]
    PKG.copy_block_bounds(bounds, [0, 2], [4, 5])
    assert torch.equal(bounds, want)


# ---------------------------------------------------------------------------
# scores
# ---------------------------------------------------------------------------
SCORES = [  # lengths, page, block, heads, kv heads, head size
    ([1, 0, 16, 17, 1000], 16, 16, 16, 8, 128),
    ([8000, 333], 256, 32, 32, 8, 128),
    ([500, 64], 64, 64, 40, 2, 64),    # 20 heads a kv head: two column blocks
    ([777], 128, 16, 3, 1, 256),
    ([95, 96, 97], 96, 48, 8, 8, 64),
]


@pytest.mark.parametrize("case", SCORES, ids=[str(i) for i in range(len(SCORES))])
def test_scores(case, dev):
    lengths, page, block, heads, kv, dim = case
    gen = _gen(5)
    table, nb = ref.tables(lengths, page, gen)
    x = torch.randn((nb, page // block, kv, 2, dim), generator=gen)
    bounds = torch.stack([x.amin(3), x.amax(3)], 3).to(torch.bfloat16)
    q = torch.randn((len(lengths), heads, dim), generator=gen).to(torch.bfloat16)
    want, tol = ref.scores(q, bounds, table, lengths, page, 0.1)
    got = PKG.block_scores(q.to(dev), bounds.to(dev), table.to(dev), _i32(lengths, dev), page_size=page,
                           scale=0.1).cpu().double()
    past = torch.isinf(want)
    assert torch.equal(torch.isinf(got), past) and (got[past] < 0).all()
    assert ((got - want).abs()[~past] <= tol[~past]).all()


def test_scores_bound_every_logit(dev):
    """No scaled logit of a block exceeds its score (but for the sums' roundings), over bounds from the pool."""
    gen = _gen(6)
    lengths, page, block = [301, 64], 64, 16
    table, nb = ref.tables(lengths, page, gen)
    cache = ref.pool(nb, page, 2, 128, gen)
    q = torch.randn((2, 8, 128), generator=gen).to(torch.bfloat16)
    cdev, tdev, ldev = cache.to(dev), table.to(dev), _i32(lengths, dev)
    bounds = PKG.new_block_bounds(cdev, block)
    PKG.update_block_bounds(bounds, cdev, tdev, ldev, _i32([0, 301, 365], dev), max_seqlen_q=301)
    got = PKG.block_scores(q.to(dev), bounds, tdev, ldev, page_size=page, scale=0.25).cpu().double()
    for b, n in enumerate(lengths):
        k = ref.rows(cache[0], table[b], 0, n)
        x = 0.25 * torch.einsum("hgd,htd->hgt", q[b].double().view(2, 4, 128), k).amax(1)
        for t in range(n):
            assert (x[:, t] <= got[b, :, t // block] + 1e-4).all()


def test_scores_strides_and_out(dev):
    gen = _gen(7)
    table, nb = ref.tables([200, 100], 64, gen)
    x = torch.randn((nb, 4, 2, 2, 128), generator=gen)
    bounds = torch.stack([x.amin(3), x.amax(3)], 3).to(torch.bfloat16)
    q = torch.randn((2, 9, 128), generator=gen).to(torch.bfloat16)
    wide = torch.full((2, 3, 20), 7.0, device=dev)
    out = wide[:, 1:, :16]
    got = PKG.block_scores(q.to(dev)[:, 1:], bounds.to(dev), table.to(dev), _i32([200, 100], dev), page_size=64,
                           scale=1.0, out=out)
    assert got is out
    want, tol = ref.scores(q[:, 1:], bounds, table, [200, 100], 64, 1.0)
    part = out.cpu().double()
    fine = ~torch.isinf(want)
    assert ((part - want).abs()[fine] <= tol[fine]).all() and torch.isinf(part[~fine]).all()
    wide[:, 1:, :16] = 7.0
    assert (wide == 7.0).all()


# ---------------------------------------------------------------------------
# selection
# ---------------------------------------------------------------------------
SELECT = [  # blocks of each sequence, width, num_selected, first, recent
    ([0, 1, 5, 8, 9, 40], 40, 8, 1, 2),
    ([1000, 1024, 700], 1030, 64, 1, 2),
    ([4097, 100, 2000], 4100, 33, 0, 0),
    ([16000, 3000], 16384, 128, 4, 4),
    ([20000, 40], 20001, 256, 1, 1),
    ([70, 90], 90, 6, 3, 3),          # nothing to choose
    ([300, 64], 300, 1, 0, 0),
    ([300, 300], 300, 299, 0, 1),
]


@pytest.mark.parametrize("ties", [False, True, "few"])
@pytest.mark.parametrize("case", SELECT, ids=[str(i) for i in range(len(SELECT))])
def test_select(case, ties, dev):
    blocks, width, num, first, recent = case
    gen = _gen(8)
    x = torch.randn((len(blocks), 2, width), generator=gen) * 5
    if ties:
        x = torch.round(x) if ties is True else torch.sign(x) * 0.0 + (x > 12)  # zeros of both signs, few ones
    lengths = [n * 32 - (7 if n else 0) for n in blocks]
    got = PKG.select_blocks(x.to(dev), _i32(lengths, dev), num, block=32, first=first, recent=recent)
    assert (got.cpu() == ref.select(x, lengths, num, 32, first, recent)).all()


def test_select_special_values(dev):
    """Infinities in order, NaN of either sign below all numbers, nothing read past a sequence's blocks."""
    x = torch.tensor([3.0, float("nan"), -math.inf, math.inf, 0.0, -0.0, -float("nan"), 1e38, -1e38, 1e-42, -1e-42,
                      math.inf, 2.0])
    for num in range(1, 13):
        full = torch.full((1, 1, 40), float("nan"))
        full[0, 0, :13] = x
        got = PKG.select_blocks(full.to(dev), _i32([13 * 16], dev), num, block=16, first=0, recent=0)
        assert torch.equal(got.cpu(), ref.select(full, [13 * 16], num, 16, 0, 0)), num


def test_select_strides(dev):
    gen = _gen(9)
    x = torch.randn((3, 6, 500), generator=gen).to(dev)
    out = torch.full((3, 4, 40), -9, dtype=torch.int32, device=dev)
    part = x[:, 1:4, 20:420]
    got = PKG.select_blocks(part, _i32([6400, 3200, 100], dev), 32, block=16, out=out[:, :3, 4:36])
    assert torch.equal(got.cpu(), ref.select(part.cpu(), [6400, 3200, 100], 32, 16, 1, 2))
    out[:, :3, 4:36] = -9
    assert (out == -9).all()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _random_selection(lengths, kv, num, block, gen):
    s = torch.full((len(lengths), kv, num), -1, dtype=torch.int32)
    for b, n in enumerate(lengths):
        blocks = -(-n // block)
        for j in range(kv):
            k = min(num, blocks)
            s[b, j, :k] = torch.sort(torch.randperm(blocks, generator=gen)[:k]).values.to(torch.int32)
    return s


SPARSE = [  # lengths, page, block, heads, kv heads, head size, entries, cap
    ([1, 15, 16, 17, 100], 16, 16, 16, 8, 128, 4, None),
    ([5000, 4097, 0, 33], 256, 32, 32, 8, 128, 64, None),
    ([3000, 50], 64, 64, 32, 8, 128, 20, 30.0),
    ([999, 400, 17], 64, 16, 40, 2, 64, 30, None),      # 20 heads a kv head
    ([2000, 300], 128, 128, 6, 2, 256, 9, None),
    ([700, 90], 32, 32, 5, 5, 256, 3, 20.0),
    ([4000], 256, 256, 8, 1, 64, 13, None),
    ([10000], 48, 48, 8, 2, 128, 150, None),
]


@pytest.mark.parametrize("case", SPARSE, ids=[str(i) for i in range(len(SPARSE))])
def test_sparse_decode(case, dev):
    lengths, page, block, heads, kv, dim, num, cap = case
    gen = _gen(10)
    table, nb = ref.tables(lengths, page, gen)
    cache = ref.pool(nb, page, kv, dim, gen)
    q = torch.randn((len(lengths), heads, dim), generator=gen).to(torch.bfloat16) * 3
    sel = _random_selection(lengths, kv, num, block, gen)
    want, tol = ref.sparse_decode(q, cache, table, lengths, sel, block, dim ** -0.5, cap)
    got = PKG.block_sparse_decode_attention(q.to(dev), cache.to(dev), table.to(dev), _i32(lengths, dev), sel.to(dev),
                                            block=block, scale=dim ** -0.5, attn_logits_soft_cap=cap)
    over = (got.cpu().double() - want).abs() - tol
    assert (over <= 0).all(), over.max()


def test_sparse_decode_any_list(dev):
    """Holes, other sequences' block numbers, an order that falls, a block twice; rows without a block are zero."""
    gen = _gen(11)
    lengths = [500, 320, 64, 0, 128]
    table, nb = ref.tables(lengths, 64, gen)
    cache = ref.pool(nb, 64, 2, 128, gen)
    q = torch.randn((5, 8, 128), generator=gen).to(torch.bfloat16)
    sel = torch.full((5, 2, 70), -1, dtype=torch.int32)
    sel[0, 0, [3, 17, 40, 69]] = _i32([15, 2, 0, 15])
    sel[0, 1, :6] = _i32([16, 31, 1 << 30, -5, 7, 6])
    sel[1, 0] = _i32(list(range(9, -1, -1)) * 7)
    sel[2, 1, 5] = 1
    sel[4, :, ::2] = 3
    want, tol = ref.sparse_decode(q, cache, table, lengths, sel, 32, 0.1)
    assert (want[2, :4] == 0).all() and (want[3] == 0).all()
    got = PKG.block_sparse_decode_attention(q.to(dev), cache.to(dev), table.to(dev), _i32(lengths, dev), sel.to(dev),
                                            block=32, scale=0.1)
    assert ((got.cpu().double() - want).abs() <= tol).all()


def test_sparse_decode_reads_nothing_else(dev):
    """NaN and infinities in blocks that are not selected and behind the length stay out; strides of q, pool, selection
    and output; lengths past the table's span are clamped to it."""
    gen = _gen(12)
    lengths = [100, 1 << 20]
    table, nb = ref.tables([100, 128], 64, gen, extra=2)
    cache = ref.pool(nb, 64, 2, 128, gen)
    sel = _i32([[[0, 3], [1, 3]], [[2, 7], [0, 5]]])
    want, tol = ref.sparse_decode(torch.ones((2, 4, 128)).to(torch.bfloat16), cache, table, lengths, sel, 16, 0.05)
    bad = torch.full(cache.shape, float("nan"), dtype=torch.bfloat16)
    bad[1] = float("inf")
    for b, n in enumerate((100, 128)):
        for j in range(2):
            for c in sel[b, j].tolist():
                for t in range(c * 16, min(n, c * 16 + 16)):
                    p, s = int(table[b, t // 64]), t % 64
                    bad[:, p, s, j] = cache[:, p, s, j]
    wide = torch.full((2, nb, 64, 3, 128), float("nan"), dtype=torch.bfloat16)
    wide[:, :, :, 1:] = bad
    q = torch.full((2, 6, 128), float("nan"), dtype=torch.bfloat16)
    q[:, 2:] = 1
    out = torch.full((2, 5, 128), 9.0, dtype=torch.bfloat16, device=dev)
    sel_wide = torch.full((2, 2, 4), 1, dtype=torch.int32)
    sel_wide[:, :, 1:3] = sel
    PKG.block_sparse_decode_attention(q.to(dev)[:, 2:], wide.to(dev)[:, :, :, 1:], table.to(dev), _i32(lengths, dev),
                                      sel_wide.to(dev)[:, :, 1:3], block=16, scale=0.05, out=out[:, 1:])
    assert ((out[:, 1:].cpu().double() - want).abs() <= tol).all()
    assert (out[:, 0] == 9).all()


def test_sparse_decode_all_blocks_is_decode(dev):
    """With every block selected the result is the dense decode's, up to both kernels' roundings."""
    gen = _gen(13)
    lengths = [1500, 700, 31]
    table, nb = ref.tables(lengths, 64, gen)
    cache = ref.pool(nb, 64, 4, 128, gen).to(dev)
    q = torch.randn((3, 16, 128), generator=gen).to(torch.bfloat16).to(dev)
    lens = _i32(lengths, dev)
    sel = PKG.select_blocks(torch.zeros((3, 4, 96), device=dev), lens, 96, block=16)
    got = PKG.block_sparse_decode_attention(q, cache, table.to(dev), lens, sel, block=16, scale=0.09)
    pages = (cache[0].permute(2, 0, 1, 3), cache[1].permute(2, 0, 1, 3))
    dense = PKG.decode_paged_attention(q, *pages, table.to(dev), lens, scale=0.09)
    _, tol = ref.sparse_decode(q.cpu(), cache.cpu(), table, lengths, sel.cpu(), 16, 0.09)
    assert ((got.double() - dense.double()).abs().cpu() <= 2 * tol).all()


def test_workspace_and_repeats(dev):
    """A given workspace gives the same bits as one made in the call, call after call; one that is too small is not
    used."""
    gen = _gen(14)
    table, nb = ref.tables([9000, 5000], 64, gen)
    cache = ref.pool(nb, 64, 2, 128, gen).to(dev)
    q = torch.randn((2, 8, 128), generator=gen).to(torch.bfloat16).to(dev)
    sel = _random_selection([9000, 5000], 2, 100, 32, gen).to(dev)
    args = (q, cache, table.to(dev), _i32([9000, 5000], dev), sel)
    need = PKG.block_sparse_workspace_bytes(2, 8, 2, 128, 100, 32)
    assert need > 0
    first = PKG.block_sparse_decode_attention(*args, block=32, scale=0.1)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=dev)
    for w in (ws, ws[:16], None):
        assert torch.equal(PKG.block_sparse_decode_attention(*args, block=32, scale=0.1, workspace=w), first)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def _expected_decode(q, cache, bounds, table, lengths, num, block, first, recent, scale, chosen):
    """The attention over ``chosen``, after checking that it is a selection by the exact scores up to their error."""
    exact, tol = ref.scores(q, bounds, table, lengths, cache.shape[2], scale)
    for b, n in enumerate(lengths):
        blocks = -(-n // block)
        for j in range(cache.shape[3]):
            mine = [c for c in chosen[b, j].tolist() if c >= 0]
            assert mine == sorted(set(mine)) and len(mine) == min(blocks, num)
            assert set(range(min(first, blocks))) <= set(mine)
            assert set(range(max(0, blocks - recent), blocks)) <= set(mine)
            rest = [c for c in range(blocks) if c not in mine]
            if rest:
                x, e = exact[b, j], tol[b, j]
                free = [c for c in mine if first <= c < blocks - recent]
                assert min(float(x[c] + e[c]) for c in free) >= max(float(x[c] - e[c]) for c in rest)
    return ref.sparse_decode(q, cache, table, lengths, chosen, block, scale)


def test_a_conversation(dev):
    """Prompts, then decode steps, through the layer seam: the pool, the bounds and each step's output."""
    gen = _gen(15)
    page, block, kv, heads, dim, num = 64, 16, 2, 8, 128, 12
    lengths = [333, 700, 20]
    final = [n + 3 for n in lengths]
    table, nb = ref.tables(final, page, gen)
    cache = torch.zeros((2, nb, page, kv, dim), dtype=torch.bfloat16, device=dev)
    bounds = PKG.new_block_bounds(cache, block)
    model = torch.zeros((2, nb, page, kv, dim), dtype=torch.bfloat16)
    mbounds = torch.zeros((nb, page // block, kv, 2, dim), dtype=torch.bfloat16)
    tdev = table.to(dev)

    def step(new, totals):
        n = sum(new)
        k, v = (torch.randn((n, kv, dim), generator=gen).to(torch.bfloat16) for _ in range(2))
        q = torch.randn((n, heads, dim), generator=gen).to(torch.bfloat16)
        slots, pos = [], []
        for b, (c, t) in enumerate(zip(new, totals)):
            for p in range(t - c, t):
                slots.append(int(table[b, p // page]) * page + p % page)
                pos.append(p)
        model[0].view(-1, kv, dim)[slots] = k
        model[1].view(-1, kv, dim)[slots] = v
        mbounds.copy_(ref.bounds(model, table, totals, new, block, mbounds))
        return q, k.to(dev), v.to(dev), _i32(slots, dev), _i32(pos, dev)

    q, k, v, slots, pos = step(lengths, lengths)
    cu = _i32([0, *torch.tensor(lengths).cumsum(0).tolist()], dev)
    meta = PKG.PrefillAttentionMetadata(pos, slots, tdev, cu, cu, None, None, max(lengths))
    _, out = PKG.block_sparse_attention(cache, bounds, q.to(dev), k, v, meta, num_selected=num)
    assert torch.equal(out, PKG.attention_stored(cache, q.to(dev), meta))
    assert torch.equal(cache.cpu(), model) and torch.equal(bounds.cpu(), mbounds)
    scale = 1 / float(torch.tensor(dim ** 0.5).to(torch.bfloat16))
    for i in range(1, 4):
        now = [n + i for n in lengths]
        q, k, v, slots, pos = step([1] * 3, now)
        lens = _i32(now, dev)
        if i == 2:  # as part of a mixed step without prefill sequences
            meta = PKG.MixedAttentionMetadata(pos, slots, tdev, _i32([0, 1, 2, 3], dev), lens, 3, 0)
        else:
            meta = PKG.DecodeAttentionMetadata(pos, slots, tdev, lens)
        _, out = PKG.block_sparse_attention(cache, bounds, q.to(dev), k, v, meta, num_selected=num)
        assert torch.equal(cache.cpu(), model) and torch.equal(bounds.cpu(), mbounds)
        chosen = PKG.select_blocks(PKG.block_scores(q.to(dev), bounds, tdev, lens, page_size=page, scale=scale), lens,
                                   num, block=block)
        want, tol = _expected_decode(q, model, mbounds, table, now, num, block, 1, 2, scale, chosen.cpu())
        assert ((out.cpu().double() - want).abs() <= tol).all()


def test_mixed_step(dev):
    """Decode sequences sparse, prefill sequences whole, in one step."""
    gen = _gen(16)
    page, block, kv, heads, dim, num = 32, 16, 2, 8, 64, 5
    lengths, new = [400, 150, 90], [1, 1, 33]
    table, nb = ref.tables(lengths, page, gen)
    model = ref.pool(nb, page, kv, dim, gen)
    cache, tdev, lens = model.to(dev), table.to(dev), _i32(lengths, dev)
    bounds = PKG.new_block_bounds(cache, block)
    PKG.update_block_bounds(bounds, cache, tdev, lens, _i32([0, 400, 550, 640], dev), max_seqlen_q=400)
    q = torch.randn((35, heads, dim), generator=gen).to(torch.bfloat16).to(dev)
    pos = [t for n, c in zip(lengths, new) for t in range(n - c, n)]
    slots = [int(table[b, t // page]) * page + t % page for b, (n, c) in enumerate(zip(lengths, new))
             for t in range(n - c, n)]
    k, v = (model[i].reshape(-1, kv, dim)[slots].to(dev) for i in (0, 1))
    meta = PKG.MixedAttentionMetadata(_i32(pos, dev), _i32(slots, dev), tdev, _i32([0, 1, 2, 35], dev), lens, 2, 33)
    _, out = PKG.block_sparse_attention(cache, bounds, q, k, v, meta, num_selected=num)
    assert torch.equal(cache.cpu(), model)
    dense = PKG.attention_stored(cache, q, meta)
    assert torch.equal(out[2:], dense[2:])
    scale = 1 / float(torch.tensor(dim ** 0.5).to(torch.bfloat16))
    chosen = PKG.select_blocks(PKG.block_scores(q[:2], bounds, tdev[:2], lens[:2], page_size=page, scale=scale),
                               lens[:2], num, block=block)
    want, tol = _expected_decode(q[:2].cpu(), model, bounds.cpu(), table[:2], lengths[:2], num, block, 1, 2, scale,
                                 chosen.cpu())
    assert ((out[:2].cpu().double() - want).abs() <= tol).all()


def test_captured_step(dev):
    """A decode step in a graph, replayed with new q, lengths and tables between eager steps on another stream."""
    gen = _gen(17)
    page, block, num = 64, 32, 20
    table, nb = ref.tables([4000, 3000, 1500], page, gen)
    cache = ref.pool(nb, page, 4, 128, gen).to(dev)
    tdev, lens = table.to(dev), _i32([4000, 3000, 1500], dev)
    bounds = PKG.new_block_bounds(cache, block)
    PKG.update_block_bounds(bounds, cache, tdev, lens, _i32([0, 4000, 7000, 8500], dev), max_seqlen_q=4000)
    q = torch.randn((3, 16, 128), generator=gen).to(torch.bfloat16).to(dev)

    def step():
        PKG.update_block_bounds(bounds, cache, tdev, lens)
        chosen = PKG.select_blocks(PKG.block_scores(q, bounds, tdev, lens, page_size=page, scale=0.1), lens, num,
                                   block=block)
        return PKG.block_sparse_decode_attention(q, cache, tdev, lens, chosen, block=block, scale=0.1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for r in range(4):
        q.copy_(torch.randn((3, 16, 128), generator=gen).to(torch.bfloat16))
        lens.copy_(_i32([4000 - 700 * r, 100 * r, 1500 - r]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        with torch.cuda.stream(side):
            eager = step()
        torch.cuda.synchronize()
        assert torch.equal(replayed, eager)
