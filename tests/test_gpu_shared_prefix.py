"""Attention of sequences that share prefixes against a plain 64-bit form of each sequence alone."""
from __future__ import annotations

import pytest
import torch

import long_context_reference as ref
from conftest import PKG

pytestmark = pytest.mark.gpu
DECODE_SCALE = 1 / 11.3125       # what attention() applies: 1 / bf16(128 ** 0.5)
PREFILL_SCALE = 0.08837890625    # bf16(128 ** -0.5)


@pytest.fixture(autouse=True)
def _share(monkeypatch):
    """The small steps here go through the kernels of shared prefixes, not through the plain decode."""
    monkeypatch.setattr(PKG.shared_prefix, "shared_prefix_pays", lambda *a: True)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(x, dev=None):
    return torch.as_tensor(x, dtype=torch.int32, device=dev)


class Batch:
    """Groups of sequences: ``groups`` = [(shared pages, [own tokens of each sequence])]."""

    def __init__(self, groups, page, kv, gen, dim=128, extra=1):
        lengths, shared, cu, lens = [], [], [0], []
        for pages, owns in groups:
            for i, n in enumerate(owns):
                empty = n is None                                    # a padding sequence
                lengths.append(0 if empty else pages * page + n)
                shared.append((cu[-1], pages) if i and pages and not empty else None)
            cu.append(cu[-1] + len(owns))
            lens.append(pages * page)
        self.table, nb = ref.tables(lengths, page, gen, shared=shared, extra=extra)
        self.lengths, self.page, self.kv = lengths, page, kv
        self.cu, self.lens = cu, lens
        self.cache = ref.pool(nb, page, kv, dim, gen)

    def prefixes(self, dev):
        return PKG.SharedPrefixes.of(self.cu, self.lens, dev)

    def args(self, dev):
        return self.cache.to(dev), self.table.to(dev), _i32(self.lengths, dev), self.prefixes(dev)


def _check(batch, heads, dev, gen, *, new=None, cap=None, zero_q=False, strict=True):
    n = sum(new) if new else len(batch.lengths)
    q = torch.randn((n, heads, 128), generator=gen).to(torch.bfloat16)
    if zero_q:
        q.zero_()
    want, tol = ref.shared(q, batch.cache, batch.table, batch.lengths, new or [1] * n, 0.09, cap)
    cu = None if new is None else _i32([0, *torch.tensor(new).cumsum(0).tolist()], dev)
    got = PKG.shared_prefix_attention(q.to(dev), *batch.args(dev), cu, max_seqlen_q=max(new or [1]), scale=0.09,
                                      attn_logits_soft_cap=cap)
    over = (got.cpu().double() - want).abs() - tol
    assert (over <= 0).all(), (over.max(), (over > 0).nonzero()[:4])
    return got


DECODE = [  # groups, page, heads, kv heads
    ([(1, [1, 5, 300])], 256, 32, 8),
    ([(9, [20, 0, 700, 64, 65]), (0, [100, 3]), (40, [1, 900])], 64, 16, 8),
    ([(2, [7]), (3, [5, 6])], 128, 8, 1),                       # a group of one
    ([(130, [40] * 30)], 16, 64, 8),                            # 240 rows of 256
    ([(70, [i for i in range(1, 71)])], 32, 32, 8),             # 280 rows: two q tiles
    ([(21, [100, 50, 7])], 48, 12, 4),                          # pages that are not of the tile's tokens
    ([(60, [9, 3, 300])], 20, 4, 4),                            # nor of 16
    ([(5, [33, 17])], 256, 40, 2),                              # 20 heads a kv head
    ([(1, [3, 4])], 48, 4, 2),                                  # less than a tile shared
    ([(24, [2000, 5000, 1])], 64, 6, 2),                        # long own parts
    ([(8, [None, 30, None, 90, None])], 64, 16, 8),             # padding sequences
]


@pytest.mark.parametrize("zero_q", [True, False])
@pytest.mark.parametrize("case", DECODE, ids=[str(i) for i in range(len(DECODE))])
def test_decode(case, zero_q, dev):
    """q of zeros weighs all tokens alike, exactly: a token too many or too few shows."""
    groups, page, heads, kv = case
    gen = _gen(1)
    _check(Batch(groups, page, kv, gen), heads, dev, gen, zero_q=zero_q)


SEVERAL = [  # groups (own tokens, the new included), new tokens, page, heads, kv heads
    ([(9, [20, 5, 700])], [5, 5, 5], 64, 32, 8),
    ([(3, [64, 65, 100]), (0, [100, 31])], [64, 1, 100, 33, 31], 256, 16, 8),
    ([(40, [3, 300, 8, 8])], [3, 300, 0, 8], 16, 8, 1),             # a sequence without new tokens
    ([(5, [17] * 20)], [17] * 20, 64, 64, 8),                       # several q tiles
    ([(11, [70, 2])], [70, 2], 48, 12, 4),
    ([(2, [10, 30])], [200, 40], 64, 8, 4),                         # new tokens reach into the shared ones
    ([(8, [None, 30, 90])], [0, 30, 4], 64, 16, 8),
    ([(30, [1, 1, 1])], [1, 1, 1], 64, 40, 2),
    ([(7, [400, 2500])], [300, 2], 64, 10, 2),                      # 5 heads a kv head: tiles of 255 rows
]


@pytest.mark.parametrize("zero_q", [True, False])
@pytest.mark.parametrize("case", SEVERAL, ids=[str(i) for i in range(len(SEVERAL))])
def test_several_new_tokens(case, zero_q, dev):
    groups, new, page, heads, kv = case
    gen = _gen(2)
    _check(Batch(groups, page, kv, gen), heads, dev, gen, new=new, zero_q=zero_q)


@pytest.mark.parametrize("new", [None, [3, 1, 2]])
def test_soft_cap(new, dev):
    gen = _gen(3)
    _check(Batch([(4, [100, 7, 30])], 64, 4, gen), 16, dev, gen, new=new, cap=5.0)


def test_long_prefix(dev):
    gen = _gen(4)
    _check(Batch([(300, [5, 90, 700, 1])], 64, 2, gen), 8, dev, gen, zero_q=True)
    _check(Batch([(300, [5, 90, 700, 1])], 64, 2, gen), 8, dev, gen, new=[5, 20, 3, 1], zero_q=True)


@pytest.mark.parametrize("new", [None, 2])
def test_more_sequences_than_the_plan_keeps_in_lds(new, dev):
    gen = _gen(13)
    batch = Batch([(4, [1 + (g + i) % 30 for i in range(3)]) for g in range(700)], 16, 1, gen)
    _check(batch, 2, dev, gen, new=new and [min(new, n - 64) for n in batch.lengths], zero_q=True)


def test_more_chunks_than_workgroups(dev):
    """Long own parts of 256 q heads a kv head: a workgroup takes several chunks."""
    gen = _gen(14)
    _check(Batch([(0, [20000]), (4, [9000, 100])], 16, 2, gen), 512, dev, gen, zero_q=True)


def test_scales_of_any_sign(dev):
    gen = _gen(15)
    for new in (None, [3, 1, 2], [70, 1, 100]):
        batch = Batch([(4, [100, 7 if new is None else 107, 300])], 64, 2, gen)
        n = sum(new) if new else 3
        q = torch.randn((n, 8, 128), generator=gen).to(torch.bfloat16)
        cu = None if new is None else _i32([0, *torch.tensor(new).cumsum(0).tolist()], dev)
        for scale in (-0.09, 0.0):
            want, _ = ref.shared(q, batch.cache, batch.table, batch.lengths, new or [1] * 3, scale)
            flipped, tol = ref.shared(-q if scale < 0 else q, batch.cache, batch.table, batch.lengths, new or [1] * 3,
                                      abs(scale))
            assert torch.allclose(flipped, want)
            got = PKG.shared_prefix_attention(q.to(dev), *batch.args(dev), cu, max_seqlen_q=max(new or [1]), scale=scale)
            assert ((got.cpu().double() - want).abs() <= tol).all(), (new, scale)


def test_matches_the_entries_it_stands_beside(dev):
    """Decode and prefill of the same sequences without sharing, up to both kernels' roundings."""
    gen = _gen(5)
    batch = Batch([(6, [50, 200, 3]), (2, [9, 40])], 64, 4, gen)
    q = torch.randn((5, 16, 128), generator=gen).to(torch.bfloat16)
    _, tol = ref.shared(q, batch.cache, batch.table, batch.lengths, [1] * 5, 0.09)
    cache, table, lens, prefixes = batch.args(dev)
    got = PKG.shared_prefix_attention(q.to(dev), cache, table, lens, prefixes, scale=0.09)
    pages = (cache[0].permute(2, 0, 1, 3), cache[1].permute(2, 0, 1, 3))
    dense = PKG.decode_paged_attention(q.to(dev), *pages, table, lens, scale=0.09)
    assert ((got.double() - dense.double()).abs().cpu() <= 2 * tol).all()
    # sharing nothing is the same call
    none = PKG.SharedPrefixes.of([0], [], dev)
    assert ((PKG.shared_prefix_attention(q.to(dev), cache, table, lens, none, scale=0.09).double()
             - dense.double()).abs().cpu() <= 2 * tol).all()


def test_plain_decode_where_sharing_does_not_pay(dev, monkeypatch):
    """The route of small steps: the plain decode's bits, out and soft cap included."""
    monkeypatch.undo()
    gen = _gen(11)
    batch = Batch([(6, [50, 200, 3, None])], 64, 4, gen)
    q = torch.randn((4, 16, 128), generator=gen).to(torch.bfloat16).to(dev)
    assert not PKG.shared_prefix_pays(4, 1, 4, batch.table.shape[1] * 64)
    cache, table, lens, prefixes = batch.args(dev)
    pages = (cache[0].permute(2, 0, 1, 3), cache[1].permute(2, 0, 1, 3))
    out = torch.empty((4, 18, 128), dtype=torch.bfloat16, device=dev)
    for cap in (None, 9.0):
        dense = PKG.decode_paged_attention(q, *pages, table, lens, scale=0.09, attn_logits_soft_cap=cap)
        got = PKG.shared_prefix_attention(q, cache, table, lens, prefixes, scale=0.09, attn_logits_soft_cap=cap)
        assert torch.equal(got, dense)
        PKG.shared_prefix_attention(q, cache, table, lens, prefixes, scale=0.09, attn_logits_soft_cap=cap,
                                    out=out[:, 1:17])
        assert torch.equal(out[:, 1:17], dense)
    # and where it pays, by the tables' width, the shared kernels'
    wide = torch.full((4, 4000), -1, dtype=torch.int32, device=dev)
    wide[:, :table.shape[1]] = table
    assert PKG.shared_prefix_pays(4, 1, 4, 4000 * 64) and not PKG.shared_prefix_pays(4, 4, 4, 4000 * 64)
    got = PKG.shared_prefix_attention(q, cache, wide, lens, prefixes, scale=0.09)
    monkeypatch.setattr(PKG.shared_prefix, "shared_prefix_pays", lambda *a: True)
    want, tol = ref.shared(q.cpu(), batch.cache, batch.table, batch.lengths, [1] * 4, 0.09)
    assert ((got.cpu().double() - want).abs() <= tol).all()


def test_attention_takes_the_groups(dev):
    """The layer seam: metadata with ``shared`` stores and attends like metadata without."""
    gen = _gen(6)
    batch = Batch([(4, [50, 200, 3])], 64, 8, gen)
    new = [4, 1, 3]
    q = torch.randn((8, 32, 128), generator=gen).to(torch.bfloat16).to(dev)
    k, v = (torch.randn((8, 8, 128), generator=gen).to(torch.bfloat16).to(dev) for _ in range(2))
    pos = [t for n, t0 in zip(new, batch.lengths) for t in range(t0 - n, t0)]
    seq = [b for b, n in enumerate(new) for _ in range(n)]
    slots = _i32([int(batch.table[b, t // 64]) * 64 + t % 64 for b, t in zip(seq, pos)], dev)
    cu_q = _i32([0, 4, 5, 8], dev)
    cu_k = _i32([0, *torch.tensor(batch.lengths).cumsum(0).tolist()], dev)
    outs = []
    for shared in (None, batch.prefixes(dev)):
        cache, table, _, _ = batch.args(dev)
        meta = PKG.SharedPrefillAttentionMetadata(_i32(pos, dev), slots, table, cu_q, cu_k, None, None, 4, shared=shared)
        pool, out = PKG.attention(cache, q, k, v, meta)
        outs.append((pool.cpu(), out.cpu().double()))
    assert torch.equal(outs[0][0], outs[1][0])
    # (the plain prefill rounds its scaled q)
    _, tol = ref.shared(q.cpu(), outs[0][0], batch.table, batch.lengths, new, PREFILL_SCALE, scaled_q=True)
    assert ((outs[0][1] - outs[1][1]).abs() <= 2 * tol).all()
    first = [0, 4, 5]
    outs = []
    for shared in (None, batch.prefixes(dev)):
        cache, table, lens, _ = batch.args(dev)
        meta = PKG.SharedDecodeAttentionMetadata(_i32(pos, dev)[first], slots[first], table, lens, shared=shared)
        pool, out = PKG.attention(cache, q[first], k[first], v[first], meta)
        outs.append((pool.cpu(), out.cpu().double()))
    assert torch.equal(outs[0][0], outs[1][0])
    _, tol = ref.shared(q[first].cpu(), outs[0][0], batch.table, batch.lengths, [1] * 3, DECODE_SCALE)
    assert ((outs[0][1] - outs[1][1]).abs() <= 2 * tol).all()


def test_rows_outside_and_strides(dev):
    """Rows behind the last sequence and past max_seqlen_q: zero in a new output, left in a given one; q, pool, tables
    and out with strides of their own; garbage behind the lengths and in other pages."""
    gen = _gen(7)
    batch = Batch([(3, [40, 9])], 64, 2, gen, extra=3)
    new = [3, 2]
    q = torch.randn((9, 8, 128), generator=gen).to(torch.bfloat16)
    want, tol = ref.shared(q[:5], batch.cache, batch.table, batch.lengths, new, 0.09)
    used = torch.zeros(batch.cache.shape[1:3], dtype=torch.bool)
    for b, n in enumerate(batch.lengths):
        for t in range(n):
            used[int(batch.table[b, t // 64]), t % 64] = True
    bad = batch.cache.clone()
    bad[:, ~used] = float("nan")
    wide = torch.full((2, bad.shape[1], 64, 5, 128), float("nan"), dtype=torch.bfloat16)
    wide[:, :, :, 1:3] = bad
    qw = torch.zeros((9, 11, 128), dtype=torch.bfloat16)
    qw[:, 2:10] = q
    tw = torch.full((2, batch.table.shape[1] + 3), 1 << 20, dtype=torch.int32)
    tw[:, :-3] = batch.table
    args = (qw.to(dev)[:, 2:10], wide.to(dev)[:, :, :, 1:3], tw.to(dev)[:, :-3], _i32(batch.lengths, dev),
            batch.prefixes(dev), _i32([0, 3, 5], dev))
    got = PKG.shared_prefix_attention(*args, max_seqlen_q=3, scale=0.09).cpu().double()
    assert ((got[:5] - want).abs() <= tol).all() and (got[5:] == 0).all()
    out = torch.full((9, 9, 128), 5.0, dtype=torch.bfloat16, device=dev)
    PKG.shared_prefix_attention(*args, max_seqlen_q=2, scale=0.09, out=out[:, :8])
    given = out.cpu().double()
    rows = [0, 1, 3, 4]
    assert ((given[rows, :8] - want[rows]).abs() <= tol[rows]).all()
    assert (given[[2, 5, 6, 7, 8]] == 5).all() and (given[:, 8] == 5).all()


def test_wrong_promises_stay_in_bounds(dev):
    """Shared lengths past the shortest sequence, negative or huge ones are cut; groups that fall, or reach past the
    batch, do not fault."""
    gen = _gen(8)
    batch = Batch([(3, [40, 9, 1])], 64, 2, gen)
    q = torch.randn((3, 8, 128), generator=gen).to(torch.bfloat16)
    cache, table, lens, _ = batch.args(dev)
    want, tol = ref.shared(q, batch.cache, batch.table, batch.lengths, [1] * 3, 0.09)
    for cu, shared in (([0, 3], [3 * 64 + 63]), ([0, 3], [-64]), ([0, 2, 3], [192, 1 << 30]), ([0, 1, 3], [192, 192])):
        got = PKG.shared_prefix_attention(q.to(dev), cache, table, lens, PKG.SharedPrefixes.of(cu, shared, dev),
                                          scale=0.09).cpu().double()
        assert ((got - want).abs() <= tol).all(), (cu, shared)
    for cu, shared in (([0, 9], [192]), ([2, 0, 3], [192, 192]), ([-5, 3], [192])):
        out = PKG.shared_prefix_attention(q.to(dev), cache, table, lens, PKG.SharedPrefixes.of(cu, shared, dev),
                                          scale=0.09)
        torch.cuda.synchronize()
        assert out.shape == q.shape


def test_workspace_and_repeats(dev):
    gen = _gen(9)
    batch = Batch([(30, [400, 9, 1, 77])], 64, 2, gen)
    q = torch.randn((4, 8, 128), generator=gen).to(torch.bfloat16).to(dev)
    args = (q, *batch.args(dev))
    need = PKG.shared_prefix_workspace_bytes(4, 1, 4, 8, 2, batch.table.shape[1], 64)
    first = PKG.shared_prefix_attention(*args, scale=0.1)
    for fill in (0, 255):
        ws = torch.full((need,), fill, dtype=torch.uint8, device=dev)
        for w in (ws, ws[:256], None):
            assert torch.equal(PKG.shared_prefix_attention(*args, scale=0.1, workspace=w), first)


@pytest.mark.parametrize("several", [False, True])
def test_captured(several, dev):
    """A step in a graph, replayed with other q, lengths and groups between eager calls on another stream."""
    gen = _gen(10)
    batch = Batch([(30, [400, 90, 130, 77])], 64, 4, gen)
    n = 8 if several else 4
    q = torch.randn((n, 16, 128), generator=gen).to(torch.bfloat16).to(dev)
    cache, table, lens, prefixes = batch.args(dev)
    prefixes = PKG.SharedPrefixes.of([0, 2, 4], [1920, 1920], dev)
    cu = _i32([0, 2, 4, 6, 8], dev) if several else None

    def step():
        return PKG.shared_prefix_attention(q, cache, table, lens, prefixes, cu, max_seqlen_q=2, scale=0.1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for r in range(4):
        q.copy_(torch.randn((n, 16, 128), generator=gen).to(torch.bfloat16))
        lens.copy_(_i32([2320 - 31 * r, 1990 + r, 0 if r == 2 else 2050, 1930]))
        prefixes.cu_groups.copy_(_i32([[0, 2, 4], [0, 4, 4], [0, 0, 4], [0, 1, 4]][r]))
        prefixes.shared_lens.copy_(_i32([1920 - 64 * r, 1000]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        with torch.cuda.stream(side):
            eager = step()
        torch.cuda.synchronize()
        assert torch.equal(replayed, eager)
        want, tol = ref.shared(q.cpu(), batch.cache, batch.table, lens.cpu(), [2] * 4 if several else [1] * 4, 0.1)
        assert ((out.cpu().double() - want).abs() <= tol).all()


def test_a_step_of_the_block_manager(dev):
    """Prompts behind a cached system prompt, then decode steps, with the groups that the manager finds: each step's
    output against the plain form."""
    from test_long_context_api import Request
    gen = _gen(12)
    mgr = PKG.KVCacheManager(64, 64, enable_prefix_caching=True)
    cache = torch.zeros((2, 64, 64, 2, 128), dtype=torch.bfloat16, device=dev)
    model = torch.zeros((2, 64, 64, 2, 128), dtype=torch.bfloat16)
    system = list(range(300))
    first = Request(0, system + [900] * 30)
    rest = [Request(i, system + [1000 + i] * (20 + 9 * i)) for i in range(1, 5)]

    def step(batch, new, decode):
        lens = [len(r) for r in batch]
        tables = [mgr.block_ids(r) for r in batch]
        table = torch.full((len(batch), max(map(len, tables))), -1, dtype=torch.int32)
        for i, t in enumerate(tables):
            table[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
        pos = [t for n, c in zip(lens, new) for t in range(n - c, n)]
        seq = [i for i, c in enumerate(new) for _ in range(c)]
        slots = [int(table[i, t // 64]) * 64 + t % 64 for i, t in zip(seq, pos)]
        q = torch.randn((len(pos), 8, 128), generator=gen).to(torch.bfloat16)
        k, v = (torch.randn((len(pos), 2, 128), generator=gen).to(torch.bfloat16) for _ in range(2))
        model[0].view(-1, 2, 128)[slots], model[1].view(-1, 2, 128)[slots] = k, v
        groups = mgr.shared_prefixes(batch)
        shared = PKG.SharedPrefixes.of(*groups, dev)
        common = (_i32(pos, dev), _i32(slots, dev), table.to(dev))
        if decode:
            meta = PKG.SharedDecodeAttentionMetadata(*common, _i32(lens, dev), shared=shared)
        else:
            cu = lambda x: _i32([0, *torch.tensor(x).cumsum(0).tolist()], dev)  # noqa: E731
            meta = PKG.SharedPrefillAttentionMetadata(*common, cu(new), cu(lens), None, None, max(new), shared=shared)
        _, out = PKG.attention(cache, q.to(dev), k.to(dev), v.to(dev), meta)
        want, tol = ref.shared(q, model, table, lens, new, DECODE_SCALE if decode else PREFILL_SCALE)
        assert torch.equal(cache.cpu(), model)
        assert ((out.cpu().double() - want).abs() <= tol).all()
        return groups

    mgr.allocate_slots(first, True)
    step([first], [330], False)
    for r in rest:
        mgr.allocate_slots(r, True)
    assert all(mgr.num_cached_tokens(r) == 256 for r in rest)
    groups = step(rest, [len(r) - 256 for r in rest], False)
    assert groups == ([0, 4], [256])
    everyone = [first, *rest]
    for _ in range(3):
        for r in everyone:
            r.token_ids.append(7)
            mgr.allocate_slots(r, False)
        assert step(everyone, [1] * 5, True) == ([0, 5], [256])
