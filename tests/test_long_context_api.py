"""The entries over long contexts without a device: the C ABI's refusals, the package's argument checks, the block
manager's groups."""
from __future__ import annotations

import random
from dataclasses import dataclass, field
from typing import List

import pytest
import torch

from conftest import PKG

LIB = PKG._lib.load()
FAKE = 0x10000  # 256-byte aligned, never dereferenced on the host


def _err():
    return LIB.pa_last_error().decode()


# ---------------------------------------------------------------------------
# C ABI
# ---------------------------------------------------------------------------
def _bounds(**over):
    a = dict(k=FAKE, pages=4, page=64, ps=64 * 256, ss=256, hs=128, bt=FAKE, bts=4, pps=4, lens=FAKE, cu=None, batch=2,
             most=1, hkv=2, dim=128, block=16, bounds=FAKE, bps=4 * 512, bbs=512, bhs=256, stream=None)
    a.update(over)
    return LIB.pa_block_bounds(*a.values())


def _scores(**over):
    a = dict(q=FAKE, qb=1024, qh=128, bounds=FAKE, pages=4, page=64, bps=4 * 512, bbs=512, bhs=256, bt=FAKE, bts=4,
             pps=4, lens=FAKE, batch=2, heads=8, hkv=2, dim=128, block=16, scale=0.1, scores=FAKE, sb=32, sh=16,
             stream=None)
    a.update(over)
    return LIB.pa_block_scores(*a.values())


def _select(**over):
    a = dict(scores=FAKE, sb=32, sh=16, width=16, lens=FAKE, batch=2, hkv=2, block=16, num=8, first=1, recent=2,
             out=FAKE, ob=16, oh=8, stream=None)
    a.update(over)
    return LIB.pa_select_blocks(*a.values())


def _sparse(**over):
    a = dict(q=FAKE, qb=1024, qh=128, k=FAKE, v=FAKE, pages=4, page=64, ps=64 * 256, ss=256, hs=128, bt=FAKE, bts=4,
             pps=4, lens=FAKE, batch=2, heads=8, hkv=2, dim=128, sel=FAKE, selb=16, selh=8, num=8, block=16, scale=0.1,
             cap=0.0, out=FAKE, ob=1024, oh=128, ws=FAKE, wsb=1 << 40, stream=None)
    a.update(over)
    return LIB.pa_block_sparse_decode(*a.values())


def _shared(**over):
    a = dict(q=FAKE, qt=1024, qh=128, k=FAKE, v=FAKE, pages=4, page=64, ps=64 * 256, ss=256, hs=128, bt=FAKE, bts=4,
             pps=4, lens=FAKE, cug=FAKE, shared=FAKE, groups=1, cu=None, batch=2, tokens=2, most=1, heads=8, hkv=2,
             dim=128, scale=0.1, cap=0.0, zero=0, out=FAKE, ot=1024, oh=128, ws=FAKE, wsb=1 << 40, stream=None)
    a.update(over)
    return LIB.pa_shared_prefix(*a.values())


@pytest.mark.parametrize("call", [_bounds, _scores, _sparse])
def test_block_refusals(call):
    assert call(batch=0) == 0
    assert call(batch=-1) == -1 and "batch=-1" in _err()
    assert call(pages=0) == -1
    assert call(pps=-1) == -1
    for block in (0, -16, 8, 24, 48, 128):
        assert call(block=block) == -1 and "block" in _err()
    for dim in (0, 32, 80, 96, 512):
        assert call(dim=dim) == -2 and "head_dim" in _err()
    assert call(pps=1 << 26) == -2 and "2^31" in _err()
    assert call(lens=None) == -1 and "null" in _err()
    assert call(bt=None) == -1


def test_bounds_refusals():
    assert _bounds(pps=0) == 0
    assert _bounds(most=-1) == -1
    assert _bounds(k=FAKE + 8) == -2 and "aligned" in _err()
    assert _bounds(bounds=FAKE + 2) == -2
    assert _bounds(ss=260) == -2 and _bounds(bhs=252) == -2
    assert _bounds(hkv=1 << 17) == -2


def test_scores_refusals():
    assert _scores(heads=9) == -1 and _scores(heads=0) == -1
    for scale in (0.0, -1.0, float("nan")):
        assert _scores(scale=scale) == -1 and "positive" in _err()
    assert _scores(q=FAKE + 8) == -2 and _scores(qh=130) == -2


def test_select_refusals():
    assert _select(batch=0) == 0
    for bad in (dict(batch=-1), dict(hkv=0), dict(width=-1), dict(block=0), dict(num=0), dict(first=-1), dict(recent=-1)):
        assert _select(**bad) == -1, bad
    assert _select(first=5, recent=4) == -1 and "fit" in _err()
    assert _select(first=0x7fffffff, recent=0x7fffffff) == -1
    assert _select(scores=None) == -1 and _select(out=None) == -1


def test_sparse_refusals():
    assert _sparse(heads=7) == -1 and _sparse(num=0) == -1
    assert _sparse(page=512, block=512) == -2 and "256" in _err()
    assert _sparse(out=FAKE + 4) == -2
    need = LIB.pa_block_sparse_decode_workspace_size(2, 8, 2, 128, 64, 32)
    assert need > 0
    assert _sparse(num=64, block=32, wsb=need - 1) == -3 and str(need) in _err()
    assert _sparse(num=64, block=32, ws=None, wsb=0) == -3
    assert LIB.pa_block_sparse_decode_workspace_size(2, 8, 3, 128, 64, 32) == 0
    # a full chip's worth of sequences takes no partials
    assert LIB.pa_block_sparse_decode_workspace_size(256, 32, 8, 128, 64, 32) == 0


def test_shared_refusals():
    assert _shared(batch=0, tokens=0) == 0
    for bad in (dict(batch=-1), dict(groups=-1), dict(tokens=-1), dict(most=-1), dict(heads=9), dict(hkv=0),
                dict(pages=0), dict(page=0), dict(pps=-1)):
        assert _shared(**bad) == -1, bad
    assert _shared(tokens=3) == -1 and "without cu_seqlens_q" in _err()
    assert _shared(pps=0) == -1 and _shared(cu=FAKE, most=0) == -1
    assert _shared(dim=64) == -2 and "128" in _err()
    assert _shared(heads=514) == -2 and "257" in _err()
    assert _shared(pps=1 << 25) == -2 and "2^31" in _err()
    assert _shared(ss=1 << 40) == -2
    assert _shared(cug=None) == -1 and _shared(shared=None) == -1
    assert _shared(q=FAKE + 8) == -2 and _shared(ws=FAKE + 128) == -2 and _shared(oh=100) == -2
    need = LIB.pa_shared_prefix_workspace_size(2, 1, 2, 1, 0, 8, 2, 4, 64)
    assert need > 0 and _shared(wsb=need - 1) == -3 and str(need) in _err()
    assert LIB.pa_shared_prefix_workspace_size(2, 1, 2, 1, 0, 9, 2, 4, 64) == 0


def test_shared_workspace_holds_what_the_plan_may_make():
    """Parts of row tiles and chunks of the widest step, counted as the plan counts them, fit what the sizes say: the
    bytes grow with each of the step's numbers."""
    base = dict(batch=8, groups=2, tokens=8, most=1, ragged=0, heads=32, hkv=8, pps=64, page=64)
    size = lambda **o: LIB.pa_shared_prefix_workspace_size(*{**base, **o}.values())  # noqa: E731
    for more in (dict(batch=16, tokens=16), dict(groups=8), dict(pps=1024), dict(heads=64)):
        assert size(**more) > size()
    many = dict(ragged=1, most=100)
    assert size(**many, tokens=800) > size(**many, tokens=100)


# ---------------------------------------------------------------------------
# the package's checks: no CPU path
# ---------------------------------------------------------------------------
def test_tensors_off_the_device():
    cache = torch.zeros((2, 4, 64, 2, 128), dtype=torch.bfloat16)
    q = torch.zeros((2, 8, 128), dtype=torch.bfloat16)
    table, lens = torch.zeros((2, 4), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    bounds = PKG.new_block_bounds(cache, 16)
    assert bounds.shape == (4, 4, 2, 2, 128)
    prefixes = PKG.SharedPrefixes.of([0, 2], [64], "cpu")
    for call in (lambda: PKG.update_block_bounds(bounds, cache, table, lens),
                 lambda: PKG.block_scores(q, bounds, table, lens, page_size=64, scale=1.0),
                 lambda: PKG.select_blocks(torch.zeros((2, 2, 16)), lens, 4, block=16),
                 lambda: PKG.block_sparse_decode_attention(q, cache, table, lens, lens.view(2, 1, 1), block=16, scale=1.0),
                 lambda: PKG.shared_prefix_attention(q, cache, table, lens, prefixes, scale=1.0)):
        with pytest.raises(ValueError, match="HIP device"):
            call()
    with pytest.raises(TypeError, match="SharedPrefixes"):
        PKG.shared_prefix_attention(q, cache, table, lens, ([0, 2], [64]), scale=1.0)
    for block in (0, 8, 24, 128, 16.0):
        with pytest.raises(ValueError, match="multiple of 16"):
            PKG.new_block_bounds(cache, block)
    with pytest.raises(ValueError, match="kv_cache"):
        PKG.new_block_bounds(cache[0], 16)


def test_where_sharing_pays():
    assert not PKG.shared_prefix_pays(4, 1, 8, 2560)           # a few chats
    assert PKG.shared_prefix_pays(128, 1, 8, 9216)             # a serving batch
    assert not PKG.shared_prefix_pays(128, 128, 8, 9216)       # no two together
    assert not PKG.shared_prefix_pays(128, 0, 8, 9216)


# ---------------------------------------------------------------------------
# the block manager's groups
# ---------------------------------------------------------------------------
@dataclass
class Request:
    id: int
    token_ids: List[int] = field(default_factory=list)

    def __len__(self):
        return len(self.token_ids)


def test_groups_of_a_cached_prompt():
    m = PKG.KVCacheManager(200, 16, enable_prefix_caching=True)
    system, other = list(range(100)), list(range(500, 600))
    batch = [Request(i, system + [1000 + i] * (5 + i)) for i in range(3)] + [Request(9, other)] + \
            [Request(20 + i, other[:64] + [7 + i] * 40) for i in range(2)]
    for r in batch:
        m.allocate_slots(r, True)
    cu, shared = m.shared_prefixes(batch)
    # 100 tokens are six whole blocks; the fourth request shares four with those behind it
    assert (cu, shared) == ([0, 3, 6], [96, 64])
    assert m.shared_prefixes(batch[:1]) == ([0, 1], [0])
    assert m.shared_prefixes([]) == ([0], [])
    assert m.shared_prefixes([batch[0], batch[3], batch[1]]) == ([0, 1, 2, 3], [0, 0, 0])


def test_groups_of_forks_and_unknown_requests():
    m = PKG.KVCacheManager(50, 16)
    parent = Request(1, list(range(40)))
    m.allocate_slots(parent, True)
    kids = [Request(2, list(range(40))), Request(3, list(range(40)))]
    for k in kids:
        m.fork(parent, k)
    assert m.shared_prefixes([parent, *kids]) == ([0, 3], [48])
    kids[0].token_ids.append(5)
    m.allocate_slots(kids[0], False)          # its third block is its own now
    assert m.shared_prefixes([parent, *kids]) == ([0, 3], [32])
    before = m.num_free_blocks
    assert m.shared_prefixes([Request(77), parent, kids[1], Request(78)]) == ([0, 1, 3, 4], [0, 48, 0])
    assert m.num_free_blocks == before


def test_groups_save_reads():
    """A neighbour that shares little does not break up those that share much."""
    m = PKG.KVCacheManager(400, 16, enable_prefix_caching=True)
    long = list(range(320))
    batch = [Request(i, long + [i]) for i in range(4)] + [Request(10, long[:16] + [5] * 100)]
    for r in batch:
        m.allocate_slots(r, True)
    assert m.shared_prefixes(batch) == ([0, 4, 5], [320, 0])
    assert m.shared_prefixes([batch[0], batch[4]]) == ([0, 2], [16])


def test_groups_against_a_plain_count():
    rng = random.Random(3)
    m = PKG.KVCacheManager(2000, 4, enable_prefix_caching=True)
    stems = [[rng.randrange(99) for _ in range(40)] for _ in range(3)]
    batch = []
    for i in range(30):
        r = Request(i, rng.choice(stems)[:rng.randrange(1, 40)] + [200 + i] * rng.randrange(1, 9))
        m.allocate_slots(r, True)
        batch.append(r)
    cu, shared = m.shared_prefixes(batch)
    assert cu[0] == 0 and cu[-1] == 30 and all(a < b for a, b in zip(cu, cu[1:]))
    for g, (a, b) in enumerate(zip(cu, cu[1:])):
        tables = [m.block_ids(r) for r in batch[a:b]]
        common = 0
        while all(len(t) > common and t[common] == tables[0][common] for t in tables):
            common += 1
        assert shared[g] == (4 * common if b - a > 1 else 0)
