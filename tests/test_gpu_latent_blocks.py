"""The block manager's page copies on a pool of latent rows."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("row", [288, 320, 544, 576])
@pytest.mark.parametrize("page", [1, 16, 7])
def test_copy_blocks_of_latent_rows(pkg, dev, row, page):
    gen = torch.Generator().manual_seed(row)
    pool = torch.randn((9, page, row), generator=gen).to(torch.bfloat16).to(dev)
    want = pool.clone()
    want[5], want[0], want[8] = pool[2], pool[7], pool[2]
    pkg.copy_blocks(pool, [2, 7, 2], [5, 0, 8])
    assert torch.equal(pool, want)
    # a layer of a wider buffer: nothing beside it is written
    wide = torch.randn((6, page + 1, row + 8), generator=gen).to(torch.bfloat16).to(dev)
    want = wide.clone()
    want[4, 1:, :row] = wide[1, 1:, :row]
    pkg.copy_blocks(wide[:, 1:, :row], [1], [4])
    assert torch.equal(wide, want)
    with pytest.raises(ValueError, match="R \\+ Dr"):
        pkg.copy_blocks(pool[0], [0], [0])


def test_fork_of_a_latent_sequence(pkg, dev):
    """A forked sequence's next token goes to a copy of the shared page: the parent's rows stay, the child sees them."""
    heads, r, dr, dn, page = 2, 256, 32, 64, 4
    gen = torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=gen).to(torch.bfloat16).to(dev)  # noqa: E731
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    pool = torch.full((4, page, r + dr), float("nan"), dtype=torch.bfloat16, device=dev)
    freqs = pkg.rotary_frequencies(dr, 1e4, device=dev)
    weights = pkg.LatentWeights(rnd(heads * 2 * dn, r), num_heads=heads, nope_dim=dn, v_dim=dn)
    x = rnd(7, r + dr)
    store = lambda t, slots: pkg.latent_store(  # noqa: E731
        x[t, :r], x[t, r:], None, i32(*range(t.start, t.stop)), i32(*slots), pool, freqs)
    store(slice(0, 6), (0, 1, 2, 3, 8, 9))             # the parent: pages 0 and 2
    parent = pool.clone()
    pkg.copy_blocks(pool, [2], [3])                    # the child's copy of its last page
    store(slice(6, 7), (14,))
    assert torch.equal(pool[:3].view(torch.int16), parent[:3].view(torch.int16))
    assert torch.equal(pool[3, :2], pool[2, :2])
    qn, qr = rnd(1, heads, dn), rnd(1, heads, dr)
    flat = torch.cat([pool[0], pool[3, :3]])[None]     # the child's rows as a pool of one page
    child = pkg.latent_decode_attention(qn, qr, pool, weights, i32(0, 3).view(1, 2), i32(7), scale=0.1)
    alone = pkg.latent_decode_attention(qn, qr, flat.contiguous(), weights, i32(0).view(1, 1), i32(7), scale=0.1)
    assert torch.isfinite(child).all() and torch.equal(child, alone)
