"""latent_decode_attention against float64 (bounds: latent_reference)."""
from __future__ import annotations

import math

import pytest
import torch

import latent_reference as ref

pytestmark = pytest.mark.gpu


def make(dev, lengths, heads, r, dr, dn, page, seed, *, width=None, gain=1.0):
    """Inputs with every cache row that no sequence owns set to NaN, pages in a random order, -1 behind them."""
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    need = [-(-n // page) for n in lengths]
    nb = sum(need) + 3
    perm = torch.randperm(nb, generator=gen)
    table = torch.full((len(lengths), width or max(need + [1])), -1, dtype=torch.int32)
    cache = torch.full((nb, page, r + dr), float("nan"))
    rows, at = [], 0
    for b, (n, k) in enumerate(zip(lengths, need)):
        ids = perm[at:at + k]
        at += k
        table[b, :k] = ids.to(torch.int32)
        x = rnd(n, r + dr).to(torch.bfloat16)
        rows.append(x.to(dev))
        flat = torch.full((k * page, r + dr), float("nan"))
        flat[:n] = x.float()
        cache[ids] = flat.view(k, page, r + dr)
    q = (rnd(len(lengths), heads, dn + dr) * gain).to(torch.bfloat16).to(dev)
    w = (rnd(heads * 2 * dn, r) * r ** -0.5).to(torch.bfloat16).to(dev)
    return dict(q=q, w=w, cache=cache.to(torch.bfloat16).to(dev), table=table.to(dev), rows=rows,
                lens=torch.tensor(lengths, dtype=torch.int32, device=dev))


def reference(c, heads, r, dn, scale, form="absorbed", lengths=None):
    w = c["w"].view(heads, 2, dn, r)
    outs = []
    for b, rows in enumerate(c["rows"]):
        per = [ref.attend(c["q"][b:b + 1, h, :dn], c["q"][b:b + 1, h, dn:], rows, w[h, 0], w[h, 1],
                          [rows.shape[0]], scale, form) for h in range(heads)]
        outs.append((torch.cat([o for o, _ in per]), torch.cat([s for _, s in per])))
    return torch.stack([o for o, _ in outs]), torch.stack([s for _, s in outs])


def run(pkg, c, heads, dn, scale, **kw):
    weights = pkg.LatentWeights(c["w"], num_heads=heads, nope_dim=dn, v_dim=dn)
    return pkg.latent_decode_attention(c["q"][..., :dn], c["q"][..., dn:], c["cache"], weights, c["table"], c["lens"],
                                       scale=scale, **kw)


@pytest.mark.parametrize("heads,r,dr,dn,page,lengths", [
    (16, 512, 64, 128, 16, [1]),
    (16, 512, 64, 128, 16, [0, 5, 0]),
    (1, 512, 64, 128, 64, [31, 32, 33, 1]),
    (5, 256, 32, 64, 7, [64, 65, 3, 127, 128, 129]),
    (20, 512, 32, 128, 1, [40, 2, 200]),
    (32, 512, 64, 128, 17, [95, 96, 97, 0, 300]),
    (33, 512, 64, 128, 256, [100, 257]),
    (64, 512, 64, 128, 64, [700, 1, 130]),
    (65, 256, 64, 64, 16, [150, 20]),
    (128, 512, 64, 128, 32, [333, 64]),
    (130, 256, 32, 128, 48, [1, 500]),
    (16, 512, 64, 64, 5, [2500]),
    (64, 256, 64, 128, 256, [4097]),
])
def test_decode(pkg, dev, heads, r, dr, dn, page, lengths):
    print(f"heads {heads} latent {r}+{dr} head {dn} page {page} lengths {lengths}", flush=True)
    c = make(dev, lengths, heads, r, dr, dn, page, seed=heads + sum(lengths))
    scale = (dn + dr) ** -0.5
    got = run(pkg, c, heads, dn, scale)
    want, spread = reference(c, heads, r, dn, scale)
    for b, n in enumerate(lengths):
        if n == 0:
            assert not got[b].any(), "a sequence without rows gives a zero row"
    ref.check(got, want, spread, "decode")
    assert torch.equal(got, run(pkg, c, heads, dn, scale)), "the same call gives the same bits"


def test_decode_many_ragged_sequences(pkg, dev):
    """More sequences than one pass of the cut's scan holds, most of them short or empty; rows checked in part."""
    gen = torch.Generator().manual_seed(9)
    lengths = torch.randint(0, 40, (700,), generator=gen).tolist()
    lengths[0], lengths[333], lengths[699] = 900, 2000, 0
    c = make(dev, lengths, 4, 256, 32, 64, 16, seed=10)
    got = run(pkg, c, 4, 64, 0.1)
    w = c["w"].view(4, 2, 64, 256)
    for b in [0, 1, 2, 100, 332, 333, 334, 511, 512, 513, 698, 699]:
        for h in (0, 3):
            o, s = ref.attend(c["q"][b:b + 1, h, :64], c["q"][b:b + 1, h, 64:], c["rows"][b], w[h, 0], w[h, 1],
                              [lengths[b]], 0.1, "absorbed")
            ref.check(got[b:b + 1, h], o, s, f"sequence {b}")


def test_decode_large_scores(pkg, dev):
    """Scores of several hundred whose maximum keeps moving: every rescale of the running maximum."""
    c = make(dev, [400, 77], 16, 512, 64, 128, 16, seed=4, gain=40.0)
    for rows, t in zip(c["rows"], range(2)):
        assert rows.shape[0] > 0
    got = run(pkg, c, 16, 128, 0.2)
    want, spread = reference(c, 16, 512, 128, 0.2)
    ref.check(got, want, spread, "large scores")


def test_decode_strides_out_and_workspace(pkg, dev):
    """A pool whose rows and pages are apart, q in head-major order, a strided out, the caller's workspace."""
    heads, r, dr, dn, page = 20, 512, 64, 128, 16
    c = make(dev, [70, 33, 5], heads, r, dr, dn, page, seed=6, width=9)
    scale = 0.07
    plain = run(pkg, c, heads, dn, scale)
    nb = c["cache"].shape[0]
    wide = torch.full((nb, 2, page + 3, r + dr + 16), float("nan"), dtype=torch.bfloat16, device=dev)
    wide[:, 1, :page, 8:8 + r + dr] = c["cache"]
    weights = pkg.LatentWeights(c["w"], num_heads=heads, nope_dim=dn, v_dim=dn)
    q_hm = c["q"].transpose(0, 1).contiguous().transpose(0, 1)
    big = torch.full((3, heads + 2, dn + 8), 9.0, dtype=torch.bfloat16, device=dev)
    ws = torch.full((pkg.latent_decode_workspace_bytes(3, weights, 9, page),), 255, dtype=torch.uint8, device=dev)
    out = pkg.latent_decode_attention(q_hm[..., :dn], q_hm[..., dn:], wide[:, 1, :page, 8:8 + r + dr], weights,
                                      c["table"], c["lens"], scale=scale, workspace=ws, out=big[:, 1:-1, 8:])
    assert torch.equal(out, plain)
    assert (big[:, 0] == 9).all() and (big[:, -1] == 9).all() and (big[..., :8] == 9).all()


def test_decode_bad_tables_and_lengths_stay_in_bounds(pkg, dev):
    """Ids outside the pool are clamped into it, lengths past the table's span to the span, negative ones to zero."""
    c = make(dev, [40, 40, 40], 16, 256, 32, 64, 16, seed=8)
    c["cache"].nan_to_num_(nan=0.5)
    c["table"][0, 1] = 1 << 30
    c["table"][1, 0] = -7
    c["lens"][1] = 1 << 30
    c["lens"][2] = -3
    got = run(pkg, c, 16, 64, 0.1)
    assert torch.isfinite(got).all() and not got[2].any()


def test_decode_graph_replays_and_streams(pkg, dev):
    """Captured and replayed with new inputs between replays, eager calls on another stream beside it."""
    heads, dn = 16, 128
    c = make(dev, [300, 17, 1000, 64], heads, 512, 64, dn, 64, seed=12)
    weights = pkg.LatentWeights(c["w"], num_heads=heads, nope_dim=dn, v_dim=dn)
    call = lambda **kw: pkg.latent_decode_attention(c["q"][..., :dn], c["q"][..., dn:], c["cache"], weights,  # noqa: E731
                                                    c["table"], c["lens"], scale=0.07, **kw)
    call()
    out = torch.empty((4, heads, dn), dtype=torch.bfloat16, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out=out)
    side = torch.cuda.Stream()
    gen = torch.Generator().manual_seed(1)
    for i in range(4):
        c["q"].copy_(torch.randn(c["q"].shape, generator=gen).to(torch.bfloat16))
        c["lens"].copy_(torch.tensor([300 - 70 * i, 17, 1000 - 300 * i, 64 * (i % 2)], dtype=torch.int32))
        out.fill_(5.0)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = call()
        torch.cuda.synchronize()
        assert torch.equal(out, call()) and torch.equal(beside, out), f"replay {i}"


def test_decode_nothing(pkg, dev):
    c = make(dev, [4], 16, 512, 64, 128, 16, seed=1)
    weights = pkg.LatentWeights(c["w"], num_heads=16, nope_dim=128, v_dim=128)
    empty = c["q"][:0]
    out = pkg.latent_decode_attention(empty[..., :128], empty[..., 128:], c["cache"], weights, c["table"][:0],
                                      c["lens"][:0], scale=1.0)
    assert tuple(out.shape) == (0, 16, 128)
    # a table without any page
    none = pkg.latent_decode_attention(c["q"][..., :128], c["q"][..., 128:], c["cache"], weights, c["table"][:, :0],
                                       c["lens"], scale=1.0)
    assert not none.any() and math.isfinite(float(none.float().sum()))
