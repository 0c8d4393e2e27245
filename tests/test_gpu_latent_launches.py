"""Latent attention in batches whose workgroups or kv bounds are many, against float64 (bounds: latent_reference)."""
from __future__ import annotations

import pytest
import torch

import latent_reference as ref
from test_gpu_latent_prefill import form, make, run

pytestmark = pytest.mark.gpu


def test_prefill_more_items_than_one_grid_holds(pkg, dev):
    """One long prompt beside many short ones: query tiles x sequences x heads pass the workgroups of a grid."""
    heads, r, dr, dn, page = 256, 256, 32, 64, 16
    seqs = [(3, 3)] * 600 + [(16500, 16500)] + [(1, 1)] * 500
    c = make(dev, seqs, heads, r, dr, dn, page, seed=9, before=1, behind=2)
    assert form(pkg, c, heads, r, dr, dn, page) == "expanded"
    assert -(-16500 // 256) * len(seqs) * heads * 512 > 1 << 32
    scale = (dn + dr) ** -0.5
    out = run(pkg, c, heads, dn, scale)
    assert not out[:1].any() and not out[-2:].any()
    w = c["w"].view(heads, 2, dn, r)
    at = 1 + 600 * 3
    for b, q0, idx in ((0, 1, [0, 2]), (599, 1 + 599 * 3, [0, 1, 2]), (600, at, [0, 255, 256, 9000, 16499]),
                       (601, at + 16500, [0]), (1100, at + 16500 + 499, [0])):
        for h in (0, 200, heads - 1):
            q = c["q"][q0:q0 + seqs[b][0], h][idx]
            o, s = ref.attend(q[:, :dn], q[:, dn:], c["rows"][b], w[h, 0], w[h, 1], [i + 1 for i in idx], scale,
                              "expanded")
            ref.check(out[q0:q0 + seqs[b][0], h][idx], o, s, f"sequence {b} head {h}")


def test_absorbed_more_units_than_one_grid_holds(pkg, dev):
    """Short tables, but more row tiles than workgroups of a grid: the work is cut instead of a workgroup a row tile."""
    heads, r, dr, dn, page, batch = 512, 256, 32, 64, 16, 16384
    some = [0, 17, 9000, batch - 1]
    seqs = [(0, 0)] * batch
    for b in some:
        seqs[b] = (20, 20)
    c = make(dev, seqs, heads, r, dr, dn, page, seed=10)
    scale = (dn + dr) ** -0.5
    kw = dict(total_kv_tokens=20 * batch, max_seqlen_q=65, lengths="lens")   # bounds, not the lengths themselves
    lib = pkg._lib.load()
    assert lib.pa_latent_prefill_route(batch, 80, 65, 20 * batch, 2, page, heads, r, dr, dn) == 1
    assert batch * (65 * heads // 64) * 512 > 1 << 32
    out = run(pkg, c, heads, dn, scale, **kw)
    w = c["w"].view(heads, 2, dn, r)
    for i, b in enumerate(some):
        q = c["q"][20 * i:20 * i + 20]
        for h in (0, 63, heads - 1):
            o, s = ref.attend(q[:, h, :dn], q[:, h, dn:], c["rows"][b], w[h, 0], w[h, 1], range(1, 21), scale, "absorbed")
            ref.check(out[20 * i:20 * i + 20, h], o, s, f"sequence {b} head {h}")


@pytest.mark.parametrize("lengths", ["cu_k", "lens"])
@pytest.mark.parametrize("heads,seqs,want", [
    (3, [(90, 150), (96, 96), (80, 300), (90, 96), (95, 97), (0, 200), (96, 96)], "expanded"),
    (16, [(3, 150), (2, 50), (1, 300), (4, 96)], "absorbed")])
def test_prefill_lengths_past_the_tables(pkg, dev, heads, seqs, want, lengths):
    """A kv length past its table row's span is clamped to it, and takes nothing from the sequences behind."""
    r, dr, dn, page, span = 512, 64, 128, 16, 96
    c = make(dev, seqs, heads, r, dr, dn, page, seed=12)
    c["table"] = c["table"][:, :span // page]
    code = pkg._lib.load().pa_latent_prefill_route(len(seqs), c["q"].shape[0], max(n for n, _ in seqs), len(seqs) * span,
                                                   span // page, page, heads, r, dr, dn)
    assert ["expanded", "absorbed"][code] == want
    scale = (dn + dr) ** -0.5
    out = run(pkg, c, heads, dn, scale, lengths=lengths, total_kv_tokens=None)
    w = c["w"].view(heads, 2, dn, r)
    at = 0
    for b, (n, t) in enumerate(seqs):
        t = min(t, span)
        for h in (0, heads - 1) if n else ():
            q = c["q"][at:at + n, h]
            o, s = ref.attend(q[:, :dn], q[:, dn:], c["rows"][b][:t], w[h, 0], w[h, 1],
                              [t - n + i + 1 for i in range(n)], scale, want)
            ref.check(out[at:at + n, h], o, s, f"sequence {b} head {h}")
        at += n
