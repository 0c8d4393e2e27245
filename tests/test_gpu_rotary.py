"""rotary_embedding and latent_store against float64.

A rotated value is two float32 products and a sum of them, rounded once: the angle is off by 2.3e-8 rad, cos and sin
by up to 2 units of 2^-24, their factor, the products and the sum by half a unit each, so under 6 units of
2^-24 (|a| + |b|) amp together, plus half a step of the output's type."""
from __future__ import annotations

import pytest
import torch

import latent_reference as ref

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _bound(want, size, dtype):
    return HALF[dtype] * want.abs() + 6 * 2.0 ** -24 * size + (2.0 ** -25 if dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,dim,rot,start", [
    (1, 1, 64, 64, 0), (7, 20, 80, 40, 0), (5, 3, 192, 64, 128), (33, 16, 128, 128, 0), (3, 65, 96, 32, 64),
    (2, 5, 50, 6, 3), (4, 2, 7, 2, 5), (3, 2, 512, 512, 0), (1, 128, 192, 64, 128), (9, 4, 256, 20, 4)])
def test_rotary(pkg, dev, tokens, heads, dim, rot, start, interleaved, dtype):
    gen = torch.Generator().manual_seed(tokens * 1000 + dim)
    x = torch.randn((tokens, heads, dim), generator=gen).to(dtype).to(dev)
    pos = torch.randint(0, 1 << 20, (tokens,), generator=gen, dtype=torch.int32).to(dev)
    pos[0] = 0
    freqs = pkg.rotary_frequencies(rot, 1e4, device=dev)
    y = pkg.rotary_embedding(x, pos, freqs, start=start, interleaved=interleaved)
    part = slice(start, start + rot)
    want, size = ref.rotate(x[..., part], pos, freqs.inv_freq, 1.0, interleaved)
    assert ((y[..., part].double() - want).abs() <= _bound(want, size, dtype)).all()
    rest = [i for i in range(dim) if not start <= i < start + rot]
    assert torch.equal(y[..., rest], x[..., rest])
    # in place, and into a strided out inside a wider tensor: the same bits, nothing else touched
    z = x.clone()
    assert pkg.rotary_embedding(z, pos, freqs, start=start, interleaved=interleaved, out=z) is z
    assert torch.equal(z, y)
    wide = torch.full((tokens, heads + 1, dim + 8), 7.0, dtype=dtype, device=dev)
    pkg.rotary_embedding(x, pos, freqs, start=start, interleaved=interleaved, out=wide[:, 1:, 8:])
    assert torch.equal(wide[:, 1:, 8:], y)
    assert (wide[:, 0] == 7).all() and (wide[..., :8] == 7).all()


def test_rotary_strided_and_unaligned_rows(pkg, dev):
    """A slice of a projection, one that starts off a 16-byte boundary, and a broadcast input."""
    gen = torch.Generator().manual_seed(3)
    base = torch.randn((6, 5, 200), generator=gen).to(torch.bfloat16).to(dev)
    pos = torch.arange(6, dtype=torch.int32, device=dev) * 1001
    freqs = pkg.rotary_frequencies(32, 1e6, device=dev)
    for x in (base[:, 1:4, 8:104], base[:, :, 3:100], base[:, :1].expand(6, 5, 200), base.transpose(0, 1)[:, :5]):
        p = pos[:x.shape[0]]
        for inter in (False, True):
            y = pkg.rotary_embedding(x, p, freqs, start=16, interleaved=inter)
            want, size = ref.rotate(x[..., 16:48], p, freqs.inv_freq, 1.0, inter)
            assert ((y[..., 16:48].double() - want).abs() <= _bound(want, size, torch.bfloat16)).all()
            assert torch.equal(y[..., :16], x[..., :16]) and torch.equal(y[..., 48:], x[..., 48:])


@pytest.mark.parametrize("scaling", [dict(type="linear", factor=4), dict(type="ntk", factor=8),
                                     dict(type="yarn", factor=32, original_max_position=4096)])
def test_rotary_scaled_far_positions(pkg, dev, scaling):
    """Positions up to 2^31 - 1, negative ones too: the angle is a float64 product."""
    freqs = pkg.rotary_frequencies(64, 1e4, scaling=scaling, device=dev)
    pos = torch.tensor([0, 1, 131071, 1 << 24, (1 << 31) - 1, -5, -(1 << 30)], dtype=torch.int32, device=dev)
    x = torch.randn((7, 4, 64), generator=torch.Generator().manual_seed(1)).to(dev)
    y = pkg.rotary_embedding(x, pos, freqs, interleaved=True)
    want, size = ref.rotate(x, pos, freqs.inv_freq, freqs.amplitude, True)
    # float64 angles of 2^31 are off by 2^-53 * 2^31 on both sides: 5e-7 rad more
    assert ((y.double() - want).abs() <= _bound(want, size, torch.float32) + 1e-6 * size).all()


def test_rotary_no_tokens(pkg, dev):
    freqs = pkg.rotary_frequencies(32, 1e4, device=dev)
    x = torch.empty((0, 4, 64), device=dev)
    assert pkg.rotary_embedding(x, torch.empty(0, dtype=torch.int32, device=dev), freqs).shape == (0, 4, 64)


# ---------------------------------------------------------------------------
# latent_store
# ---------------------------------------------------------------------------
def _store_case(dev, tokens, heads, r, dr, nb, bs, seed):
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=gen).to(torch.bfloat16).to(dev)  # noqa: E731
    projected = rnd(tokens, r + dr + 8) * 3
    q = rnd(tokens, max(heads, 1), 128 + dr)
    slots = torch.randperm(nb * bs, generator=gen)[:tokens].to(torch.int32)
    pos = torch.randint(0, 200000, (tokens,), generator=gen, dtype=torch.int32)
    return projected, q, slots.to(dev), pos.to(dev), (1 + 0.2 * rnd(r).float()).to(torch.bfloat16), rnd(nb, bs, r + dr)


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,r,dr,nb,bs", [
    (1, 16, 512, 64, 3, 16), (4, 0, 512, 64, 2, 7), (37, 5, 512, 32, 50, 1), (19, 128, 256, 64, 4, 256),
    (65, 33, 256, 32, 9, 17)])
def test_store(pkg, dev, tokens, heads, r, dr, nb, bs, interleaved):
    projected, q, slots, pos, w, cache = _store_case(dev, tokens, heads, r, dr, nb, bs, tokens + r)
    latent, k_rope, q_rope = projected[:, :r], projected[:, r:r + dr], q[..., 128:]
    if tokens > 3:
        slots[1], slots[3] = -1, nb * bs  # padding tokens: outside the pool
    freqs = pkg.rotary_frequencies(dr, 1e4, device=dev)
    for norm in (w, None):
        before = cache.clone()
        got, q_rot = pkg.latent_store(latent, k_rope, norm, pos, slots, before, freqs, eps=1e-5,
                                      interleaved=interleaved, q_rope=q_rope if heads else None)
        assert got is before
        c = latent.double()
        if norm is not None:
            c = c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-5) * w.double()
        kr, size = ref.rotate(k_rope[:, None], pos, freqs.inv_freq, 1.0, interleaved)
        ok = (slots >= 0) & (slots < nb * bs)
        rows = before.view(nb * bs, r + dr)
        written = slots[ok].long()
        # the mean of 512 squares, its root and quotient and two products: 8 units of 2^-24
        cap = (2.0 ** -8 + (0 if norm is None else 8 * 2.0 ** -24)) * c[ok].abs()
        assert ((rows[written, :r].double() - c[ok]).abs() <= (cap if norm is not None else 0)).all()
        assert ((rows[written, r:].double() - kr[ok, 0]).abs() <= _bound(kr, size, torch.bfloat16)[ok, 0]).all()
        others = torch.ones(nb * bs, dtype=torch.bool, device=dev)
        others[written] = False
        assert torch.equal(rows[others], cache.view(nb * bs, r + dr)[others])
        if heads:
            want, size = ref.rotate(q_rope, pos, freqs.inv_freq, 1.0, interleaved)
            assert ((q_rot.double() - want).abs() <= _bound(want, size, torch.bfloat16)).all()
            qq = q.clone()   # in place on the slice of q's heads: the rest of q stays
            _, out = pkg.latent_store(latent, k_rope, norm, pos, slots, before, freqs, eps=1e-5,
                                      interleaved=interleaved, q_rope=qq[..., 128:], q_out=qq[..., 128:])
            assert torch.equal(qq[..., 128:], q_rot) and torch.equal(qq[..., :128], q[..., :128])
        else:
            assert q_rot is None


def test_store_strided_pool_past_32_bits(pkg, dev):
    """Pages more than 2^31 elements apart (a pool that is one layer of a larger buffer)."""
    r, dr, bs = 256, 32, 4
    stride = (1 << 31) + 8
    buf = torch.zeros(stride + bs * (r + dr), dtype=torch.bfloat16, device=dev)
    cache = buf.as_strided((2, bs, r + dr), (stride, r + dr, 1))
    x = torch.randn((2, r + dr), generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(dev)
    freqs = pkg.rotary_frequencies(dr, 1e4, device=dev)
    zero = torch.zeros(2, dtype=torch.int32, device=dev)
    pkg.latent_store(x[:, :r], x[:, r:], None, zero, torch.tensor([1, 6], dtype=torch.int32, device=dev), cache, freqs)
    assert torch.equal(cache[0, 1], x[0]) and torch.equal(cache[1, 2], x[1])
    assert int((cache[1].abs().sum(-1) != 0).sum()) == 1
