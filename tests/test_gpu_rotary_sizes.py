"""rotary_embedding at the far ends of the sizes that it takes."""
from __future__ import annotations

import pytest
import torch

import latent_reference as ref
from test_gpu_rotary import _bound

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,heads,dim,rot,interleaved", [
    (torch.float32, 4036, 4156, 64, True), (torch.bfloat16, 1003, 16712, 64, True),
    (torch.float32, 64, 32952, 128, False), (torch.bfloat16, 64, 65840, 128, False),
    (torch.float32, 2048, 6128, 64, False), (torch.float16, 1, 1 << 24, 512, False),
    (torch.float16, 1 << 23, 2, 2, True)])
def test_rotary_largest_rows(pkg, dev, dtype, heads, dim, rot, interleaved):
    """Close to 2^24 elements a token, where a piece's number needs all its bits to give its head: every element is
    rotated or copied, and nothing behind the rows is written."""
    print(f"{dtype} {heads} heads of {dim}, {rot} rotated", flush=True)
    gen = torch.Generator(device=dev).manual_seed(dim)
    x = torch.randn((2, heads, dim), generator=gen, device=dev).to(dtype)
    pos = torch.tensor([3, 70001], dtype=torch.int32, device=dev)
    freqs = pkg.rotary_frequencies(rot, 1e4, device=dev)
    start = dim - rot if heads > 64 else 0
    buf = torch.full((x.numel() + 4096,), 7.0, dtype=dtype, device=dev)
    out = buf[:x.numel()].view(x.shape)
    pkg.rotary_embedding(x, pos, freqs, start=start, interleaved=interleaved, out=out)
    assert (buf[x.numel():] == 7).all()
    want, size = ref.rotate(x[..., start:start + rot], pos, freqs.inv_freq, 1.0, interleaved)
    assert ((out[..., start:start + rot].double() - want).abs() <= _bound(want, size, dtype)).all()
    assert torch.equal(out[..., :start], x[..., :start]) and torch.equal(out[..., start + rot:], x[..., start + rot:])


def test_rotary_many_tokens(pkg, dev):
    """More tokens than one grid has workgroups of 256 threads for."""
    tokens = (1 << 24) + 5
    gen = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn((tokens, 1, 4), generator=gen, device=dev)
    pos = torch.arange(tokens, dtype=torch.int32, device=dev)
    freqs = pkg.rotary_frequencies(2, 1e4, device=dev)
    buf = torch.full((x.numel() + 64,), 7.0, device=dev)
    y = pkg.rotary_embedding(x, pos, freqs, start=1, out=buf[:x.numel()].view(x.shape))
    assert (buf[x.numel():] == 7).all()
    assert torch.equal(y[..., 0], x[..., 0]) and torch.equal(y[..., 3], x[..., 3])
    for t0 in range(0, tokens, 1 << 22):
        t = slice(t0, min(tokens, t0 + (1 << 22)))
        want, size = ref.rotate(x[t, :, 1:3], pos[t], freqs.inv_freq, 1.0, False)
        assert ((y[t, :, 1:3].double() - want).abs() <= _bound(want, size, torch.float32)).all()


def test_store_many_tokens(pkg, dev):
    """One row stored by the last tokens of more than a grid has workgroups for; the padding tokens before them write
    nothing."""
    tokens, r, dr = (1 << 26) + 3, 256, 32
    gen = torch.Generator().manual_seed(2)
    row = torch.randn((1, r + dr), generator=gen).to(torch.bfloat16).to(dev)
    slots = torch.full((tokens,), -1, dtype=torch.int32, device=dev)
    at = torch.tensor([0, 1 << 23, (1 << 24) - 1, 1 << 25, tokens - 1], device=dev)
    slots[at] = torch.arange(5, dtype=torch.int32, device=dev)
    pos = torch.arange(tokens, dtype=torch.int32, device=dev)
    cache = torch.full((2, 4, r + dr), 3.0, dtype=torch.bfloat16, device=dev)
    freqs = pkg.rotary_frequencies(dr, 1e4, device=dev)
    x = row.expand(tokens, r + dr)
    pkg.latent_store(x[:, :r], x[:, r:], None, pos, slots, cache, freqs)
    rows = cache.view(8, r + dr)
    assert torch.equal(rows[:5, :r], row[:, :r].expand(5, r)) and (rows[5:] == 3).all()
    want, size = ref.rotate(row[:, None, r:].expand(5, 1, dr), pos[at], freqs.inv_freq, 1.0, True)
    assert ((rows[:5, r:].double() - want[:, 0]).abs() <= _bound(want, size, torch.bfloat16)[:, 0]).all()
