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
