"""How often the absorbed attention rounds a softmax weight.

Every token's latent row is a unit vector and W_uv picks some of them out, so that an output is one token's weight: the
product with V adds nothing to it.  It is rounded to bf16 where the matrix cores take it and as the latent-wide result;
the projection takes that times one, which rounds nothing more.  Two roundings, by half a step each: (1 + 2^-8)^2 - 1,
and 2^-17 for the float32 exponentials, sums and quotient at scores of up to 44 in log2 units."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("spread", [3.0, 30.0])
@pytest.mark.parametrize("tokens", [32, 64, 200])
def test_weights_are_rounded_once(pkg, dev, tokens, spread):
    r, dr, dn, batch = 256, 32, 64, 2048
    gen = torch.Generator().manual_seed(tokens)
    s = (torch.rand((batch, tokens), generator=gen) * spread).to(torch.bfloat16).to(dev)
    cache = torch.zeros((batch, tokens, r + dr), dtype=torch.bfloat16, device=dev)
    cache[:, :, :tokens] = torch.eye(tokens, dtype=torch.bfloat16, device=dev)
    cache[:, :, r] = s
    some = torch.randperm(tokens, generator=gen)[:dn].to(dev)
    w = torch.zeros((2 * dn, r), dtype=torch.bfloat16, device=dev)
    w[dn + torch.arange(len(some), device=dev), some] = 1
    weights = pkg.LatentWeights(w, num_heads=1, nope_dim=dn, v_dim=dn)
    q_nope = torch.zeros((batch, 1, dn), dtype=torch.bfloat16, device=dev)
    q_rope = torch.zeros((batch, 1, dr), dtype=torch.bfloat16, device=dev)
    q_rope[..., 0] = 1
    table = torch.arange(batch, dtype=torch.int32, device=dev)[:, None]
    lens = torch.full((batch,), tokens, dtype=torch.int32, device=dev)
    out = pkg.latent_decode_attention(q_nope, q_rope, cache, weights, table, lens, scale=1.0)[:, 0, :len(some)]
    want = torch.softmax(s.double(), 1)[:, some]
    worst = float((out.double() / want - 1).abs().max())
    bound = (1 + 2.0 ** -8) ** 2 - 1 + 2.0 ** -17
    print(f"{tokens} tokens: off by {worst * 256:.3f} half steps of {bound * 256:.3f}", flush=True)
    assert worst <= bound
