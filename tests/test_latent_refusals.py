"""Calls of the latent store and the rotation that are refused, or mended, before anything is launched."""
from __future__ import annotations

import math

import pytest
import torch

from conftest import PKG
from test_latent_api import FAKE, _err, _store


def test_store_in_place_needs_one_layout():
    """q_out on q_rope's memory with other strides: a token's workgroup would write rows that another still reads."""
    same = dict(q=2 * FAKE, qo=2 * FAKE, heads=4, tokens=3, qt=4 * 192, qh=192)
    for other in (dict(qot=4 * 64, qoh=64), dict(qot=4 * 192, qoh=64), dict(qot=2 * 192, qoh=192)):
        assert _store(**{**same, **other}) == -1 and "in place" in _err(), other


@pytest.mark.parametrize("factor", [0.25, 1.0, 1.5, 40.0])
def test_yarn_amplitude(factor):
    """The factor on cos and sin is 1 where nothing is stretched, never below it, and the caller's where it is given."""
    scaling = dict(type="yarn", factor=factor, original_max_position=4096)
    amplitude = PKG.rotary_frequencies(64, 1e4, scaling=scaling, device="cpu").amplitude
    assert math.isclose(amplitude, 0.1 * math.log(factor) + 1 if factor > 1 else 1.0)
    own = PKG.rotary_frequencies(64, 1e4, scaling=dict(scaling, attention_factor=0.9), device="cpu")
    assert own.amplitude == 0.9


def test_wide_tables_are_not_refused():
    """Without a bound the kv lengths may be as long as the tables are wide: however wide, the call is planned."""
    total = PKG.latent._total_kv(1024, 4096, 1 << 22, None, None, False)
    assert total == (1 << 31) - 1
    assert PKG.latent._total_kv(3, 10, 1 << 22, 100, None, False) == 300
    assert PKG.latent._total_kv(3, 10, 64, 100, None, False) == 192
    assert PKG.latent._total_kv(3, 10, 64, 100, 120, False) == 120
    assert PKG.latent._total_kv(3, 10, 64, None, None, True) == 10
    with pytest.raises(ValueError, match="bounded"):
        PKG.latent._total_kv(3, 10, 64, None, -1, False)
    lib = PKG._lib.load()
    args = (8, 4096, 512, total, 1 << 16, 64, 16, 512, 64, 128)
    assert lib.pa_latent_prefill_route(*args) == PKG._lib.PA_LATENT_ABSORBED
    assert lib.pa_latent_prefill_workspace_size(*args) < 1 << 30
    # one head of 16.8 M tokens (8 GiB) is still expanded
    args = (8, 4096, 512, 1 << 24, 1 << 9, 4096, 16, 512, 64, 128)
    assert lib.pa_latent_prefill_workspace_size(*args) < 11 << 30


def test_seam_passes_the_metadata_bounds(monkeypatch):
    """latent_attention hands the host's bounds of prefill and mixed steps on to the prefill."""
    seen = {}
    weights = object.__new__(PKG.LatentWeights)
    weights.num_heads, weights.nope_dim, weights.v_dim, weights.latent_dim = 2, 64, 64, 256
    monkeypatch.setattr(PKG.latent, "latent_store", lambda *a, q_rope, **k: (None, q_rope))
    monkeypatch.setattr(PKG.latent, "latent_decode_attention", lambda *a, out=None, **k: out)

    def prefill(q_nope, *a, **kw):
        seen.update(kw)
        return torch.zeros((q_nope.shape[0], 2, 64))

    monkeypatch.setattr(PKG.latent, "latent_prefill_attention", prefill)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    args = (None, torch.zeros((5, 2, 96)), None, None, None, weights, None)
    table = torch.zeros((3, 1000), dtype=torch.int32)
    mixed = (i32(0), i32(0), table, i32(0, 1, 2, 5), i32(4, 5, 6), 2, 3)
    prompts = (i32(0), i32(0), table, i32(0, 1, 2, 5), i32(0, 4, 9, 15), None)
    for meta, longest in [
            (PKG.MixedAttentionMetadata(*mixed), None),
            (PKG.MixedAttentionMetadata(*mixed, max_seqlen_k=6), 6),
            (PKG.MixedAttentionMetadata(*mixed, max_seqlen_k=torch.tensor(6)), 6),
            (PKG.PrefillAttentionMetadata(*prompts, max_seqlen_k=None, max_seqlen_bucket=3), None),
            (PKG.PrefillAttentionMetadata(*prompts, max_seqlen_k=6, max_seqlen_bucket=3), 6)]:
        for total in (None, 15):
            seen.clear()
            PKG.latent_attention(*args, meta, scale=1.0, total_kv_tokens=total)
            assert seen["max_seqlen_k"] == longest and seen["total_kv_tokens"] == total
