"""Calls of the latent store and the rotation that are refused, or mended, before anything is launched."""
from __future__ import annotations

import math

import pytest

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
