"""Calls of the latent store and the rotation that are refused, or mended, before anything is launched."""
from __future__ import annotations

from test_latent_api import FAKE, _err, _store

def test_store_in_place_needs_one_layout():
    """q_out on q_rope's memory with other strides: a token's workgroup would write rows that another still reads."""
    same = dict(q=2 * FAKE, qo=2 * FAKE, heads=4, tokens=3, qt=4 * 192, qh=192)
    for other in (dict(qot=4 * 64, qoh=64), dict(qot=4 * 192, qoh=64), dict(qot=2 * 192, qoh=192)):
        assert _store(**{**same, **other}) == -1 and "in place" in _err(), other
