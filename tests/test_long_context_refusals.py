"""What the entries over long contexts refuse, they refuse at every size and before they change anything (no device)."""
from __future__ import annotations

import importlib

import pytest
import torch

from conftest import PKG

ATTENTION = importlib.import_module(PKG.__name__ + ".attention")


def _bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


NOT_SHARED = [  # kv heads, q heads, head size, what the message names
    (2, 8, 64, "head size"),
    (2, 8, 256, "head size"),
    (2, 514, 128, "256 q heads"),
]


@pytest.mark.parametrize("pages", [1, 1 << 20])
@pytest.mark.parametrize("hkv,heads,dim,message", NOT_SHARED)
def test_shared_prefixes_of_other_heads_at_every_width(hkv, heads, dim, message, pages):
    """Tables narrow enough for the plain decode, and wide ones."""
    prefixes = PKG.SharedPrefixes.of([0, 2], [64], "cpu")
    q, cache, table = _bf16(2, heads, dim), _bf16(2, 1, 16, hkv, dim), _i32(1, 1).expand(2, pages)
    assert PKG.shared_prefix_pays(2, 1, hkv, 16 * pages) == (pages > 1)
    for cu in (None, _i32(3)):
        with pytest.raises(ValueError, match=message):
            PKG.shared_prefix_attention(q, cache, table, _i32(2), prefixes, cu, scale=1.0)


@pytest.mark.parametrize("prefill", [False, True])
def test_attention_refuses_groups_before_the_store(prefill, monkeypatch):
    stored = []
    monkeypatch.setattr(ATTENTION, "update_kv_cache", lambda cache, *a: stored.append(1) or cache)
    monkeypatch.setattr(ATTENTION, "qk_norm_rope_store", lambda q, *a, **k: stored.append(1) or (q, a[-1]))

    def meta(shared):
        if prefill:
            return PKG.SharedPrefillAttentionMetadata(_i32(2), _i32(2), _i32(2, 1), _i32(3), _i32(3), None, None, 1,
                                                      shared=shared)
        return PKG.SharedDecodeAttentionMetadata(_i32(2), _i32(2), _i32(2, 1), _i32(2), shared=shared)

    groups = PKG.SharedPrefixes.of([0, 2], [64], "cpu")
    cases = [(_bf16(2, 1, 16, hkv, dim), heads, groups, ValueError, message) for hkv, heads, dim, message in NOT_SHARED]
    cases += [(_bf16(2, 1, 16, 2, 128), 8, ([0, 2], [64]), TypeError, "SharedPrefixes"),
              (_bf16(3, 1, 16, 2, 128), 8, groups, ValueError, "the pool")]
    for cache, heads, shared, error, message in cases:
        hkv, dim = cache.shape[3:]
        q, k, w = _bf16(2, heads, dim), _bf16(2, hkv, dim), _bf16(dim)
        with pytest.raises(error, match=message):
            PKG.attention(cache, q, k, k, meta(shared))
        with pytest.raises(error, match=message):
            PKG.qwen3_attention_core(cache, q, k, k, w, w, meta(shared), eps=1e-6, rope_theta=1e6)
    assert not stored
