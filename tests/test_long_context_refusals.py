"""What the entries over long contexts refuse, they refuse at every size and before they change anything (no device)."""
from __future__ import annotations

import contextlib
import importlib

import pytest
import torch

from conftest import PKG

ATTENTION = importlib.import_module(PKG.__name__ + ".attention")


def _bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.fixture
def host_tensors(monkeypatch):
    """The entries' checks take host tensors; nothing is launched."""
    for module in ("shared_prefix", "_operands", "rotary"):
        monkeypatch.setattr(importlib.import_module(f"{PKG.__name__}.{module}"), "require_device", lambda *a: None)
    monkeypatch.setattr(PKG.shared_prefix, "on_device", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(PKG.shared_prefix, "stream_handle", lambda t: None)


NOT_SHARED = [  # kv heads, q heads, head size, what the message names
    (2, 8, 64, "head size"),
    (2, 8, 256, "head size"),
    (2, 514, 128, "256 q heads"),
]


@pytest.mark.parametrize("pages", [1, 1 << 20])
@pytest.mark.parametrize("hkv,heads,dim,message", NOT_SHARED)
def test_shared_prefixes_of_other_heads_at_every_width(hkv, heads, dim, message, pages, host_tensors):
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
              (_bf16(2, 1, 16, 2, 128), 8, PKG.SharedPrefixes([0, 2], [64]), TypeError, "cu_groups"),
              (_bf16(2, 1, 16, 2, 128), 8, PKG.SharedPrefixes(_i32(3), _i32(1)), ValueError, "cu_groups"),
              (_bf16(2, 1, 16, 2, 128), 8, PKG.SharedPrefixes(_i32(2), _i32(1, 1)), ValueError, "shared_lens"),
              (_bf16(3, 1, 16, 2, 128), 8, groups, ValueError, "the pool")]
    for cache, heads, shared, error, message in cases:
        hkv, dim = cache.shape[3:]
        q, k, w = _bf16(2, heads, dim), _bf16(2, hkv, dim), _bf16(dim)
        with pytest.raises(error, match=message):
            PKG.attention(cache, q, k, k, meta(shared))
        with pytest.raises(error, match=message):
            PKG.qwen3_attention_core(cache, q, k, k, w, w, meta(shared), eps=1e-6, rope_theta=1e6)
    assert not stored


# ---------------------------------------------------------------------------
# selected blocks
# ---------------------------------------------------------------------------
SPARSE = importlib.import_module(PKG.__name__ + ".block_sparse")


def _steps(batch, pages, shared=None):
    """A decode, a prefill and a mixed step of ``batch`` sequences by one token."""
    row, table, cu = _i32(batch), _i32(batch, pages), _i32(batch + 1)
    return [PKG.SharedDecodeAttentionMetadata(row, row, table, row, shared=shared),
            PKG.SharedPrefillAttentionMetadata(row, row, table, cu, cu, None, None, 1, shared=shared),
            PKG.MixedAttentionMetadata(row, row, table, cu, row, batch, 1)]


@pytest.mark.parametrize("pages", [1, 300])
def test_sparse_attention_refuses_before_the_store(pages, monkeypatch):
    """Tables narrower than the selection (whole contexts, by attention()) and wider ones."""
    stored = []
    monkeypatch.setattr(SPARSE, "update_kv_cache", lambda cache, *a: stored.append(1) or cache)
    monkeypatch.setattr(SPARSE, "update_block_bounds", lambda *a, **k: stored.append(1))
    cache = _bf16(2, 3, 512, 2, 128)
    fine = dict(cache=cache, bounds=_bf16(3, 4, 2, 2, 128), num=8)

    def call(m, cache, bounds, num, **kw):
        d = cache.shape[-1]
        PKG.block_sparse_attention(cache, bounds, _bf16(2, 8, d), _bf16(2, 2, d), _bf16(2, 2, d), m, num_selected=num, **kw)

    cases = [(dict(bounds=_bf16(3, 1, 2, 2, 128)), "blocks of 512"),
             (dict(cache=_bf16(2, 3, 512, 2, 96), bounds=_bf16(3, 4, 2, 2, 96)), "head size 96"),
             (dict(bounds=_bf16(3, 64, 2, 2, 128)), "multiple of 16"),
             (dict(bounds=_bf16(3, 3, 2, 2, 128)), "do not fit"),
             (dict(bounds=_bf16(3, 0, 2, 2, 128)), "do not fit"),
             (dict(bounds=_bf16(2, 4, 2, 2, 128)), "do not fit"),
             (dict(bounds=_bf16(3, 4, 2, 128)), "bounds must be"),
             (dict(cache=cache[0]), "kv_cache must be"),
             (dict(num=0), "num_selected 0"),
             (dict(num=2), "num_selected 2"),
             (dict(num=4, first=3, recent=2), "the first 3")]
    for m in _steps(2, pages):
        for over, message in cases:
            with pytest.raises(ValueError, match=message):
                call(m, **{**fine, **over})
    groups = PKG.SharedPrefixes.of([0, 2], [64], "cpu")
    for m in _steps(2, pages, groups)[:2]:
        with pytest.raises(ValueError, match="head size"):
            call(m, _bf16(2, 3, 512, 2, 64), _bf16(3, 4, 2, 2, 64), 8)
    for decodes in (-1, 3):
        m = _steps(2, pages)[2]
        m.num_decodes = decodes
        with pytest.raises(ValueError, match=f"num_decodes {decodes}"):
            call(m, **fine)
    m = _steps(3, pages)[2]  # three decode sequences, two tokens
    with pytest.raises(ValueError, match="num_decodes 3"):
        call(m, **fine)
    with pytest.raises(TypeError, match="metadata"):
        call(None, **fine)
    assert not stored


def test_bounds_that_no_decode_takes():
    for block in (512, 1024):
        with pytest.raises(ValueError, match=f"blocks of {block}"):
            PKG.new_block_bounds(_bf16(2, 3, 1024, 2, 128), block)
    with pytest.raises(ValueError, match="head size 96"):
        PKG.new_block_bounds(_bf16(2, 3, 64, 2, 96), 16)
    assert PKG.new_block_bounds(_bf16(2, 3, 512, 2, 256), 256).shape == (3, 2, 2, 2, 256)


# ---------------------------------------------------------------------------
# workspaces
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("pays", [False, True])
def test_workspaces_that_do_not_fit_are_replaced(pays, host_tensors, monkeypatch):
    """The plain decode writes through the workspace's address: on either route only one that is contiguous, aligned and
    large enough gets there."""
    used = []
    sp = PKG.shared_prefix
    monkeypatch.setattr(sp, "decode_checked", lambda *a: used.append((a[8].data_ptr(), a[8].numel() * a[8].element_size(),
                                                                      a[8].is_contiguous())))
    monkeypatch.setattr(sp._lib, "call", lambda name, *a: used.append((a[-3], a[-2], True)))
    monkeypatch.setattr(sp, "shared_prefix_pays", lambda *a: pays)
    q, cache, table = _bf16(2, 8, 128), _bf16(2, 4, 256, 2, 128), _i32(2, 64)
    prefixes = PKG.SharedPrefixes.of([0, 2], [64], "cpu")
    need = PKG.shared_prefix_workspace_bytes(2, 1, 2, 8, 2, 64, 256) if pays else \
        importlib.import_module(PKG.__name__ + ".kernels.decode_paged_attention").decode_workspace_bytes(2, 8, 128, 64, 256)
    assert need > 512
    room = torch.empty(4 * need + 1024, dtype=torch.uint8)
    at = -room.data_ptr() % 256
    fits = room[at:at + need]
    unfit = [room[at + 16:at + 16 + need], room[at:at + need - 1], room[at:at + 2 * need:2], room[:0]]
    for ws in (fits, room[at:].view(torch.int8)):
        PKG.shared_prefix_attention(q, cache, table, _i32(2), prefixes, scale=1.0, workspace=ws)
        assert used.pop()[0] == ws.data_ptr()
    # (what a new one's address is on the host is the host allocator's matter)
    for ws in unfit:
        PKG.shared_prefix_attention(q, cache, table, _i32(2), prefixes, scale=1.0, workspace=ws)
        ptr, given, contiguous = used.pop()
        assert given >= need and contiguous and not room.data_ptr() <= ptr < room.data_ptr() + room.numel()


@pytest.mark.gpu
def test_workspaces_off_the_device(dev):
    """Refused on both routes, by name."""
    groups = PKG.SharedPrefixes.of([0, 2], [64], dev)
    q, cache = _bf16(2, 8, 128).to(dev), _bf16(2, 1, 16, 2, 128).to(dev)
    for pages in (4, 1 << 20):
        table = _i32(2, 1).to(dev).expand(2, pages)
        assert PKG.shared_prefix_pays(2, 1, 2, 16 * pages) == (pages > 4)
        with pytest.raises(ValueError, match="workspace must live on a HIP device"):
            PKG.shared_prefix_attention(q, cache, table, _i32(2).to(dev), groups, scale=1.0,
                                        workspace=torch.empty(1 << 20, dtype=torch.uint8))


# ---------------------------------------------------------------------------
# steps that share nothing
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("cu_groups", [[0], [0, 1, 2], [0, 0, 2, 2]])
def test_attention_without_a_shared_token_is_the_plain_one(cu_groups, host_tensors, monkeypatch):
    """As many groups as sequences (what the block manager returns for unrelated requests), or none: the plain kernels,
    which put no partials aside; a group of two takes the shared ones where they pay."""
    took = []
    monkeypatch.setattr(ATTENTION, "prefill_pool", lambda *a, **k: took.append("prefill"))
    monkeypatch.setattr(ATTENTION, "decode_pool", lambda *a, **k: took.append("decode"))
    monkeypatch.setattr(ATTENTION, "shared_prefix_attention", lambda *a, **k: took.append("shared"))
    q, cache = _bf16(2, 8, 128), _bf16(2, 4, 16, 2, 128)
    groups = PKG.SharedPrefixes.of(cu_groups, [16] * (len(cu_groups) - 1), "cpu")
    pair = PKG.SharedPrefixes.of([0, 2], [16], "cpu")
    decode, prefill = _steps(2, 4, groups)[:2]
    PKG.attention_stored(cache, q, decode)
    PKG.attention_stored(cache, q, prefill)
    for m in _steps(2, 4, pair)[:2]:
        PKG.attention_stored(cache, q, m)
    assert took == ["decode", "prefill", "shared", "prefill"]  # (the entry itself chooses for decode)
    # groups that do not fit together are refused there too
    for m in (decode, prefill):
        m.shared = PKG.SharedPrefixes(_i32(3), _i32(3))
        with pytest.raises(ValueError, match="cu_groups"):
            PKG.attention_stored(cache, q, m)
    assert len(took) == 4


@pytest.mark.parametrize("qwen", [False, True])
def test_prefill_steps_with_groups_take_the_faster_kernels(qwen, host_tensors, monkeypatch):
    """Few rows a sequence behind wide tables: the shared kernels; many rows, whose partials would take time and room, or
    narrow tables: the plain prefill."""
    took = []
    monkeypatch.setattr(ATTENTION, "prefill_pool", lambda *a, **k: took.append("prefill"))
    monkeypatch.setattr(ATTENTION, "shared_prefix_attention", lambda *a, **k: took.append("shared"))
    monkeypatch.setattr(ATTENTION, "update_kv_cache", lambda cache, *a: cache)
    monkeypatch.setattr(ATTENTION, "qk_norm_rope_store", lambda q, *a, **k: (q, cache))
    cache = _bf16(2, 1, 256, 8, 128)
    groups = PKG.SharedPrefixes.of([0, 16], [4096], "cpu")
    for heads, pages, tokens, name in ((32, 17, 16, "shared"), (32, 17, 8191, "shared"), (32, 17, 8192, "prefill"),
                                       (32, 15, 16, "prefill"), (64, 17, 4095, "shared"), (64, 17, 4096, "prefill"),
                                       (8, 17, 32767, "shared"), (8, 17, 32768, "prefill"), (32, 4096, 8192, "prefill")):
        q, k, w = _bf16(1, heads, 128).expand(tokens, heads, 128), _bf16(1, 8, 128).expand(tokens, 8, 128), _bf16(128)
        m = PKG.SharedPrefillAttentionMetadata(_i32(tokens), _i32(tokens), _i32(16, 1).expand(16, pages), _i32(17),
                                               _i32(17), None, None, tokens, shared=groups)
        if qwen:
            PKG.qwen3_attention_core(cache, q, k, k, w, w, m, eps=1e-6, rope_theta=1e6)
        else:
            PKG.attention(cache, q, k, k, m)
        assert took.pop() == name and not took, (heads, pages, tokens)


@pytest.mark.gpu
def test_a_step_of_unrelated_requests(dev):
    """The bits of the same step without groups."""
    gen = torch.Generator().manual_seed(21)
    rand = lambda *s: torch.randn(s, generator=gen).to(torch.bfloat16).to(dev)  # noqa: E731
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    cache, table = rand(2, 12, 64, 2, 128), i32([[3, 1, 7], [0, 9, 2], [11, 4, 5]])
    lens, new = [150, 64, 190], [70, 1, 33]
    q, k, v = rand(104, 8, 128), rand(104, 2, 128), rand(104, 2, 128)
    pos = [t for n, c in zip(lens, new) for t in range(n - c, n)]
    slots = [int(table[b, t // 64]) * 64 + t % 64 for b, (n, c) in enumerate(zip(lens, new)) for t in range(n - c, n)]
    outs = []
    for shared in (None, PKG.SharedPrefixes.of([0, 1, 2, 3], [0, 0, 0], dev), PKG.SharedPrefixes.of([0], [], dev)):
        meta = PKG.SharedPrefillAttentionMetadata(i32(pos), i32(slots), table, i32([0, 70, 71, 104]), i32([0, 150, 214, 404]),
                                                  None, None, 70, shared=shared)
        outs.append(PKG.attention(cache.clone(), q, k, v, meta))
    for pool, out in outs[1:]:
        assert torch.equal(pool, outs[0][0]) and torch.equal(out, outs[0][1])


# ---------------------------------------------------------------------------
# devices
# ---------------------------------------------------------------------------
def test_page_copies_launch_on_the_pools_device(host_tensors, monkeypatch):
    """Bounds and pools on another device than the current one: the launch is made with theirs current."""
    events = []
    common = importlib.import_module(PKG.__name__ + ".kernels._common")

    @contextlib.contextmanager
    def on_device(t):
        events.append("enter")
        yield
        events.append("leave")

    monkeypatch.setattr(importlib.import_module(PKG.__name__ + ".rotary"), "on_device", on_device)
    monkeypatch.setattr(common, "require_device", lambda *a: None)
    monkeypatch.setattr(common, "stream_handle", lambda t: None)
    monkeypatch.setattr(PKG.kv_cache_manager._lib, "call", lambda name, *a: events.append(name))
    PKG.copy_block_bounds(_bf16(3, 4, 2, 2, 128), [0], [2])
    PKG.copy_blocks(_bf16(2, 3, 16, 2, 128), [0], [2])
    assert events == ["enter", "pa_copy_blocks", "leave"] * 2
    PKG.copy_block_bounds(_bf16(3, 4, 2, 2, 128), [], [])
    assert len(events) == 6
