"""Decode over the blocks of a long context that a cheap score selects.

A page of the K/V pool is cut into blocks of ``block`` tokens.  Beside the pool
lie the bounds of every block: the elementwise minimum and maximum of its keys,
``[NB, BS / block, Hkv, 2, d]`` bf16 (:func:`new_block_bounds`).  A step

* stores its tokens and updates the bounds of the blocks they fall into
  (:func:`update_block_bounds`),
* bounds the logits of each block for the step's queries: ``q . k <= sum_d
  max(q_d min_d, q_d max_d)`` (:func:`block_scores`),
* selects, per sequence and kv head, the first and the last blocks and those of
  the largest scores (:func:`select_blocks`),
* attends to the tokens of the selected blocks
  (:func:`block_sparse_decode_attention`).

:func:`block_sparse_attention` is the layer seam over these, with the arguments
of ``attention()``.  One block costs ``4 d`` bytes a kv head to score and ``4 d
block`` to read, so that of a context of ``n`` tokens about ``n / block +
num_selected block`` rows are read in place of ``n``.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .attention import (AttentionMetadata, DecodeAttentionMetadata, MixedAttentionMetadata, PrefillAttentionMetadata,
                        attention_stored, update_kv_cache)
from ._operands import check_heads, check_output, check_pool, check_table, check_workspace, operand
from .kernels._common import bf16_round, pool_pointers, require_device, stream_handle
from .kernels.mixed_paged_attention import mixed_paged_attention
from .kv_cache_manager import copy_pages
from .rotary import check_tokens, on_device
from .shared_prefix import check_shared

HEAD_DIMS = (64, 128, 256)
MAX_BLOCK = 256  # tokens of a block that block_sparse_decode_attention takes


def _check_block(block: int, page_size: int) -> int:
    if not isinstance(block, int) or block <= 0 or block % 16 or page_size % block:
        raise ValueError(f"block {block} must be a multiple of 16 that divides the page size {page_size}")
    return block


def _check_decode(block: int, head_dim: int) -> None:
    """What the decode over selected blocks takes."""
    if block > MAX_BLOCK:
        raise ValueError(f"blocks of {block} tokens, {MAX_BLOCK} at most")
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head size {head_dim} not supported ({', '.join(map(str, HEAD_DIMS))})")


def _check_picks(num_selected: int, first: int, recent: int) -> None:
    if num_selected <= 0 or first < 0 or recent < 0 or first + recent > num_selected:
        raise ValueError(f"num_selected {num_selected} must be positive and hold the first {first} and the last "
                         f"{recent} blocks")


def _check_bounds(bounds: torch.Tensor, like: Optional[torch.Tensor] = None):
    """Shape and (page, block, head) strides of bounds ``[NB, blocks, Hkv, 2, d]``."""
    stride = operand("bounds", bounds, 5, like)
    if bounds.shape[3] != 2 or stride[3] != bounds.shape[4]:
        raise ValueError(f"bounds must be [NB, BS / block, Hkv, 2, d], contiguous in the last two dimensions, got "
                         f"{tuple(bounds.shape)} with strides {tuple(stride)}")
    return bounds.shape, stride[:3]


def _check_fit(bounds: torch.Tensor, kv_cache: torch.Tensor) -> None:
    nb, per, hkv, _, d = bounds.shape
    if (nb, hkv, d) != (kv_cache.shape[1], *kv_cache.shape[3:]) or per == 0 or kv_cache.shape[2] % per:
        raise ValueError(f"bounds {tuple(bounds.shape)} do not fit a pool {tuple(kv_cache.shape)}")


def new_block_bounds(kv_cache: torch.Tensor, block: int) -> torch.Tensor:
    """Bounds for every block of ``block`` tokens of a layer's pool ``[2, NB,
    BS, Hkv, d]``: bf16 ``[NB, BS / block, Hkv, 2, d]``, zero until
    :func:`update_block_bounds` writes them.  ``block`` is a multiple of 16 that
    divides ``BS``, 256 at most, and ``d`` one of 64, 128 and 256."""
    if kv_cache.dim() != 5 or kv_cache.shape[0] != 2:
        raise ValueError(f"kv_cache must be [2, NB, BS, Hkv, d], got {tuple(kv_cache.shape)}")
    _, nb, bs, hkv, d = kv_cache.shape
    _check_block(block, bs)
    _check_decode(block, d)
    return torch.zeros((nb, bs // block, hkv, 2, d), dtype=torch.bfloat16, device=kv_cache.device)


def update_block_bounds(bounds: torch.Tensor, kv_cache: torch.Tensor, block_tables: torch.Tensor,
                        lengths: torch.Tensor, cu_seqlens_q: Optional[torch.Tensor] = None, *,
                        max_seqlen_q: int = 1) -> torch.Tensor:
    """Writes the bounds of the blocks that hold the last tokens of each
    sequence, in place: the newest one of ``lengths[b]`` tokens, or with
    ``cu_seqlens_q`` ``[B + 1]`` the last ``cu_seqlens_q[b + 1] -
    cu_seqlens_q[b]``, of which ``max_seqlen_q`` is the largest.

    The tokens' keys are in the pool already (``update_kv_cache``).  A block is
    computed from all its keys below the length, so that what a reused page held
    before does not show; other blocks' bounds are left as they were.  Blocks
    whose table entry is not a page of the pool are left out.  Two sequences of
    a call with new tokens in one block race, as their stores do.
    """
    (nb, per, hkv, _, d), bounds_stride = _check_bounds(bounds)
    (_, bs, _, _), cache_stride = check_pool(kv_cache, bounds)
    _check_fit(bounds, kv_cache)
    require_device("lengths", lengths)
    batch = lengths.numel()
    lens = check_tokens("lengths", lengths, batch, bounds)
    table, _keep = check_table(block_tables, batch, bounds)
    cu = None if cu_seqlens_q is None else check_tokens("cu_seqlens_q", cu_seqlens_q, batch + 1, bounds)
    if not 0 <= max_seqlen_q <= 0x7fffffff:
        raise ValueError(f"max_seqlen_q {max_seqlen_q}")
    if batch == 0:
        return bounds
    with on_device(bounds):
        _lib.call("pa_block_bounds", kv_cache.data_ptr(), nb, bs, *cache_stride, *table, lens.data_ptr(),
                  None if cu is None else cu.data_ptr(), batch, max_seqlen_q, hkv, d, bs // per, bounds.data_ptr(),
                  *bounds_stride, stream_handle(bounds))
    return bounds


def copy_block_bounds(bounds: torch.Tensor, src: Sequence[int], dst: Sequence[int]) -> None:
    """``bounds[dst[i]] <- bounds[src[i]]``: what ``copy_blocks`` does for the
    pool when the block manager's copy-on-write moves a sequence to a new page."""
    _check_bounds(bounds)
    copy_pages(bounds[:, :, :, 0], bounds[:, :, :, 1], src, dst)


def block_scores(q: torch.Tensor, bounds: torch.Tensor, block_tables: torch.Tensor, lengths: torch.Tensor, *,
                 page_size: int, scale: float, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """For each sequence, kv head and block the largest bound of its q heads'
    scaled logits, ``scale * max_h sum_d max(q_d min_d, q_d max_d)``: q ``[B, H,
    d]`` -> float32 ``[B, Hkv, blocks of the tables' width]``, ``-inf`` for the
    blocks that start at or past ``lengths[b]``.

    Products are exact and sums 32-bit.  ``scale`` is positive (the attention's).
    Several rows of one sequence (drafted tokens) are rows with the same table
    row and each its own length.
    """
    (nb, per, hkv, _, d), bounds_stride = _check_bounds(bounds)
    q_stride = check_heads(q, hkv, d)
    if bounds.get_device() != q.get_device():
        raise ValueError(f"bounds lives on {bounds.device}, q on {q.device}")
    batch, heads, _ = q.shape
    if per == 0 or page_size <= 0 or page_size % per:
        raise ValueError(f"bounds of {per} blocks a page do not fit pages of {page_size} tokens")
    block = _check_block(page_size // per, page_size)
    table, _keep = check_table(block_tables, batch, q)
    lens = check_tokens("lengths", lengths, batch, q)
    width = table[2] * per
    if out is None:
        out = torch.empty((batch, hkv, width), dtype=torch.float32, device=q.device)
    else:
        require_device("out", out)
        if out.dtype is not torch.float32 or out.shape != (batch, hkv, width) or out.get_device() != q.get_device() \
                or (width > 1 and out.stride(2) != 1):
            raise ValueError(f"out must be float32 [{batch}, {hkv}, {width}] on {q.device}, contiguous in its last "
                             f"dimension, got {out.dtype} {tuple(out.shape)} on {out.device}")
    if batch == 0 or width == 0:
        return out
    with on_device(q):
        _lib.call("pa_block_scores", q.data_ptr(), q_stride[0], q_stride[1], bounds.data_ptr(), nb, page_size,
                  *bounds_stride, *table, lens.data_ptr(), batch, heads, hkv, d, block, float(scale), out.data_ptr(),
                  out.stride(0), out.stride(1), stream_handle(q))
    return out


def select_blocks(scores: torch.Tensor, lengths: torch.Tensor, num_selected: int, *, block: int, first: int = 1,
                  recent: int = 2, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The blocks to attend to, int32 ``[B, Hkv, num_selected]``, ascending:
    the first ``first`` and the last ``recent`` of a sequence's ``ceil(lengths[b]
    / block)`` blocks, and of the others those of the largest ``scores``
    ``[B, Hkv, width]`` (float32; equal scores by the lower index, NaN below all
    numbers).  A sequence of at most ``num_selected`` blocks has all of them,
    then -1.  Scores past a sequence's blocks are not read.
    """
    require_device("scores", scores)
    if scores.dtype is not torch.float32 or scores.dim() != 3 or (scores.shape[2] > 1 and scores.stride(2) != 1):
        raise ValueError(f"scores must be float32 [B, Hkv, blocks], contiguous in the last dimension, got "
                         f"{scores.dtype} {tuple(scores.shape)}")
    batch, hkv, width = scores.shape
    _check_picks(num_selected, first, recent)
    if block <= 0:
        raise ValueError(f"block {block}")
    lens = check_tokens("lengths", lengths, batch, scores)
    shape = (batch, hkv, num_selected)
    if out is None:
        out = torch.empty(shape, dtype=torch.int32, device=scores.device)
    else:
        require_device("out", out)
        if out.dtype is not torch.int32 or out.shape != shape or out.get_device() != scores.get_device() \
                or (num_selected > 1 and out.stride(2) != 1):
            raise ValueError(f"out must be int32 {shape} on {scores.device}, contiguous in its last dimension, got "
                             f"{out.dtype} {tuple(out.shape)} on {out.device}")
    if batch == 0 or hkv == 0:
        return out
    with on_device(scores):
        _lib.call("pa_select_blocks", scores.data_ptr(), scores.stride(0), scores.stride(1), width, lens.data_ptr(),
                  batch, hkv, block, num_selected, first, recent, out.data_ptr(), out.stride(0), out.stride(1),
                  stream_handle(scores))
    return out


def block_sparse_decode_attention(q: torch.Tensor, kv_cache: torch.Tensor, block_tables: torch.Tensor,
                                  lengths: torch.Tensor, selected: torch.Tensor, *, block: int, scale: float,
                                  attn_logits_soft_cap: Optional[float] = None,
                                  workspace: Optional[torch.Tensor] = None,
                                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One new token a sequence over its selected blocks: q ``[B, H, d]``
    against the tokens below ``lengths[b]`` of the blocks ``selected[b, kv
    head]`` (int32 ``[B, Hkv, S]``) -> ``[B, H, d]`` bf16.

    Entries of ``selected`` that are not a block of the sequence (-1) are skipped
    wherever they stand; a block that stands twice counts twice.  A row without
    a token is zero.  Scores, softmax statistics and sums are 32-bit, the
    weights are rounded to bf16 for the matrix cores.  How a selection is split over
    workgroups follows the batch, the heads and ``S``, and with it the last bits.
    Tokens that are not selected are not read; those that are have to be finite.
    """
    (nb, bs, hkv, d), cache_stride = check_pool(kv_cache)
    q_stride = check_heads(q, hkv, d)
    if kv_cache.get_device() != q.get_device():
        raise ValueError(f"kv_cache lives on {kv_cache.device}, q on {q.device}")
    batch, heads, _ = q.shape
    _check_block(block, bs)
    table, _keep = check_table(block_tables, batch, q)
    lens = check_tokens("lengths", lengths, batch, q)
    require_device("selected", selected)
    if selected.dtype is not torch.int32 or selected.dim() != 3 or selected.shape[:2] != (batch, hkv) \
            or selected.shape[2] == 0 or selected.get_device() != q.get_device():
        raise ValueError(f"selected must be int32 [{batch}, {hkv}, S] on {q.device}, got {selected.dtype} "
                         f"{tuple(selected.shape)} on {selected.device}")
    if selected.shape[2] > 1 and selected.stride(2) != 1:
        selected = selected.contiguous()
    num = selected.shape[2]
    out, out_stride = check_output(out, q)
    if batch == 0:
        return out
    need = block_sparse_workspace_bytes(batch, heads, hkv, d, num, block)
    _ws, ws_args = check_workspace(workspace, need, q)
    k, v = pool_pointers(kv_cache)
    cap = 0.0 if attn_logits_soft_cap is None else float(attn_logits_soft_cap)
    with on_device(q):
        _lib.call("pa_block_sparse_decode", q.data_ptr(), q_stride[0], q_stride[1], k, v, nb, bs, *cache_stride,
                  *table, lens.data_ptr(), batch, heads, hkv, d, selected.data_ptr(), selected.stride(0),
                  selected.stride(1), num, block, float(scale), cap, out.data_ptr(), *out_stride, *ws_args,
                  stream_handle(q))
    return out


def block_sparse_workspace_bytes(batch: int, num_heads: int, num_kv_heads: int, head_dim: int, num_selected: int,
                                 block: int) -> int:
    """Bytes of the workspace of a :func:`block_sparse_decode_attention` call (0: none)."""
    return int(_lib.load().pa_block_sparse_decode_workspace_size(batch, num_heads, num_kv_heads, head_dim,
                                                                 num_selected, block))


def _check_step(kv_cache, bounds, q, m, num_selected, first, recent) -> None:
    """The seam's arguments by shapes alone, whatever the step and however wide its tables."""
    if not isinstance(m, (DecodeAttentionMetadata, PrefillAttentionMetadata, MixedAttentionMetadata)):
        raise TypeError(f"metadata of type {type(m).__name__}")
    for name, t, pair, shape in (("kv_cache", kv_cache, 0, "[2, NB, BS, Hkv, d]"),
                                 ("bounds", bounds, 3, "[NB, BS / block, Hkv, 2, d]")):
        if not isinstance(t, torch.Tensor) or t.dim() != 5 or t.shape[pair] != 2:
            raise ValueError(f"{name} must be {shape}")
    _check_fit(bounds, kv_cache)
    bs, d = kv_cache.shape[2], kv_cache.shape[4]
    _check_decode(_check_block(bs // bounds.shape[1], bs), d)
    _check_picks(num_selected, first, recent)
    if getattr(m, "shared", None) is not None:
        check_shared(q, kv_cache, m.shared)
    if isinstance(m, MixedAttentionMetadata) and not 0 <= m.num_decodes <= min(m.block_tables.shape[0], q.shape[0]):
        raise ValueError(f"num_decodes {m.num_decodes} of {m.block_tables.shape[0]} sequences and {q.shape[0]} tokens")


def block_sparse_attention(kv_cache: torch.Tensor, bounds: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                           v: torch.Tensor, metadata: AttentionMetadata, *, num_selected: int, first: int = 1,
                           recent: int = 2) -> Tuple[torch.Tensor, torch.Tensor]:
    """``attention()`` with decode over selected blocks: stores the step's
    tokens and their blocks' bounds, then attends, decode sequences to the
    ``num_selected`` blocks that :func:`select_blocks` picks, prefill sequences
    to their whole context.  Returns ``(kv_cache, out)``.

    Where the block tables are no wider than ``num_selected`` blocks, decode is
    ``attention()``'s.  What wider tables would be refused for is refused here too,
    before anything is stored.
    """
    _check_step(kv_cache, bounds, q, metadata, num_selected, first, recent)
    kv_cache = update_kv_cache(kv_cache, metadata.slot_mapping, k, v)
    m = metadata
    bs, per = kv_cache.shape[2], bounds.shape[1]

    def sparse(rows, tables, lens, out=None):
        scale = 1.0 / bf16_round(float(rows.shape[-1]) ** 0.5)
        scores = block_scores(rows, bounds, tables, lens, page_size=bs, scale=scale)
        chosen = select_blocks(scores, lens, num_selected, block=bs // per, first=first, recent=recent)
        return block_sparse_decode_attention(rows, kv_cache, tables, lens, chosen, block=bs // per, scale=scale,
                                             out=out)

    whole = m.block_tables.shape[1] * per <= num_selected
    if isinstance(m, DecodeAttentionMetadata):
        update_block_bounds(bounds, kv_cache, m.block_tables, m.context_lens)
        return kv_cache, attention_stored(kv_cache, q, m) if whole else sparse(q, m.block_tables, m.context_lens)
    if isinstance(m, PrefillAttentionMetadata):
        lens = m.cu_seqlens_k[1:] - m.cu_seqlens_k[:-1]
        update_block_bounds(bounds, kv_cache, m.block_tables, lens, m.cu_seqlens_q, max_seqlen_q=m.max_seqlen_bucket)
        return kv_cache, attention_stored(kv_cache, q, m)
    update_block_bounds(bounds, kv_cache, m.block_tables, m.kv_lens, m.cu_seqlens_q, max_seqlen_q=m.max_seqlen_q)
    nd = m.num_decodes
    if whole or nd == 0:
        return kv_cache, attention_stored(kv_cache, q, m)
    if nd < m.block_tables.shape[0]:
        pages = (kv_cache[0].permute(2, 0, 1, 3), kv_cache[1].permute(2, 0, 1, 3))
        out = mixed_paged_attention(q, *pages, m.block_tables[nd:], m.cu_seqlens_q[nd:], m.kv_lens[nd:],
                                    m.input_positions, 0, max_seqlen_q=m.max_seqlen_q,
                                    decode_scale=1.0 / bf16_round(float(q.shape[-1]) ** 0.5))
    else:
        out = torch.zeros(q.shape, dtype=torch.bfloat16, device=q.device)
    sparse(q[:nd], m.block_tables[:nd], m.kv_lens[:nd], out=out[:nd])
    return kv_cache, out
