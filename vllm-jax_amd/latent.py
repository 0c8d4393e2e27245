"""Latent attention: one latent vector and one rotated key part a token in the
cache, in place of K and V rows per head.

A token's cache row is ``[c | k_r]``: the normalised latent ``c`` (``R``
elements) and the rotary key part ``k_r`` (``Dr``), shared by all heads.  Head
``h`` attends with ``K[h] = [W_uk[h] c | k_r]`` and ``V[h] = W_uv[h] c``.  The
path mirrors ``attention()``'s: a store (:func:`latent_store`), a decode and a
prefill entry, and the layer seam :func:`latent_attention` over the same
metadata types.  The pool is ``[NB, BS, R + Dr]`` bf16, addressed by the same
slot mappings and block tables as the engine's K/V pool.

Decode runs in the absorbed form: q goes through ``W_uk[h]`` once, scores and
values are taken against the cache rows themselves, and ``W_uv[h]`` maps the
result back, so a cached token costs one row of ``R + Dr`` elements whatever
the number of heads.  Prefill expands K and V of a group of heads at a time
where many new tokens share the cost, and runs absorbed otherwise.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .attention import (AttentionMetadata, DecodeAttentionMetadata, MixedAttentionMetadata, PrefillAttentionMetadata,
                        _checking_slots, _host_bound, check_slot_mapping)
from .kernels._common import require_bf16, require_device, stream_handle
from .rotary import RotaryFrequencies, check_frequencies, check_tokens, on_device

LATENT_DIMS, ROPE_DIMS, HEAD_DIMS = (256, 512), (32, 64), (64, 128)


class LatentWeights:
    """The up projection of a layer, laid out once for the kernels.

    ``w_kv`` is ``[num_heads * (nope_dim + v_dim), R]`` bf16: the rows of
    ``W_uk[h]``, then those of ``W_uv[h]``, head by head.  Kept as it is (a
    contiguous copy if it is not) and with ``W_uk`` transposed, for the
    absorbed form.  A changed ``w_kv`` needs a new object.
    """

    def __init__(self, w_kv: torch.Tensor, *, num_heads: int, nope_dim: int, v_dim: int):
        require_device("w_kv", w_kv)
        if w_kv.dtype != torch.bfloat16:
            raise ValueError(f"w_kv must be bfloat16, got {w_kv.dtype}")
        if num_heads <= 0 or nope_dim not in HEAD_DIMS or v_dim != nope_dim:
            raise ValueError(f"num_heads {num_heads}, nope_dim {nope_dim}, v_dim {v_dim}: nope_dim and v_dim must be "
                             f"equal and one of {HEAD_DIMS}")
        if w_kv.dim() != 2 or w_kv.shape[0] != num_heads * (nope_dim + v_dim) or w_kv.shape[1] not in LATENT_DIMS:
            raise ValueError(f"w_kv must be [{num_heads * (nope_dim + v_dim)}, R] with R one of {LATENT_DIMS}, got "
                             f"{tuple(w_kv.shape)}")
        self.num_heads, self.nope_dim, self.v_dim, self.latent_dim = num_heads, nope_dim, v_dim, w_kv.shape[1]
        self.w_kv = w_kv.detach().contiguous().view(num_heads, nope_dim + v_dim, self.latent_dim)
        if self.w_kv.data_ptr() % 16:
            self.w_kv = self.w_kv.clone()
        self.w_uk_t = self.w_kv[:, :nope_dim].transpose(1, 2).contiguous()  # [H, R, Dn]


def _bf16(name: str, t: torch.Tensor, dims: int, like: Optional[torch.Tensor] = None) -> Tuple[int, ...]:
    """Strides of a bf16 device operand of ``dims`` dimensions, contiguous in
    the last, on ``like``'s device (one call each: this runs on every call)."""
    require_device(name, t)
    stride = t.stride()
    if t.dtype is not torch.bfloat16 or len(stride) != dims or stride[-1] != 1:
        require_bf16(name, t)
        raise ValueError(f"{name} must have {dims} dimensions, got {tuple(t.shape)}")
    if like is not None and t.get_device() != like.get_device():
        raise ValueError(f"{name} lives on {t.device}, the other operands on {like.device}")
    return stride


def _check_cache(latent_cache: torch.Tensor, like: torch.Tensor):
    """(pages, page size, row length), (page, slot) strides of a pool ``[NB, BS, R + Dr]``."""
    stride = _bf16("latent_cache", latent_cache, 3, like)
    return latent_cache.shape, stride[:2]


def latent_store(latent: torch.Tensor, k_rope: torch.Tensor, norm_weight: Optional[torch.Tensor],
                 positions: torch.Tensor, slot_mapping: torch.Tensor, latent_cache: torch.Tensor,
                 freqs: RotaryFrequencies, *, eps: float = 1e-6, interleaved: bool = True,
                 q_rope: Optional[torch.Tensor] = None,
                 q_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The layer step between the down projections and attention, in one
    kernel: ``cache[slot] = [rmsnorm(latent) | rope(k_rope)]`` in place, and
    ``rope(q_rope)``.  Returns ``(latent_cache, q_out)``.

    ``latent`` ``[T, R]`` and ``k_rope`` ``[T, Dr]`` may be slices of one
    projection; ``norm_weight`` ``[R]``, or ``None`` for rows that come
    normalised.  ``q_rope`` ``[T, H, Dr]`` (a slice of q's heads) is rotated
    for every token, into ``q_out`` (``q_rope`` itself, or a tensor that shares
    no memory with it; a new one by default).  Slots outside the pool (padding
    tokens) are skipped.
    """
    latent_stride = _bf16("latent", latent, 2)
    k_stride = _bf16("k_rope", k_rope, 2, latent)
    t_count, r = latent.shape
    (nb, bs, row), cache_stride = _check_cache(latent_cache, latent)
    k_count, dr = k_rope.shape
    if r not in LATENT_DIMS or dr not in ROPE_DIMS or row != r + dr or k_count != t_count:
        raise ValueError(f"latent {tuple(latent.shape)} and k_rope {tuple(k_rope.shape)} do not fit a cache of rows of "
                         f"{row} (R one of {LATENT_DIMS}, Dr one of {ROPE_DIMS})")
    check_frequencies(freqs, latent)
    if freqs.rotary_dim != dr:
        raise ValueError(f"the frequencies are of rotary_dim {freqs.rotary_dim}, k_rope of {dr}")
    norm = None
    if norm_weight is not None:
        _bf16("norm_weight", norm_weight, 1, latent)
        if norm_weight.shape != (r,):
            raise ValueError(f"norm_weight must be [{r}], got {tuple(norm_weight.shape)}")
        norm = norm_weight.data_ptr()
    pos = check_tokens("positions", positions, t_count, latent)
    slots = check_tokens("slot_mapping", slot_mapping, t_count, latent)
    q_args = (None, 0, 0, 0, None, 0, 0)
    if q_rope is not None:
        q_stride = _bf16("q_rope", q_rope, 3, latent)
        heads = q_rope.shape[1]
        if q_rope.shape != (t_count, heads, dr) or heads == 0:
            raise ValueError(f"q_rope must be [{t_count}, H, {dr}], got {tuple(q_rope.shape)}")
        if q_out is None:
            q_out = torch.empty_like(q_rope, memory_format=torch.contiguous_format)
            out_stride = (heads * dr, dr)
        else:
            out_stride = _bf16("q_out", q_out, 3, latent)
            if q_out.shape != q_rope.shape:
                raise ValueError(f"q_out must have shape {tuple(q_rope.shape)}")
        q_args = (q_rope.data_ptr(), q_stride[0], q_stride[1], heads, q_out.data_ptr(), out_stride[0], out_stride[1])
    elif q_out is not None:
        raise ValueError("q_out without q_rope")
    if _checking_slots():
        check_slot_mapping(slots, nb * bs)
    if t_count == 0:
        return latent_cache, q_out
    with on_device(latent):
        _lib.call("pa_latent_store", latent.data_ptr(), latent_stride[0], k_rope.data_ptr(), k_stride[0], norm,
                  float(eps), freqs.inv_freq.data_ptr(), freqs.amplitude, int(bool(interleaved)), pos.data_ptr(),
                  slots.data_ptr(), t_count, r, dr, *q_args, latent_cache.data_ptr(), nb, bs, *cache_stride,
                  stream_handle(latent))
    return latent_cache, q_out


def _check_q(q_nope, q_rope, latent_cache, weights):
    """Checked shapes of an attention call: tokens, (nope, v, rope) sizes, pages, page size, and the leading arguments
    of the C entries (q and cache pointers and strides)."""
    if not isinstance(weights, LatentWeights):
        raise TypeError(f"weights must be LatentWeights, got {type(weights).__name__}")
    heads, dn = weights.num_heads, weights.nope_dim
    qn = _bf16("q_nope", q_nope, 3)
    (nb, bs, row), cache_stride = _check_cache(latent_cache, q_nope)
    dr = row - weights.latent_dim
    if dr not in ROPE_DIMS:
        raise ValueError(f"latent_cache rows of {row} do not fit latent_dim {weights.latent_dim} (rope_dim must be one "
                         f"of {ROPE_DIMS})")
    qr = _bf16("q_rope", q_rope, 3, q_nope)
    tokens = q_nope.shape[0]
    for name, t, d in (("q_nope", q_nope, dn), ("q_rope", q_rope, dr)):
        if t.shape != (tokens, heads, d):
            raise ValueError(f"{name} must be [{tokens}, {heads}, {d}], got {tuple(t.shape)}")
    if weights.w_kv.get_device() != q_nope.get_device():
        raise ValueError(f"the weights live on {weights.w_kv.device}, q on {q_nope.device}")
    return tokens, dr, nb, bs, (q_nope.data_ptr(), qn[0], qn[1], q_rope.data_ptr(), qr[0], qr[1],
                                latent_cache.data_ptr(), nb, bs, *cache_stride)


def _check_table(block_tables: torch.Tensor, batch: int, like: torch.Tensor):
    """(pointer, row stride, pages) of int32 ``[batch, pages]`` block tables, and the tensor they are in."""
    require_device("block_tables", block_tables)
    if block_tables.dtype is not torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] != batch:
        raise ValueError(f"block_tables must be int32 [{batch}, pages], got {block_tables.dtype} "
                         f"{tuple(block_tables.shape)}")
    if block_tables.get_device() != like.get_device():
        raise ValueError(f"block_tables lives on {block_tables.device}, q on {like.device}")
    stride = block_tables.stride()
    if stride[1] != 1 and block_tables.shape[1] > 1:
        block_tables = block_tables.contiguous()
        stride = block_tables.stride()
    return (block_tables.data_ptr(), stride[0], block_tables.shape[1]), block_tables


def _output(out, shape, like):
    """The output tensor and its (token, head) strides."""
    if out is None:
        return torch.empty(shape, dtype=torch.bfloat16, device=like.device), (shape[1] * shape[2], shape[2])
    stride = _bf16("out", out, 3, like)
    if out.shape != shape:
        raise ValueError(f"out must have shape {shape}, got {tuple(out.shape)}")
    return out, stride[:2]


def _workspace(workspace, need, like):
    """The caller's workspace where it is large enough, else a new one; and its bytes."""
    if workspace is not None:
        require_device("workspace", workspace)
        if workspace.get_device() != like.get_device():
            raise ValueError(f"workspace lives on {workspace.device}, q on {like.device}")
        given = workspace.numel() * workspace.element_size()
        if workspace.is_contiguous() and given >= need and workspace.data_ptr() % 16 == 0:
            return workspace, given
    need = max(need, 1)
    return torch.empty(need, dtype=torch.uint8, device=like.device), need


def latent_decode_attention(q_nope: torch.Tensor, q_rope: torch.Tensor, latent_cache: torch.Tensor,
                            weights: LatentWeights, block_tables: torch.Tensor, lengths: torch.Tensor, *,
                            scale: float, workspace: Optional[torch.Tensor] = None,
                            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One new token a sequence over the paged latent cache (absorbed form):
    q_nope ``[B, H, Dn]`` and the rotated q_rope ``[B, H, Dr]`` against the
    first ``lengths[b]`` rows of sequence ``b`` -> ``[B, H, Dv]`` bf16.

    ``scale`` multiplies the scores (``(Dn + Dr) ** -0.5`` for an unscaled
    model).  A length of zero gives a zero row; lengths past the block table's
    span are clamped to it.  The absorbed q, the latent-wide result and the
    split's partials go through ``workspace`` (``latent_decode_workspace_bytes``;
    made here if it is not given or too small).  Scores, softmax statistics and
    sums are float32; the absorbed q, the softmax weights and the latent-wide
    result are rounded to bf16 for the matrix cores.  How a sequence is cut
    follows the batch's lengths and the table's width, and with it a row's last
    bits.  Cached rows below a length have to be finite.
    """
    batch, dr, nb, bs, rows = _check_q(q_nope, q_rope, latent_cache, weights)
    table, _keep = _check_table(block_tables, batch, q_nope)
    lens = check_tokens("lengths", lengths, batch, q_nope)
    w = weights
    out, out_stride = _output(out, (batch, w.num_heads, w.v_dim), q_nope)
    if batch == 0:
        return out
    need = latent_decode_workspace_bytes(batch, w, table[2], bs)
    ws, ws_bytes = _workspace(workspace, need, q_nope)
    with on_device(q_nope):
        _lib.call("pa_latent_decode", *rows, *table, lens.data_ptr(), batch, w.num_heads, w.latent_dim, dr, w.nope_dim,
                  w.v_dim, w.w_uk_t.data_ptr(), w.w_kv.data_ptr(), float(scale), out.data_ptr(), *out_stride,
                  ws.data_ptr(), ws_bytes, stream_handle(q_nope))
    return out


def latent_decode_workspace_bytes(batch: int, weights: LatentWeights, pages_per_seq: int, page_size: int) -> int:
    """Bytes of the workspace of a :func:`latent_decode_attention` call."""
    return int(_lib.load().pa_latent_decode_workspace_size(batch, weights.num_heads, weights.latent_dim,
                                                           pages_per_seq, page_size))


def latent_prefill_attention(q_nope: torch.Tensor, q_rope: torch.Tensor, latent_cache: torch.Tensor,
                             weights: LatentWeights, block_tables: torch.Tensor, cu_seqlens_q: torch.Tensor,
                             cu_seqlens_k: Optional[torch.Tensor] = None, *, max_seqlen_q: int, scale: float,
                             kv_lens: Optional[torch.Tensor] = None, max_seqlen_k: Optional[int] = None,
                             total_kv_tokens: Optional[int] = None, workspace: Optional[torch.Tensor] = None,
                             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Ragged causal attention of new tokens over the paged latent cache:
    q_nope ``[T, H, Dn]`` and the rotated q_rope ``[T, H, Dr]``, sequence ``b``
    being rows ``cu_seqlens_q[b] .. cu_seqlens_q[b + 1]`` -> ``[T, H, Dv]`` bf16.

    The kv lengths ``lk`` (cached rows, the new ones included; already stored) come as
    ``cu_seqlens_k`` (differences), as ``kv_lens`` ``[B]``, or, with neither,
    equal the new tokens'; row ``i`` of a sequence sees its first ``lk - lq +
    i + 1`` rows, and is zero if that is none.  Cached rows below a length
    have to be finite (those that a row does not see, too).  At most ``max_seqlen_q`` rows
    of a sequence are computed.  Rows outside the sequences are zero in a new output and
    left as they were in a given ``out``.

    ``total_kv_tokens`` bounds the sum of the kv lengths on the host (it has to
    hold: rows past it may be left out); without it ``max_seqlen_k``, or the block tables'
    span, times the sequences.  Tight bounds keep the workspace
    (``latent_prefill_workspace_bytes``) small and choose the form:
    expanded K and V rows (bf16) for a group of heads at a time, or the absorbed
    form where few new tokens stand behind long contexts (or where one head's
    rows would pass 8 GiB and the absorbed form's workspace is smaller).
    """
    tokens, dr, nb, bs, rows = _check_q(q_nope, q_rope, latent_cache, weights)
    w = weights
    require_device("cu_seqlens_q", cu_seqlens_q)
    if cu_seqlens_q.dim() != 1 or cu_seqlens_q.numel() < 1:
        raise ValueError(f"cu_seqlens_q must be int32 [B + 1], got {tuple(cu_seqlens_q.shape)}")
    batch = cu_seqlens_q.numel() - 1
    table, _keep = _check_table(block_tables, batch, q_nope)
    cu_q = check_tokens("cu_seqlens_q", cu_seqlens_q, batch + 1, q_nope)
    if cu_seqlens_k is not None and kv_lens is not None:
        raise ValueError("cu_seqlens_k and kv_lens are given both")
    cu_k = lens = None
    if kv_lens is not None:
        lens = check_tokens("kv_lens", kv_lens, batch, q_nope)
    elif cu_seqlens_k is not None:
        cu_k = check_tokens("cu_seqlens_k", cu_seqlens_k, batch + 1, q_nope)
    else:
        cu_k = cu_q
    if max_seqlen_q < 0 or max_seqlen_q > 0x7fffffff:
        raise ValueError(f"max_seqlen_q {max_seqlen_q}")
    total = _total_kv(batch, tokens, table[2] * bs, max_seqlen_k, total_kv_tokens, cu_k is cu_q)
    zero_rest = out is None
    out, out_stride = _output(out, (tokens, w.num_heads, w.v_dim), q_nope)
    if tokens == 0:
        return out
    need = latent_prefill_workspace_bytes(batch, tokens, max_seqlen_q, total, w, dr, table[2], bs) if batch else 0
    ws, ws_bytes = _workspace(workspace, need, q_nope)
    with on_device(q_nope):
        _lib.call("pa_latent_prefill", *rows, *table, cu_q.data_ptr(), None if cu_k is None else cu_k.data_ptr(),
                  None if lens is None else lens.data_ptr(), batch, tokens, max_seqlen_q, total, w.num_heads,
                  w.latent_dim, dr, w.nope_dim, w.v_dim, w.w_uk_t.data_ptr(), w.w_kv.data_ptr(), float(scale),
                  int(zero_rest), out.data_ptr(), *out_stride, ws.data_ptr(), ws_bytes, stream_handle(q_nope))
    return out


def _total_kv(batch, tokens, span, max_seqlen_k, total_kv_tokens, fresh) -> int:
    """Bound of the kv lengths' sum, from what the host knows; where only widths are known, at most the C entries'
    largest number."""
    if total_kv_tokens is not None:
        total = int(total_kv_tokens)
    elif fresh:
        total = tokens
    else:
        total = min(batch * min(span, span if max_seqlen_k is None else int(max_seqlen_k)), 0x7fffffff)
    if total < 0 or total > 0x7fffffff:
        raise ValueError(f"the kv lengths' sum is bounded by {total} (0 to 2^31 - 1 can be given)")
    return total


def latent_prefill_workspace_bytes(batch: int, num_tokens: int, max_seqlen_q: int, total_kv_tokens: int,
                                   weights: LatentWeights, rope_dim: int, pages_per_seq: int, page_size: int) -> int:
    """Bytes of the workspace of a :func:`latent_prefill_attention` call."""
    return int(_lib.load().pa_latent_prefill_workspace_size(batch, num_tokens, max_seqlen_q, total_kv_tokens,
                                                            pages_per_seq, page_size, weights.num_heads,
                                                            weights.latent_dim, rope_dim, weights.nope_dim))


def latent_attention(latent_cache: torch.Tensor, q: torch.Tensor, latent: torch.Tensor, k_rope: torch.Tensor,
                     norm_weight: Optional[torch.Tensor], weights: LatentWeights, freqs: RotaryFrequencies,
                     metadata: AttentionMetadata, *, scale: float, eps: float = 1e-6,
                     interleaved: bool = True,
                     total_kv_tokens: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """A layer's whole step between its projections, beside ``attention()``:
    the latent store with both rotations (:func:`latent_store`), then decode,
    prefill or a mixed step by ``metadata``, whose three types and fields are
    ``attention()``'s.  q is ``[T, H, Dn + Dr]`` (not rotated; not changed).
    Returns ``(latent_cache, out [T, H, Dv])``; rows outside the sequences are
    zero.

    ``total_kv_tokens`` and the metadata's ``max_seqlen_k`` bound the kv lengths
    of the step's prefill sequences, their sum and each, and have to hold (see
    :func:`latent_prefill_attention`); a step that gives neither is planned for
    the block tables' whole width.
    """
    if not isinstance(weights, LatentWeights):
        raise TypeError(f"weights must be LatentWeights, got {type(weights).__name__}")
    dn = weights.nope_dim
    if q.dim() != 3 or q.shape[2] <= dn:
        raise ValueError(f"q must be [T, {weights.num_heads}, {dn} + rope_dim], got {tuple(q.shape)}")
    _, q_rope = latent_store(latent, k_rope, norm_weight, metadata.input_positions, metadata.slot_mapping,
                             latent_cache, freqs, eps=eps, interleaved=interleaved, q_rope=q[..., dn:])
    q_nope = q[..., :dn]
    m = metadata
    if isinstance(m, DecodeAttentionMetadata):
        return latent_cache, latent_decode_attention(q_nope, q_rope, latent_cache, weights, m.block_tables,
                                                     m.context_lens, scale=scale)
    if isinstance(m, PrefillAttentionMetadata):
        out = latent_prefill_attention(q_nope, q_rope, latent_cache, weights, m.block_tables, m.cu_seqlens_q,
                                       None if m.cu_seqlens_k is m.cu_seqlens_q else m.cu_seqlens_k,
                                       max_seqlen_q=m.max_seqlen_bucket, scale=scale,
                                       max_seqlen_k=_host_bound(m.max_seqlen_k) or None,
                                       total_kv_tokens=total_kv_tokens)
        return latent_cache, out
    if not isinstance(m, MixedAttentionMetadata):
        raise TypeError(f"metadata of type {type(m).__name__}")
    nd = m.num_decodes
    if not 0 <= nd <= m.block_tables.shape[0] or nd > q.shape[0]:
        raise ValueError(f"num_decodes {nd} of {m.block_tables.shape[0]} sequences and {q.shape[0]} tokens")
    if nd == m.block_tables.shape[0]:
        out = torch.zeros((q.shape[0], weights.num_heads, weights.v_dim), dtype=torch.bfloat16, device=q.device)
    else:
        out = latent_prefill_attention(q_nope, q_rope, latent_cache, weights, m.block_tables[nd:],
                                       m.cu_seqlens_q[nd:], kv_lens=m.kv_lens[nd:], max_seqlen_q=m.max_seqlen_q,
                                       max_seqlen_k=_host_bound(m.max_seqlen_k) or None,
                                       total_kv_tokens=total_kv_tokens, scale=scale)
    if nd:
        latent_decode_attention(q_nope[:nd], q_rope[:nd], latent_cache, weights, m.block_tables[:nd], m.kv_lens[:nd],
                                scale=scale, out=out[:nd])
    return latent_cache, out
