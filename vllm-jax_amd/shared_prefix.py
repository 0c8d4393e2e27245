"""Attention of a batch whose sequences share prefixes.

Prefix caching lets sequences share the pages of a common prefix, and forks
those of their parent, but decode and prefill still read a shared page once for
every sequence.  :func:`shared_prefix_attention` takes the batch in groups of
sequences that share their first pages: all rows of a group attend to the
shared tokens together, as the rows of one matrix product over pages that are
read once, each sequence to its own tokens behind them, and the two are added
by their log-sum-exp.  The result is that of ``decode_paged_attention`` and
``prefill_paged_attention`` up to rounding.

The block manager finds the groups of a step (``KVCacheManager.shared_prefixes``);
a step's metadata carries them to ``attention()`` (``SharedDecodeAttentionMetadata``,
``SharedPrefillAttentionMetadata``).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import _lib
from ._operands import check_heads, check_output, check_pool, check_table, check_workspace
from .kernels._common import pool_pointers, require_device, stream_handle
from .kernels.decode_paged_attention import decode_checked, decode_workspace_bytes
from .rotary import check_tokens, on_device


HEAD_DIM = 128   # the head size of the kernels of shared prefixes
MAX_GROUP = 256  # and the most q heads a kv head


@dataclass
class SharedPrefixes:
    """Groups of a batch's sequences: group ``g`` is sequences ``cu_groups[g] ..
    cu_groups[g + 1] - 1``, and their first ``shared_lens[g]`` tokens lie in the
    same pages.  int32 ``[groups + 1]`` and ``[groups]`` on the device."""
    cu_groups: torch.Tensor
    shared_lens: torch.Tensor

    @classmethod
    def of(cls, cu_groups: Sequence[int], shared_lens: Sequence[int], device) -> "SharedPrefixes":
        """From the numbers that ``KVCacheManager.shared_prefixes`` returns."""
        return cls(torch.as_tensor(list(cu_groups), dtype=torch.int32, device=device),
                   torch.as_tensor(list(shared_lens), dtype=torch.int32, device=device))


def shared_prefix_pays(batch: int, num_groups: int, num_kv_heads: int, span: int, rows: int = 1) -> bool:
    """Whether a step of ``batch`` sequences in ``num_groups`` groups, over block
    tables of ``span`` tokens, is cut at the shared prefixes; else the plain kernels
    read shared pages again and again, most of them from the caches.  ``rows``: the new
    tokens of a sequence, on average, times the q heads of a kv head.

    It takes more sequences than groups, and tables of 256 MB of K and V in all.
    Whole calls, 32 / 8 heads, one group: 16 sequences of 4096 shared tokens (289 MB)
    36.7 us by the plain decode, 29.7 so; 64 of 1024 (352 MB) 52.3 and 30.6; 4 of
    16384 (273 MB) 39.2 and 35.4; 2 of 32768 (271 MB) 50.4 and 49.3; 16 of 2048
    (155 MB) 25.7 and 28.7.

    Of several new tokens 400 ragged steps were measured (16 to 64 q heads, 4 to 64
    sequences, 512 to 131 072 shared tokens).  With narrower tables the plain prefill was
    faster in all but one (16 by 35 behind 1024, 80 MB: 30.5 us plain, 43.9 shared; 64 by
    66 behind 512, 192 MB: 80 and 127).  With 2048 rows or more its 256-row tiles are
    full enough, and it writes no partials: never slower, 1.18 times as fast on average
    (64 by 760 behind 2048: 1.76 and 2.33 ms).  Between them it depends on the lengths: 64
    by 4 behind 2048 77 us plain and 44 shared; by 60 behind 32 768 2.12 and 1.69 ms, by
    60 behind 2048 147 and 182 us.

    Lengths and shared lengths are on the device and are not looked at, so tables far
    wider than the lengths, or groups that share little, are cut for nothing (device
    times in a graph): 16 chats of 556 tokens, 256 of them shared, in tables of 32k
    18.4 us plain and 24.2 so; 64 of them 31.1 and 35.0; 256 sequences of 4k of which
    two share 256 tokens 731 and 783.  A caller that knows as much leaves the groups
    out of the step's metadata."""
    return batch > num_groups > 0 and rows < 2048 and batch * span * num_kv_heads * 512 >= 256 << 20


def check_shared(q: torch.Tensor, kv_cache: torch.Tensor, prefixes: SharedPrefixes) -> None:
    """Refuses what the kernels of shared prefixes do not take, by types and shapes alone: ``attention()`` has the
    answer before it stores the step's keys and values."""
    if not isinstance(prefixes, SharedPrefixes):
        raise TypeError(f"prefixes must be SharedPrefixes, got {type(prefixes).__name__}")
    cu_groups, shared_lens = getattr(prefixes.cu_groups, "shape", None), getattr(prefixes.shared_lens, "shape", None)
    if cu_groups is None or shared_lens is None:
        raise TypeError("cu_groups and shared_lens must be torch.Tensors")
    if len(shared_lens) != 1 or cu_groups != (shared_lens[0] + 1,):
        raise ValueError(f"cu_groups {tuple(cu_groups)} and shared_lens {tuple(shared_lens)} must be [groups + 1] and "
                         "[groups]")
    pool, rows = getattr(kv_cache, "shape", ()), getattr(q, "shape", ())
    if len(pool) != 5 or pool[0] != 2:
        raise ValueError("shared prefixes need the pool [2, NB, BS, Hkv, d]")
    check_sharing_heads(rows[1] if len(rows) == 3 else 0, pool[3], pool[4])


def check_sharing_heads(heads: int, num_kv_heads: int, head_dim: int) -> None:
    if head_dim != HEAD_DIM:
        raise ValueError(f"shared prefixes need a head size of {HEAD_DIM}, got {head_dim}")
    if heads > MAX_GROUP * num_kv_heads:
        raise ValueError(f"shared prefixes take up to {MAX_GROUP} q heads a kv head, got {heads} for {num_kv_heads}")


def check_groups(prefixes: SharedPrefixes, like: torch.Tensor):
    """(groups, cu_groups, shared_lens): their number, and both as the kernels take them."""
    require_device("shared_lens", prefixes.shared_lens)
    groups = prefixes.shared_lens.numel()
    return (groups, check_tokens("cu_groups", prefixes.cu_groups, groups + 1, like),
            check_tokens("shared_lens", prefixes.shared_lens, groups, like))


def shared_prefix_attention(q: torch.Tensor, kv_cache: torch.Tensor, block_tables: torch.Tensor,
                            lengths: torch.Tensor, prefixes: SharedPrefixes,
                            cu_seqlens_q: Optional[torch.Tensor] = None, *, max_seqlen_q: int = 1, scale: float,
                            attn_logits_soft_cap: Optional[float] = None,
                            workspace: Optional[torch.Tensor] = None,
                            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """New tokens of sequences that share prefixes in groups: q ``[T, H, 128]``
    over the pool ``[2, NB, BS, Hkv, 128]``, whose rows for the new tokens are
    stored, -> ``[T, H, 128]`` bf16.

    Without ``cu_seqlens_q`` each sequence has one new token, row ``b`` of q
    (a length of zero gives a zero row).  With it the rows of sequence ``b`` are
    ``cu_seqlens_q[b] .. cu_seqlens_q[b + 1]``, at most ``max_seqlen_q`` of them
    are computed, and row ``i`` of ``n`` sees the first ``lengths[b] - n + i + 1``
    tokens (and is zero if that is none; ``cu_seqlens_q`` does not fall).  Rows outside the sequences are zero
    in a new output and left as they were in a given ``out``.

    ``prefixes.shared_lens`` is a promise about the block tables: it is rounded
    down to 64 tokens and cut to the shortest length of its group (sequences
    of no tokens aside), and the shared tokens are read through the table of the group's
    first sequence that has tokens.  Groups do not overlap; sequences outside them
    share nothing.  Cached rows below a length have to be finite.  Other head sizes
    and more than 256 q heads a kv head are refused, whatever the tables' width.

    Scores, softmax statistics and sums are 32-bit; the weights are rounded to
    bf16 for the matrix cores, and q is not rounded again.  How the parts are cut
    follows the whole batch, and with it a row's last bits.  One new token a sequence is computed by the plain decode
    where sharing does not pay (:func:`shared_prefix_pays`).  With ``cu_seqlens_q``
    every row goes through 32-bit partials in the workspace, also where the plain
    prefill is faster; ``attention()`` takes that there.  The workspace
    (``shared_prefix_workspace_bytes``; the plain decode's is smaller) is made here if
    none is given, or one that is too small, not contiguous or not 256-byte aligned.
    """
    if not isinstance(prefixes, SharedPrefixes):
        raise TypeError(f"prefixes must be SharedPrefixes, got {type(prefixes).__name__}")
    (nb, bs, hkv, d), cache_stride = check_pool(kv_cache)
    q_stride = check_heads(q, hkv, d)
    check_sharing_heads(q.shape[1], hkv, d)
    if kv_cache.get_device() != q.get_device():
        raise ValueError(f"kv_cache lives on {kv_cache.device}, q on {q.device}")
    tokens, heads, _ = q.shape
    if cu_seqlens_q is None:
        batch, cu, longest = tokens, None, 1
    else:
        require_device("cu_seqlens_q", cu_seqlens_q)
        if cu_seqlens_q.dim() != 1 or cu_seqlens_q.numel() < 1:
            raise ValueError(f"cu_seqlens_q must be int32 [B + 1], got {tuple(cu_seqlens_q.shape)}")
        batch, longest = cu_seqlens_q.numel() - 1, max_seqlen_q
        cu = check_tokens("cu_seqlens_q", cu_seqlens_q, batch + 1, q)
    if not 0 <= max_seqlen_q <= 0x7fffffff:
        raise ValueError(f"max_seqlen_q {max_seqlen_q}")
    table, _keep = check_table(block_tables, batch, q)
    lens = check_tokens("lengths", lengths, batch, q)
    groups, cu_groups, shared = check_groups(prefixes, q)
    zero_rest = out is None
    out, out_stride = check_output(out, q)
    if tokens == 0:
        return out
    if batch == 0 or longest == 0:
        return out.zero_() if zero_rest else out
    if cu is None and not shared_prefix_pays(batch, groups, hkv, table[2] * bs):
        if workspace is not None:
            workspace, _ = check_workspace(workspace, max(1, decode_workspace_bytes(batch, heads, d, table[2], bs)), q)
        return decode_checked(q, (hkv, nb, bs, d), pool_pointers(kv_cache), cache_stride, _keep, lens,
                              attn_logits_soft_cap, scale, workspace, out)
    need = shared_prefix_workspace_bytes(batch, groups, tokens, heads, hkv, table[2], bs,
                                         max_seqlen_q=None if cu is None else longest)
    _ws, ws_args = check_workspace(workspace, need, q)
    k, v = pool_pointers(kv_cache)
    cap = 0.0 if attn_logits_soft_cap is None else float(attn_logits_soft_cap)
    with on_device(q):
        _lib.call("pa_shared_prefix", q.data_ptr(), q_stride[0], q_stride[1], k, v, nb, bs, *cache_stride, *table,
                  lens.data_ptr(), cu_groups.data_ptr(), shared.data_ptr(), groups,
                  None if cu is None else cu.data_ptr(), batch, tokens, longest, heads, hkv, d, float(scale), cap,
                  int(zero_rest), out.data_ptr(), *out_stride, *ws_args, stream_handle(q))
    return out


def shared_prefix_workspace_bytes(batch: int, num_groups: int, num_tokens: int, num_heads: int, num_kv_heads: int,
                                  pages_per_seq: int, page_size: int, *, max_seqlen_q: Optional[int] = None) -> int:
    """Bytes of the workspace of a :func:`shared_prefix_attention` call; ``max_seqlen_q`` None: without cu_seqlens_q."""
    return int(_lib.load().pa_shared_prefix_workspace_size(
        batch, num_groups, num_tokens, 1 if max_seqlen_q is None else max_seqlen_q, int(max_seqlen_q is not None),
        num_heads, num_kv_heads, pages_per_seq, page_size))
