"""Checks of the operands that the entries over long contexts share."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .kernels._common import require_bf16, require_device


def operand(name: str, t: torch.Tensor, dims: int, like: Optional[torch.Tensor] = None) -> Tuple[int, ...]:
    """Strides of a bf16 device operand of ``dims`` dimensions, contiguous in the last, on ``like``'s device."""
    require_device(name, t)
    stride = t.stride()
    if t.dtype is not torch.bfloat16 or len(stride) != dims or stride[-1] != 1:
        require_bf16(name, t)
        raise ValueError(f"{name} must have {dims} dimensions, got {tuple(t.shape)}")
    if like is not None and t.get_device() != like.get_device():
        raise ValueError(f"{name} lives on {t.device}, the other operands on {like.device}")
    return stride


def check_pool(kv_cache: torch.Tensor, like: Optional[torch.Tensor] = None):
    """Shape ``(NB, BS, Hkv, d)`` and (page, slot, head) strides of the engine's pool ``[2, NB, BS, Hkv, d]``."""
    stride = operand("kv_cache", kv_cache, 5, like)
    if kv_cache.shape[0] != 2:
        raise ValueError(f"kv_cache must be [2, NB, BS, Hkv, d], got {tuple(kv_cache.shape)}")
    return kv_cache.shape[1:], stride[1:4]


def check_table(block_tables: torch.Tensor, batch: int, like: torch.Tensor):
    """(pointer, row stride, pages) of int32 ``[batch, pages]`` block tables, and the tensor they are in."""
    require_device("block_tables", block_tables)
    if block_tables.dtype is not torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] != batch:
        raise ValueError(f"block_tables must be int32 [{batch}, pages], got {block_tables.dtype} "
                         f"{tuple(block_tables.shape)}")
    if block_tables.get_device() != like.get_device():
        raise ValueError(f"block_tables lives on {block_tables.device}, the other operands on {like.device}")
    stride = block_tables.stride()
    if stride[1] != 1 and block_tables.shape[1] > 1:
        block_tables = block_tables.contiguous()
        stride = block_tables.stride()
    return (block_tables.data_ptr(), stride[0], block_tables.shape[1]), block_tables


def check_output(out: Optional[torch.Tensor], q: torch.Tensor):
    """The output tensor like q ``[T, H, d]`` and its (token, head) strides."""
    if out is None:
        _, heads, dim = q.shape
        return torch.empty(q.shape, dtype=torch.bfloat16, device=q.device), (heads * dim, dim)
    stride = operand("out", out, 3, q)
    if out.shape != q.shape:
        raise ValueError(f"out must have shape {tuple(q.shape)}, got {tuple(out.shape)}")
    return out, stride[:2]


def check_workspace(workspace: Optional[torch.Tensor], need: int, like: torch.Tensor):
    """(the tensor, its pointer and bytes): the caller's workspace where it is large enough, else a new one."""
    if workspace is not None:
        require_device("workspace", workspace)
        if workspace.get_device() != like.get_device():
            raise ValueError(f"workspace lives on {workspace.device}, the other operands on {like.device}")
        given = workspace.numel() * workspace.element_size()
        if workspace.is_contiguous() and given >= need and workspace.data_ptr() % 256 == 0:
            return workspace, (workspace.data_ptr(), given)
    if need == 0:
        return None, (None, 0)
    workspace = torch.empty(need, dtype=torch.uint8, device=like.device)
    return workspace, (workspace.data_ptr(), need)


def check_heads(q: torch.Tensor, num_kv_heads: int, head_dim: int):
    """Checked strides of q ``[T, H, d]`` for a pool of these heads."""
    stride = operand("q", q, 3)
    _, heads, dim = q.shape
    if dim != head_dim or heads == 0 or heads % num_kv_heads:
        raise ValueError(f"q must be [T, H, {head_dim}] with H a multiple of {num_kv_heads}, got {tuple(q.shape)}")
    return stride
