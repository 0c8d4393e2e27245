"""Rotary position embedding: interleaved and half layouts, part of the head,
frequencies scaled for long contexts.

``qk_norm_rope_store`` rotates whole 128-wide heads the way the reference's
``apply_rope`` does (qwen3.py:59-78: interleaved pairs, bf16 tables, positions
divided by a factor).  :func:`rotary_embedding` is the general form: any even
part of any head size, either pair layout, bf16 / fp16 / fp32 rows, and
frequencies made once by :func:`rotary_frequencies`.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .kernels._common import require_device, stream_handle

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_ROTARY_DIM = 512


@dataclass(frozen=True)
class RotaryFrequencies:
    """Angle per position of each pair (float64 ``[rotary_dim / 2]`` on the
    device) and the factor on cos and sin.  Made once per model by
    :func:`rotary_frequencies`, or by the caller from its own frequencies."""
    inv_freq: torch.Tensor
    amplitude: float = 1.0

    def __post_init__(self):
        f = self.inv_freq
        if not isinstance(f, torch.Tensor) or f.dtype != torch.float64 or f.dim() != 1 or f.numel() < 1:
            raise ValueError("inv_freq must be a float64 tensor [rotary_dim / 2]")
        if f.numel() * 2 > MAX_ROTARY_DIM:
            raise ValueError(f"rotary_dim must be at most {MAX_ROTARY_DIM}, got {2 * f.numel()}")
        if not f.is_contiguous():
            raise ValueError("inv_freq must be contiguous")

        # (frozen: set once, read on every call)
        object.__setattr__(self, "rotary_dim", 2 * f.numel())
        object.__setattr__(self, "amplitude", float(self.amplitude))


def rotary_frequencies(rotary_dim: int, base: float, *, scaling: Optional[dict] = None,
                       device: torch.device | str = "cuda") -> RotaryFrequencies:
    """Frequencies ``f_i = base ** (-2 i / rotary_dim)``, scaled for contexts
    longer than the trained one (``scaling``, a dict with a ``"type"``):

    * ``"linear"``: ``f_i / factor`` (positions divided by the factor);
    * ``"ntk"``: ``base * factor ** (r / (r - 2))`` for the base, so that the
      slowest pair turns ``factor`` times slower and the fastest as before;
    * ``"yarn"``: pairs that turn more than ``beta_fast`` (32) times over
      ``original_max_position`` positions keep ``f_i``, those below
      ``beta_slow`` (1) turns take ``f_i / factor``, a linear ramp over the pair
      index between; cos and sin are multiplied by ``attention_factor``
      (``0.1 ln(factor) + 1``, 1 for factors below 1).  Models that put that
      factor into the softmax scale instead, squared, pass 1 here.
    """
    if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > MAX_ROTARY_DIM:
        raise ValueError(f"rotary_dim must be even and at most {MAX_ROTARY_DIM}, got {rotary_dim}")
    if not (base > 0 and math.isfinite(base)):
        raise ValueError(f"base must be positive, got {base}")
    kind = None if scaling is None else scaling.get("type")
    if kind not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown rotary scaling type {kind!r} (linear, ntk or yarn)")
    factor = 1.0
    if kind is not None:
        factor = float(scaling.get("factor", 1.0))
        if not (factor > 0 and math.isfinite(factor)):
            raise ValueError(f"the scaling factor must be positive, got {factor}")
    amplitude = 1.0
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    if kind == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs more than one pair")
        base = float(base) * factor ** (rotary_dim / (rotary_dim - 2))
    freq = torch.pow(torch.tensor(float(base), dtype=torch.float64), -2.0 * i / rotary_dim)
    if kind == "linear":
        freq = freq / factor
    elif kind == "yarn":
        span = scaling.get("original_max_position")
        if span is None or span <= 0:
            raise ValueError("yarn scaling needs original_max_position")
        if base <= 1:
            raise ValueError("yarn scaling needs a base above 1")
        fast, slow = float(scaling.get("beta_fast", 32)), float(scaling.get("beta_slow", 1))
        if not fast > 0 or not slow > 0:
            raise ValueError("beta_fast and beta_slow must be positive")

        def pair_of(turns: float) -> float:
            return rotary_dim * math.log(span / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair_of(fast)), 0)
        high = min(math.ceil(pair_of(slow)), rotary_dim - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq / factor * ramp + freq * (1 - ramp)
        amplitude = float(scaling.get("attention_factor", 0.1 * math.log(max(factor, 1.0)) + 1))
    return RotaryFrequencies(freq.to(device), amplitude)


class _Nothing:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_NOTHING = _Nothing()


def on_device(t: torch.Tensor):
    """Context in which launches go to ``t``'s device (nothing to do, and
    nothing spent, where that is the current one)."""
    return _NOTHING if t.get_device() == torch._C._cuda_getDevice() else torch.cuda.device(t.device)


def check_frequencies(freqs: RotaryFrequencies, like: torch.Tensor) -> None:
    if not isinstance(freqs, RotaryFrequencies):
        raise TypeError(f"freqs must be RotaryFrequencies, got {type(freqs).__name__}")
    if freqs.inv_freq.get_device() != like.get_device():
        raise ValueError(f"the frequencies live on {freqs.inv_freq.device}, the rows on {like.device}")


def check_tokens(name: str, t: torch.Tensor, count: int, like: torch.Tensor) -> torch.Tensor:
    """int32 ``[T]`` metadata on the rows' device, contiguous."""
    require_device(name, t)
    if t.dtype != torch.int32 or t.shape != (count,):
        raise ValueError(f"{name} must be int32 of shape [{count}], got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != like.get_device():
        raise ValueError(f"{name} lives on {t.device}, the rows on {like.device}")
    return t if t.is_contiguous() else t.contiguous()


def rotary_embedding(x: torch.Tensor, positions: torch.Tensor, freqs: RotaryFrequencies, *, start: int = 0,
                     interleaved: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotates ``x[t, h, start : start + rotary_dim]`` by the angles of
    ``positions[t]``; the other elements are copied.

    ``x`` is ``[T, H, d]`` (bf16, fp16 or fp32, contiguous in ``d``); pair
    ``i`` is elements ``(2i, 2i + 1)`` of the part if ``interleaved``, else
    ``(i, i + rotary_dim / 2)``.  Angles are float64 products, the rotation is
    float32, rounded once.  ``out`` may be ``x`` itself (rows outside the part
    are then not touched); any other overlap is not supported.
    """
    require_device("x", x)
    if x.dim() != 3:
        raise ValueError(f"x must be [T, H, d], got {tuple(x.shape)}")
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise ValueError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    stride = x.stride()
    if stride[2] != 1:
        raise ValueError("x must be contiguous in its last dimension")
    check_frequencies(freqs, x)
    t, h, d = x.shape
    r = freqs.rotary_dim
    if start < 0 or start + r > d:
        raise ValueError(f"the rotated part [{start}, {start + r}) lies outside a head of {d}")
    pos = check_tokens("positions", positions, t, x)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        out_stride = (h * d, d, 1)
    else:
        require_device("out", out)
        out_stride = out.stride()
        if out.shape != x.shape or out.dtype != x.dtype or out.get_device() != x.get_device() or out_stride[2] != 1:
            raise ValueError(f"out must be {x.dtype} of shape {(t, h, d)} on {x.device}, contiguous in its last "
                             "dimension")
    if t == 0 or h == 0:
        return out
    with on_device(x):
        _lib.call("pa_rotary_embedding", code, x.data_ptr(), stride[0], stride[1], pos.data_ptr(),
                  freqs.inv_freq.data_ptr(),
                  freqs.amplitude, t, h, d, start, r, int(bool(interleaved)), out.data_ptr(), out_stride[0],
                  out_stride[1], stream_handle(x))
    return out
