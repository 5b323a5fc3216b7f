"""Rotary positions: tables of (far, stretched, per-axis) positions, and queries and keys turned by them.

The decoder stack threads ``position_embeddings = [cos, sin]`` through its layers and FrameFusion gathers them with the tokens;
``rotary_tables`` makes such tables and ``apply_rotary`` uses them, one launch for queries and keys together.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from ._lib import FrameFusionHipError

_get_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


_CODE = _lib.DTYPE_CODE


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: Optional[dict] = None) -> Tuple[torch.Tensor, float]:
    """(float64 frequencies [dim / 2] on the CPU, factor on cosine and sine) for ``rotary_tables``.  ``scaling`` stretches the
    positions for contexts longer than the trained one, in transformers' ``rope_parameters`` spelling:

    * ``{"rope_type": "linear", "factor": s}``: every frequency divided by s;
    * ``{"rope_type": "ntk", "factor": s}``: the base raised to base * s^(dim / (dim - 2)), which divides the slowest pair by s and
      leaves the fastest alone;
    * ``{"rope_type": "yarn", "factor": s, "original_max_position_embeddings": n[, "beta_fast": 32, "beta_slow": 1,
      "attention_factor": 0.1 ln s + 1]}``: pairs that turn more than beta_fast times over n positions are left alone, those below
      beta_slow turns divided by s, the ones between blended by their index;
    * ``{"rope_type": "llama3", "factor": s, "low_freq_factor": a, "high_freq_factor": b, "original_max_position_embeddings": n}``:
      pairs with a wavelength above n / a divided by s, below n / b left alone, blended by n / wavelength between.
    """
    if dim < 2 or dim % 2:
        raise FrameFusionHipError(f"rotary dimension must be even and positive, got {dim}")
    pair = torch.arange(0, dim, 2, dtype=torch.float64)
    inv = float(base) ** (-pair / dim)
    if scaling is None:
        return inv, 1.0
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "default":
        return inv, 1.0
    s = float(scaling["factor"])
    if s <= 0:
        raise FrameFusionHipError(f"rotary scaling factor must be positive, got {s}")
    if kind == "linear":
        return inv / s, 1.0
    if kind == "ntk":
        if dim == 2:
            raise FrameFusionHipError("ntk scaling needs more than one pair")
        return (float(base) * s ** (dim / (dim - 2))) ** (-pair / dim), 1.0
    if kind == "yarn":
        n = float(scaling["original_max_position_embeddings"])
        fast, slow = float(scaling.get("beta_fast") or 32), float(scaling.get("beta_slow") or 1)

        def index_of(turns):                      # the (fractional) pair index that turns `turns` times over n positions
            return dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(float(base)))
        low, high = max(math.floor(index_of(fast)), 0), min(math.ceil(index_of(slow)), dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        factor = scaling.get("attention_factor")
        if factor is None:
            factor = 0.1 * math.log(s) + 1.0 if s > 1 else 1.0
        return inv / s * ramp + inv * (1 - ramp), float(factor)
    if kind == "llama3":
        n = float(scaling["original_max_position_embeddings"])
        a, b = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        turns = n * inv / (2 * math.pi)                                 # n / wavelength
        keep = ((turns - a) / (b - a)).clamp(0, 1)
        return inv / s * (1 - keep) + inv * keep, 1.0
    raise FrameFusionHipError(f"rotary scaling {kind!r} is not one of default, linear, ntk, yarn, llama3")


def rotary_tables(positions: torch.Tensor, inv_freq: torch.Tensor, dtype: torch.dtype = torch.bfloat16, factor: float = 1.0,
                  interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin) of shape ``positions.shape + (2 * len(inv_freq),)``: int64 positions [B, L] or, one row an axis, [3, B, L];
    ``inv_freq`` float64 on the same device.  The angle is formed and reduced in 64 bits, so a far position loses nothing."""
    dev = positions.device
    if positions.dtype != torch.int64 or inv_freq.dtype != torch.float64 or inv_freq.ndim != 1 or inv_freq.device != dev:
        raise FrameFusionHipError("rotary_tables: positions must be int64, inv_freq a float64 vector on the same device")
    code = _CODE.get(dtype)
    if code is None:
        raise FrameFusionHipError(f"rotary_tables: dtype {dtype} is not float32, bfloat16 or float16")
    if positions.requires_grad or inv_freq.requires_grad:
        raise FrameFusionHipError("rotary_tables has no gradient")
    if dev.type != "cuda":
        _lib.require_gpu(positions, "rotary_tables")
    if dev.index != _get_device():
        with torch.cuda.device(dev):
            return rotary_tables(positions, inv_freq, dtype, factor, interleaved)
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    half = inv_freq.shape[0]
    both = inv_freq.new_empty((2,) + positions.shape + (2 * half,), dtype=dtype)
    cos, sin = both.select(0, 0), both.select(0, 1)
    rc = _lib.load().ff_rotary_tables(positions.data_ptr(), positions.numel(), inv_freq.data_ptr(), half, float(factor),
                                      1 if interleaved else 0, code, cos.data_ptr(), sin.data_ptr(), _lib.stream_ptr()) if half and positions.numel() else 0
    if rc:
        _lib.check(rc, "ff_rotary_tables")
    return cos, sin


def _apply(query, key, cos, sin, sections, interleaved, transpose):
    dev = query.get_device()
    if dev != _get_device():
        with torch.cuda.device(dev):
            return _apply(query, key, cos, sin, sections, interleaved, transpose)
    qb, qh, qn, last = query.stride()
    if last != 1:
        query = query.contiguous()
        qb, qh, qn, _ = query.stride()
    kb, kh, kn, last = key.stride()
    if last != 1:
        key = key.contiguous()
        kb, kh, kn, _ = key.stride()
    B, H, L, dh = query.shape
    q_out, k_out = torch.empty_like(query), torch.empty_like(key)          # (in the inputs' own order where they are dense)
    qob, qoh, qon, last = q_out.stride()
    if last != 1:
        q_out = torch.empty_like(query, memory_format=torch.contiguous_format)
        qob, qoh, qon, _ = q_out.stride()
    kob, koh, kon, last = k_out.stride()
    if last != 1:
        k_out = torch.empty_like(key, memory_format=torch.contiguous_format)
        kob, koh, kon, _ = k_out.stride()
    shape, st = cos.shape, cos.stride()
    args = _lib.ROTARY.pack(query.data_ptr(), key.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                            _CODE[query.dtype], _CODE[cos.dtype], B, L, H, key.shape[1], dh, shape[-1],
                            qb, qh, qn, kb, kh, kn, qob, qoh, qon, kob, koh, kon,
                            st[0] if len(shape) == 4 else 0, st[-3] if shape[-3] > 1 else 0, st[-2],
                            sections[0] if sections else 0, sections[1] if sections else 0, 1 if interleaved else 0, 1 if transpose else 0,
                            _raw_stream(dev))
    if B and L:
        rc = _lib.load().ff_rotary_apply(args)
        if rc:
            _lib.check(rc, "ff_rotary_apply")
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    """y = R x for both inputs; the gradient is R^T (itself a rotation call, so it can be differentiated again)."""

    @staticmethod
    def forward(ctx, query, key, cos, sin, sections, interleaved, transpose):
        ctx.save_for_backward(cos, sin)
        ctx.how = (sections, interleaved, transpose)
        return _apply(query, key, cos, sin, sections, interleaved, transpose)

    @staticmethod
    def backward(ctx, dq, dk):
        cos, sin = ctx.saved_tensors
        sections, interleaved, transpose = ctx.how
        turn = _Rotary.apply if torch.is_grad_enabled() else _apply           # (differentiated again, or the end of the line)
        dq, dk = turn(dq, dk, cos, sin, sections, interleaved, not transpose)
        return dq, dk, None, None, None, None, None


def apply_rotary(query: torch.Tensor, key: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, sections: Optional[Sequence[int]] = None,
                 interleaved: bool = False, transpose: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """query [B, H, L, dh] and key [B, H_kv, L, dh] (any strides with whole channels) turned by tables [B or 1, L, rot], or
    [3, B or 1, L, rot] with ``sections`` (the pairs of each axis, M-RoPE); rot <= dh, channels behind rot are copied.  Half
    layout: pair (i, i + rot / 2); ``interleaved``: (2i, 2i + 1).  fp32 inside, one rounding to the inputs' type.  Tables: the
    inputs' type or float32.  ``transpose`` applies the transposed rotation - the gradient, without autograd.

    Differentiable in query and key (the tables are constants).  A differentiable call is not captured into a graph: capture
    ``transpose=True`` calls on the gradients instead."""
    qs, ks, cs, dtype, dev = query.shape, key.shape, cos.shape, query.dtype, query.get_device()
    if len(qs) != 4 or len(ks) != 4 or qs[0] != ks[0] or qs[2:] != ks[2:]:
        raise FrameFusionHipError(f"apply_rotary: query {tuple(qs)} and key {tuple(ks)} must be [B, H, L, dh] and [B, H_kv, L, dh]")
    if dtype not in _CODE or key.dtype is not dtype:
        raise FrameFusionHipError(f"apply_rotary: dtypes {dtype} / {key.dtype} must be the same of float32, bfloat16, float16")
    if cos.dtype is not dtype and cos.dtype is not torch.float32 or sin.dtype is not cos.dtype or sin.shape != cs:
        raise FrameFusionHipError("apply_rotary: cos and sin must have one shape and the inputs' dtype or float32")
    if key.get_device() != dev or cos.get_device() != dev or sin.get_device() != dev:
        raise FrameFusionHipError("apply_rotary: all tensors must be on one device")
    if sections is not None:
        sections = tuple([int(x) for x in sections])
        if len(sections) != 3 or min(sections) < 1 or len(cs) != 4 or cs[0] != 3 or 2 * sum(sections) != cs[-1] or interleaved:
            raise FrameFusionHipError(f"apply_rotary: sections {sections} need tables [3, B, L, 2 * sum] in the half layout, got {tuple(cs)}")
    elif len(cs) != 3:
        raise FrameFusionHipError(f"apply_rotary: tables must be [B or 1, L, rot] (or [3, ...] with sections), got {tuple(cs)}")
    if cs[-3] not in (1, qs[0]) or cs[-2] != qs[2] or cs[-1] % 2 or not 2 <= cs[-1] <= qs[3]:
        raise FrameFusionHipError(f"apply_rotary: tables {tuple(cs)} do not fit query {tuple(qs)}")
    if cos.requires_grad or sin.requires_grad:
        raise FrameFusionHipError("apply_rotary: the tables are constants, they have no gradient")
    if dev < 0:
        _lib.require_gpu(query, "apply_rotary")
    if cos.stride(-1) != 1 or sin.stride() != cos.stride():
        cos, sin = cos.contiguous(), sin.contiguous()
    if (query.requires_grad or key.requires_grad) and torch.is_grad_enabled():
        if torch.cuda.is_current_stream_capturing():
            raise FrameFusionHipError("apply_rotary: a differentiable call cannot be captured into a graph (use transpose=True on the gradients)")
        return _Rotary.apply(query, key, cos, sin, sections, interleaved, transpose)
    return _apply(query, key, cos, sin, sections, interleaved, transpose)
