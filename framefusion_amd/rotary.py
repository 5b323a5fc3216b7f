"""Rotary positions: tables of (far, stretched, per-axis) positions, and queries and keys turned by them.

The decoder stack threads ``position_embeddings = [cos, sin]`` through its layers and FrameFusion gathers them with the tokens;
``rotary_tables`` makes such tables and ``apply_rotary`` uses them, one launch for queries and keys together.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import FrameFusionHipError

_get_device = torch._C._cuda_getDevice


_CODE = _lib.DTYPE_CODE


# what a scaling dictionary may hold beside rope_type (or type) and rope_theta: (needed, optional)
_SCALING = {"default": ((), ()), "linear": (("factor",), ()), "ntk": (("factor",), ()),
            "yarn": (("factor", "original_max_position_embeddings"), ("beta_fast", "beta_slow", "attention_factor", "mscale", "mscale_all_dim", "truncate")),
            "llama3": (("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"), ())}


def rotary_frequencies(dim: int, base: Optional[float] = None, scaling: Optional[dict] = None) -> Tuple[torch.Tensor, float]:
    """(float64 frequencies [dim / 2] on the CPU, factor on cosine and sine) for ``rotary_tables``.  ``dim`` is the number of rotated
    channels; ``base`` is 10000, or what ``scaling`` says under "rope_theta".  ``scaling`` stretches the positions for contexts longer than
    the trained one, in transformers' ``rope_parameters`` spelling:

    * ``{"rope_type": "linear", "factor": s}``: every frequency divided by s;
    * ``{"rope_type": "ntk", "factor": s}``: the base raised to base * s^(dim / (dim - 2)), which divides the slowest pair by s and
      leaves the fastest alone;
    * ``{"rope_type": "yarn", "factor": s, "original_max_position_embeddings": n[, "beta_fast": 32, "beta_slow": 1, "truncate": True,
      "attention_factor", or "mscale" with "mscale_all_dim"]}``: pairs that turn more than beta_fast times over n positions are left
      alone, those below beta_slow turns divided by s, the ones between blended by their index (its ends rounded to whole pairs unless
      "truncate" is false).  The factor is "attention_factor", else g(mscale) / g(mscale_all_dim) where both are there, else g(1), with
      g(m) = 0.1 m ln s + 1 (1 for s <= 1);
    * ``{"rope_type": "llama3", "factor": s, "low_freq_factor": a, "high_freq_factor": b, "original_max_position_embeddings": n}``:
      pairs with a wavelength above n / a divided by s, below n / b left alone, blended by n / wavelength between.

    An entry of None counts as left out, "mrope_section" (which is ``apply_rotary``'s) is passed over, any other entry is refused."""
    if dim < 2 or dim % 2:
        raise FrameFusionHipError(f"rotary dimension must be even and positive, got {dim}")
    scaling = {k: v for k, v in (scaling or {}).items() if v is not None and k != "mrope_section"}
    theta = scaling.pop("rope_theta", None)
    if base is not None and theta is not None and float(base) != float(theta):
        raise FrameFusionHipError(f"rotary base {base} and rope_theta {theta} differ")
    base = float(base if base is not None else theta if theta is not None else 10000.0)
    if not base > 0:
        raise FrameFusionHipError(f"rotary base must be positive, got {base}")
    if scaling.pop("partial_rotary_factor", 1) != 1:
        raise FrameFusionHipError("rotary dimension is the number of rotated channels: pass head_dim * partial_rotary_factor and leave the entry out")
    older = scaling.pop("type", "default")
    kind = scaling.pop("rope_type", older)
    if kind not in _SCALING:
        raise FrameFusionHipError(f"rotary scaling {kind!r} is not one of {', '.join(_SCALING)}")
    needed, optional = _SCALING[kind]
    missing, unknown = [k for k in needed if k not in scaling], [k for k in scaling if k not in needed + optional]
    if missing or unknown:
        raise FrameFusionHipError(f"rotary scaling {kind!r}" + (f" needs {', '.join(missing)}" if missing else "") + (f" does not know {', '.join(unknown)}" if unknown else ""))
    pair = torch.arange(0, dim, 2, dtype=torch.float64)
    inv = base ** (-pair / dim)
    if kind == "default":
        return inv, 1.0
    s = float(scaling["factor"])
    if not s > 0:
        raise FrameFusionHipError(f"rotary scaling factor must be positive, got {s}")
    if kind == "linear":
        return inv / s, 1.0
    if kind == "ntk":
        if dim == 2:
            raise FrameFusionHipError("ntk scaling needs more than one pair")
        return (base * s ** (dim / (dim - 2))) ** (-pair / dim), 1.0
    n = float(scaling["original_max_position_embeddings"])
    if not n > 0:
        raise FrameFusionHipError(f"original_max_position_embeddings must be positive, got {n}")
    if kind == "yarn":
        fast, slow = float(scaling.get("beta_fast") or 32), float(scaling.get("beta_slow") or 1)
        if not (base > 1 and fast > 0 and slow > 0):
            raise FrameFusionHipError(f"yarn scaling needs a base above 1 and positive beta_fast and beta_slow, got {base}, {fast}, {slow}")

        def index_of(turns):                      # the (fractional) pair index that turns `turns` times over n positions
            return dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))

        def gain(m):
            return 0.1 * m * math.log(s) + 1.0 if s > 1 else 1.0
        low, high = index_of(fast), index_of(slow)
        if scaling.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        factor = scaling.get("attention_factor")
        if factor is None:
            one, other = scaling.get("mscale"), scaling.get("mscale_all_dim")
            factor = gain(float(one)) / gain(float(other)) if one and other else gain(1.0)
        return inv / s * ramp + inv * (1 - ramp), float(factor)
    a, b = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
    if not b > a:
        raise FrameFusionHipError(f"llama3 scaling needs high_freq_factor above low_freq_factor, got {b} and {a}")
    turns = n * inv / (2 * math.pi)                                     # n / wavelength
    keep = ((turns - a) / (b - a)).clamp(0, 1)
    return inv / s * (1 - keep) + inv * keep, 1.0


def _has_tangent(*tensors) -> bool:
    """Whether forward-mode differentiation asks for a derivative with respect to one of them."""
    return forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def rotary_tables(positions: torch.Tensor, inv_freq: torch.Tensor, dtype: torch.dtype = torch.bfloat16, factor: float = 1.0,
                  interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin) of shape ``positions.shape + (2 * len(inv_freq),)``: int64 positions [B, L] or, one row an axis, [3, B, L];
    ``inv_freq`` float64 on the same device.  The angle is formed and brought into one turn in 64 bits (which costs a position of a million
    2^-31 of a turn, one of 2^31 2^-21) and goes to fp32 there: a turn within 2^-25, cosine and sine within 4 steps of fp32, one
    rounding to ``dtype``."""
    dev = positions.device
    if positions.dtype != torch.int64 or inv_freq.dtype != torch.float64 or inv_freq.ndim != 1 or inv_freq.device != dev:
        raise FrameFusionHipError("rotary_tables: positions must be int64, inv_freq a float64 vector on the same device")
    code = _CODE.get(dtype)
    if code is None:
        raise FrameFusionHipError(f"rotary_tables: dtype {dtype} is not float32, bfloat16 or float16")
    if positions.requires_grad or inv_freq.requires_grad or _has_tangent(inv_freq):
        raise FrameFusionHipError("rotary_tables has no gradient")
    _lib.host().not_traced("rotary_tables")
    if dev.type != "cuda":
        _lib.require_gpu(positions, "rotary_tables")
    if dev.index != _get_device():
        with torch.cuda.device(dev):
            return rotary_tables(positions, inv_freq, dtype, factor, interleaved)
    positions, inv_freq = positions.resolve_neg().contiguous(), inv_freq.resolve_neg().contiguous()
    half = inv_freq.shape[0]
    both = inv_freq.new_empty((2,) + positions.shape + (2 * half,), dtype=dtype)
    cos, sin = both.select(0, 0), both.select(0, 1)
    rc = _lib.load().ff_rotary_tables(positions.data_ptr(), positions.numel(), inv_freq.data_ptr(), half, float(factor),
                                      1 if interleaved else 0, code, cos.data_ptr(), sin.data_ptr(), _lib.stream_ptr()) if half and positions.numel() else 0
    if rc:
        _lib.check(rc, "ff_rotary_tables")
    return cos, sin


class _Rotary(torch.autograd.Function):
    """y = R x for both inputs; the gradient is R^T, the tangent R (rotation calls themselves, so they can be differentiated again)."""

    @staticmethod
    def forward(ctx, query, key, cos, sin, sections, interleaved, transpose):
        ctx.save_for_backward(cos, sin)
        ctx.save_for_forward(cos, sin)
        ctx.how = (sections, interleaved, transpose)
        return _lib.host().rotary(query, key, cos, sin, sections, interleaved, transpose)

    @staticmethod
    def backward(ctx, dq, dk):
        if dq.is_cuda and torch.cuda.is_current_stream_capturing():
            raise FrameFusionHipError("apply_rotary: a differentiable call cannot be captured into a graph (use transpose=True on the gradients)")
        cos, sin = ctx.saved_tensors
        sections, interleaved, transpose = ctx.how
        dq, dk = apply_rotary(dq, dk, cos, sin, sections, interleaved, not transpose)          # (differentiated again where that is asked for)
        return dq, dk, None, None, None, None, None

    @staticmethod
    def jvp(ctx, dq, dk, *constants):
        cos, sin = ctx.saved_tensors
        sections, interleaved, transpose = ctx.how
        return apply_rotary(dq, dk, cos, sin, sections, interleaved, transpose)


def apply_rotary(query: torch.Tensor, key: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, sections: Optional[Sequence[int]] = None,
                 interleaved: bool = False, transpose: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """query [B, H, L, dh] and key [B, H_kv, L, dh] (any strides with whole channels) turned by tables [B or 1, L, rot], or
    [3, B or 1, L, rot] with ``sections`` (the pairs of each axis, M-RoPE); rot <= dh, channels behind rot are copied.  Half
    layout: pair (i, i + rot / 2); ``interleaved``: (2i, 2i + 1).  fp32 inside, one rounding to the inputs' type.  Tables: the
    inputs' type or float32.  ``transpose`` applies the transposed rotation - the gradient, without autograd.

    Differentiable in query and key, backward and forward (the tables are constants).  A differentiable call is not captured into a graph: capture
    ``transpose=True`` calls on the gradients instead."""
    if (query.requires_grad or key.requires_grad) and torch.is_grad_enabled() or _has_tangent(query, key):
        if _has_tangent(cos, sin):
            raise FrameFusionHipError("apply_rotary: the tables are constants, they have no gradient")
        if query.is_cuda and torch.cuda.is_current_stream_capturing():
            raise FrameFusionHipError("apply_rotary: a differentiable call cannot be captured into a graph (use transpose=True on the gradients)")
        return _Rotary.apply(query, key, cos, sin, sections, interleaved, transpose)
    return _lib.host().rotary(query, key, cos, sin, sections, interleaved, transpose)
