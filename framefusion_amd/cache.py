"""A paged cache of keys and values - as they are, or in 8 or 4 bits - and the attention of new tokens over it.

A reduced prefill leaves another length in every layer.  Here all of them share one pool of pages: a *cache* is four tensors,

    keys, values            [pages, kv_heads, page_size, head_dim]   in T, float8_e4m3fn, or uint8 with two e2m1 codes a byte
    key_scales, value_scales [pages, kv_heads, page_size, head_dim / 32] uint8, or None for a cache in T

(`new_cache` makes them), and a *table* int32 [B, width] lists the pages of each sequence (or of each layer): position p is row
p % page_size of page table[b, p // page_size].  An entry outside [0, pages) means "no page": such positions are not written, read
as zeros and are not attended to.  `start` int32 [B] is the number of tokens a sequence holds before the call's own ones; a
negative entry marks a padding row of the batch.

A stored value is code * 2^(scale byte - 127), one scale for 32 channels; scales are powers of two, so quantising rounds each
channel once and reading back rounds nothing.  A block that holds a NaN or an infinity is stored as NaN.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from ._lib import FrameFusionHipError

_get_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_STORES = {"fp8": torch.float8_e4m3fn, "fp4": torch.uint8}
_STORE_CODE = {torch.float8_e4m3fn: _lib.STORE_E4M3, torch.uint8: _lib.STORE_E2M1, torch.float32: _lib.FF_F32,
               torch.bfloat16: _lib.FF_BF16, torch.float16: _lib.FF_F16}


class CacheTensors(NamedTuple):
    keys: torch.Tensor
    values: torch.Tensor
    key_scales: Optional[torch.Tensor]
    value_scales: Optional[torch.Tensor]


def new_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16, store: Optional[str] = None,
              device="cuda") -> CacheTensors:
    """An empty cache: ``store`` None keeps keys and values in ``dtype``, "fp8" in 8 bits, "fp4" in 4."""
    if store is not None and store not in _STORES:
        raise FrameFusionHipError(f"new_cache: store must be None, 'fp8' or 'fp4', got {store!r}")
    if dtype not in _lib.DTYPE_CODE:
        raise FrameFusionHipError(f"new_cache: dtype {dtype} is not float32, bfloat16 or float16")
    if pages < 0 or kv_heads < 1 or page_size < 16 or page_size % 16 or page_size > 65536 or head_dim < 32 or head_dim % 32 or head_dim > 256:
        raise FrameFusionHipError("new_cache: page_size must be a multiple of 16 up to 65536, head_dim a multiple of 32 up to 256")
    width = head_dim // 2 if store == "fp4" else head_dim
    rows = (pages, kv_heads, page_size)
    keys, values = (torch.zeros(rows + (width,), dtype=_STORES.get(store, dtype), device=device) for _ in range(2))
    if store is None:
        return CacheTensors(keys, values, None, None)
    return CacheTensors(keys, values, *(torch.zeros(rows + (head_dim // 32,), dtype=torch.uint8, device=device) for _ in range(2)))


def _head(what, cache, table, start, n, dtype):
    """The fields of ff_cache_t, every one checked: (fields, kv_heads, head_dim)."""
    keys, values, key_scales, value_scales = cache
    shape, store = keys.shape, _STORE_CODE.get(keys.dtype)
    dev = keys.device
    if store is None or len(shape) != 4 or values.shape != shape or values.dtype != keys.dtype or values.device != dev:
        raise FrameFusionHipError(f"{what}: keys and values of a cache must be alike, [pages, kv_heads, page_size, head_dim]")
    pages, kv_heads, page_size, head_dim = shape
    code = _lib.DTYPE_CODE.get(dtype)
    if code is None:
        raise FrameFusionHipError(f"{what}: dtype {dtype} is not float32, bfloat16 or float16")
    if store >= _lib.STORE_E2M1:
        if store == _lib.STORE_E2M1:
            head_dim *= 2
        want = (pages, kv_heads, page_size, head_dim // 32)
        if (key_scales is None or value_scales is None or key_scales.shape != want or value_scales.shape != want or key_scales.dtype != torch.uint8
                or value_scales.dtype != torch.uint8 or not key_scales.is_contiguous() or not value_scales.is_contiguous()
                or key_scales.device != dev or value_scales.device != dev):
            raise FrameFusionHipError(f"{what}: a cache of codes needs contiguous uint8 scales {want}")
        ks, vs = key_scales.data_ptr(), value_scales.data_ptr()
    else:
        if store != code or key_scales is not None or value_scales is not None:
            raise FrameFusionHipError(f"{what}: a cache in {keys.dtype} holds no scales and serves that type alone, not {dtype}")
        ks = vs = 0
    if not keys.is_contiguous() or not values.is_contiguous():
        raise FrameFusionHipError(f"{what}: the cache's tensors must be contiguous")
    if table.dtype != torch.int32 or table.ndim != 2 or start.dtype != torch.int32 or start.ndim != 1 or start.shape[0] != table.shape[0] \
            or table.device != dev or start.device != dev or not table.is_contiguous() or not start.is_contiguous():
        raise FrameFusionHipError(f"{what}: table must be int32 [B, width] and start int32 [B], contiguous, on the cache's device")
    if dev.type != "cuda":
        _lib.require_gpu(keys, what)
    B, width = table.shape
    return (keys.data_ptr(), values.data_ptr(), ks, vs, table.data_ptr(), start.data_ptr(), store, pages, kv_heads, page_size, head_dim,
            width, B, n, code)


def _no_gradient(what, *tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise FrameFusionHipError(f"{what} has no gradient (serving only): call it under torch.no_grad()")


def _rows(t):
    """`t` [B, heads, n, dh] itself if the kernels can read it in place, else a contiguous copy: (tensor, strides)."""
    st, sh = t.stride(), t.shape
    per = 16 // t.element_size()
    # (the stride of a dimension of one is never used)
    b, h, n = st[0] if sh[0] > 1 else 0, st[1] if sh[1] > 1 else 0, st[2] if sh[2] > 1 else 0
    if st[3] != 1 or (b | h | n) % per or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        b, h, n = t.stride()[:3]
    return t, (b, h, n)


def cache_write(cache, key: torch.Tensor, value: torch.Tensor, table: torch.Tensor, start: torch.Tensor) -> None:
    """Stores key and value [B, kv_heads, n, head_dim] at positions start[b] .. start[b] + n - 1 of each sequence (rounded to the
    cache's 8 or 4 bits on the way).  Positions without a page and padding rows are left out; nothing else changes."""
    _no_gradient("cache_write", key, value)
    head = _head("cache_write", cache, table, start, key.shape[2] if key.ndim == 4 else -1, key.dtype)
    want = (head[12], head[8], head[13], head[10])
    if key.shape != want or value.shape != want or value.dtype != key.dtype or key.device != cache[0].device or value.device != key.device:
        raise FrameFusionHipError(f"cache_write: key and value must be {want} of one dtype on the cache's device, got {tuple(key.shape)} and {tuple(value.shape)}")
    dev = key.device
    if dev.index != _get_device():
        with torch.cuda.device(dev):
            return cache_write(cache, key, value, table, start)
    if key.numel() == 0:
        return
    key, ks = _rows(key)
    value, vs = _rows(value)
    rc = _lib.load().ff_cache_write(_lib.CACHE_ROWS.pack(*head, key.data_ptr(), value.data_ptr(), *ks, *vs, _lib.stream_ptr()))
    if rc:
        _lib.check(rc, "ff_cache_write")


def cache_read(cache, table: torch.Tensor, start: torch.Tensor, count: int, dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(key, value) [B, kv_heads, count, head_dim] of ``dtype`` (the cache's own, or bfloat16 for one of codes): the values of
    positions start[b] .. start[b] + count - 1; zeros where a position has no page and in padding rows."""
    if count < 0:
        raise FrameFusionHipError("cache_read: count must not be negative")
    if dtype is None:
        dtype = cache[0].dtype if cache[0].dtype in _lib.DTYPE_CODE else torch.bfloat16
    head = _head("cache_read", cache, table, start, count, dtype)
    dev = cache[0].device
    if dev.index != _get_device():
        with torch.cuda.device(dev):
            return cache_read(cache, table, start, count, dtype)
    B, kv_heads, dh = head[12], head[8], head[10]
    both = torch.empty((2, B, kv_heads, count, dh), dtype=dtype, device=dev)
    key, value = both[0], both[1]
    if key.numel():
        st = key.stride()[:3]
        rc = _lib.load().ff_cache_read(_lib.CACHE_ROWS.pack(*head, key.data_ptr(), value.data_ptr(), *st, *st, _lib.stream_ptr()))
        if rc:
            _lib.check(rc, "ff_cache_read")
    return key, value


def cache_keep(cache, table: torch.Tensor, start: torch.Tensor, accepted: torch.Tensor) -> None:
    """Keeps the accepted ones of the tokens written behind start[b]: row start[b] + i becomes a copy of row
    start[b] + accepted[b, i].  ``accepted`` int32 [B, m], each list strictly increasing; it ends at the first entry that is negative
    (or out of order, or without a page).  The caller then holds start[b] + (length of the list) tokens."""
    head = _head("cache_keep", cache, table, start, 0, torch.bfloat16 if cache[0].dtype not in _lib.DTYPE_CODE else cache[0].dtype)
    dev = cache[0].device
    if accepted.dtype != torch.int32 or accepted.ndim != 2 or accepted.shape[0] != head[12] or accepted.device != dev or not accepted.is_contiguous():
        raise FrameFusionHipError("cache_keep: accepted must be a contiguous int32 [B, m] on the cache's device")
    if dev.index != _get_device():
        with torch.cuda.device(dev):
            return cache_keep(cache, table, start, accepted)
    if accepted.numel() == 0:
        return
    rc = _lib.load().ff_cache_keep(_lib.CACHE.pack(*head), accepted.data_ptr(), accepted.shape[1], _lib.stream_ptr())
    if rc:
        _lib.check(rc, "ff_cache_keep")


def cache_attention(query: torch.Tensor, cache, table: torch.Tensor, start: torch.Tensor, mask: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> torch.Tensor:
    """Attention of n new tokens of each sequence over the cache: query [B, H, n, head_dim], their keys and values already written
    behind the start[b] earlier tokens.  Every new token sees all earlier ones and, of the new ones, those where ``mask`` - bool
    [n, n] or [B, n, n], a tree of drafted tokens: its ancestors and itself - is true; without a mask new token j <= i.  What a
    token does not see contributes nothing, whatever is stored there; one that sees nothing (and a padding row) gets zeros.

    H is a multiple of the cache's heads, head_dim 32, 64, 128 or 256.  Returns [B, H, n, head_dim], laid out so that
    ``out.transpose(1, 2)`` is contiguous."""
    _no_gradient("cache_attention", query)
    if query.ndim != 4:
        raise FrameFusionHipError(f"cache_attention: query must be [B, H, n, head_dim], got {tuple(query.shape)}")
    B, H, n, dh = query.shape
    dev = query.device
    if mask is not None and (mask.dtype != torch.bool or mask.device != dev or mask.shape not in ((n, n), (B, n, n))):
        raise FrameFusionHipError(f"cache_attention: mask must be bool [{n}, {n}] or [{B}, {n}, {n}], got {mask.dtype} {tuple(mask.shape)}")
    if dh not in (32, 64, 128, 256):
        raise FrameFusionHipError(f"cache_attention: head_dim must be 32, 64, 128 or 256, got {dh}")
    head = _head("cache_attention", cache, table, start, n, query.dtype)
    if B != head[12] or dh != head[10] or H < 1 or H % head[8] or dev != cache[0].device:
        raise FrameFusionHipError(f"cache_attention: query {tuple(query.shape)} does not fit a table of {head[12]} sequences and {head[8]} heads of {head[10]}")
    if dev.index != _get_device():
        with torch.cuda.device(dev):
            return cache_attention(query, cache, table, start, mask, scale)
    mask_ptr = mask_batch = 0
    if mask is not None:
        mask = mask.contiguous()
        mask_ptr, mask_batch = mask.data_ptr(), n * n if mask.ndim == 3 else 0
    out = torch.empty((B, n, H, dh), dtype=query.dtype, device=dev)
    if out.numel():
        query, qs = _rows(query)
        lib = _lib.load()
        scale = dh ** -0.5 if scale is None else float(scale)
        fields = (*head, query.data_ptr(), out.data_ptr(), mask_ptr)
        rest = (H, *qs, n * H * dh, dh, H * dh, mask_batch, scale, _lib.stream_ptr())
        need = lib.ff_cache_attention_workspace_bytes(_lib.CACHE_ATTENTION.pack(*fields, 0, 0, *rest))
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        rc = lib.ff_cache_attention(_lib.CACHE_ATTENTION.pack(*fields, ws.data_ptr() if need else 0, need, *rest))
        if rc:
            _lib.check(rc, "ff_cache_attention")
    return out.transpose(1, 2)
