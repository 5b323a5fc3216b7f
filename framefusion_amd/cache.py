"""A paged cache of keys and values - as they are, or in 8 or 4 bits - and the attention of new tokens over it.

A reduced prefill leaves another length in every layer.  Here all of them share one pool of pages: a *cache* is four tensors,

    keys, values            [pages, kv_heads, page_size, head_dim]   in T, float8_e4m3fn, or uint8 with two e2m1 codes a byte
    key_scales, value_scales [pages, kv_heads, page_size, head_dim / 32] uint8, or None for a cache in T

(`new_cache` makes them), and a *table* int32 [B, width] lists the pages of each sequence (or of each layer): position p is row
p % page_size of page table[b, p // page_size].  An entry outside [0, pages) means "no page": such positions are not written, read
as zeros and are not attended to.  `start` int32 [B] is the number of tokens a sequence holds before the call's own ones; a
negative entry marks a padding row of the batch.

A stored value is code * 2^(scale byte - 127), one scale for 32 channels; scales are powers of two, so quantising rounds each
channel once and reading back in the type that was written rounds nothing.  A block that holds a NaN or an infinity is stored as NaN.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from ._lib import FrameFusionHipError

_STORES = {"fp8": torch.float8_e4m3fn, "fp4": torch.uint8}


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


def cache_write(cache, key: torch.Tensor, value: torch.Tensor, table: torch.Tensor, start: torch.Tensor) -> None:
    """Stores key and value [B, kv_heads, n, head_dim] at positions start[b] .. start[b] + n - 1 of each sequence (rounded to the
    cache's 8 or 4 bits on the way).  Positions without a page and padding rows are left out; nothing else changes."""
    _lib.host().write(cache, key, value, table, start)


def cache_read(cache, table: torch.Tensor, start: torch.Tensor, count: int, dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(key, value) [B, kv_heads, count, head_dim] of ``dtype`` (the cache's own, or bfloat16 for one of codes): the values of
    positions start[b] .. start[b] + count - 1; zeros where a position has no page and in padding rows."""
    return _lib.host().read(cache, table, start, count, dtype)


def cache_keep(cache, table: torch.Tensor, start: torch.Tensor, accepted: torch.Tensor) -> None:
    """Keeps the accepted ones of the tokens written behind start[b]: row start[b] + i becomes a copy of row
    start[b] + accepted[b, i].  ``accepted`` int32 [B, m], each list strictly increasing; it ends at the first entry that is negative
    (or out of order, or without a page).  The caller then holds start[b] + (length of the list) tokens."""
    _lib.host().keep(cache, table, start, accepted)


def cache_attention(query: torch.Tensor, cache, table: torch.Tensor, start: torch.Tensor, mask: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> torch.Tensor:
    """Attention of n new tokens of each sequence over the cache: query [B, H, n, head_dim], their keys and values already written
    behind the start[b] earlier tokens.  Every new token sees all earlier ones and, of the new ones, those where ``mask`` - bool
    [n, n] or [B, n, n], a tree of drafted tokens: its ancestors and itself - is true; without a mask new token j <= i.  What a
    token does not see contributes nothing, whatever is stored there; one that sees nothing (and a padding row) gets zeros.

    Scores, statistics and sums are held in fp32; a weight is rounded to the inputs' type before it meets the value.  An infinity among the
    values of earlier tokens comes out as one, or as NaN where its weight is below that type's smallest number.

    H is a multiple of the cache's heads, head_dim 32, 64, 128 or 256, n * H at most 983 024.  Returns [B, H, n, head_dim], laid out so that
    ``out.transpose(1, 2)`` is contiguous."""
    return _lib.host().attention(query, cache, table, start, mask, scale)


class ReducedCache:
    """The keys and values of one sequence behind a reduced prefill: another length in every layer, all layers in one pool of pages.

    Passed as ``past_key_values`` to a Qwen2 / Qwen2-VL model patched by ``apply_framefusion`` it takes the place of transformers'
    DynamicCache: the prefill writes each layer's (rotated, reduced) keys and values once, in 16, 8 or 4 bits, and every later call
    runs ``cache_attention`` over them.  A call with ``tree_mask`` (bool [n, n]) attends as a tree of drafted tokens and leaves them
    pending until ``keep(accepted)``.

    ``seen`` counts the tokens that the model was given, before any reduction: where the next one's position follows on (every layer
    holds fewer, even the first, whose call comes behind a reduction).  ``lengths`` is what each layer holds.

    ``max_tokens`` bounds the length of every layer; ``pages`` the pool (default: enough for ``max_tokens`` everywhere - a reduced
    prefill needs far fewer).  One instance serves one stream of calls, like the reference's module; after a step that raised, ``reset``."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, max_tokens: int, dtype: torch.dtype = torch.bfloat16,
                 store: Optional[str] = None, page_size: int = 64, pages: Optional[int] = None, device="cuda"):
        if layers < 1 or max_tokens < 1:
            raise FrameFusionHipError("ReducedCache: layers and max_tokens must be positive")
        width = -(-max_tokens // page_size) if page_size > 0 else 0
        self.tensors = new_cache(layers * width if pages is None else pages, page_size, kv_heads, head_dim, dtype, store, device)
        self.dtype, self.page_size, self.max_tokens = dtype, page_size, max_tokens
        self.seen = 0                               # tokens given to the model, without pending ones
        self.lengths = [0] * layers                 # tokens held, without pending ones
        self.pending = [0] * layers                 # tokens written behind them by the current step
        self._pages = [[] for _ in range(layers)]
        self._free = list(range(self.tensors.keys.shape[0] - 1, -1, -1))
        dev = self.tensors.keys.device
        self._table = torch.full((layers, width), -1, dtype=torch.int32, device=dev)
        self._start = torch.zeros(layers, dtype=torch.int32, device=dev)
        self._rows = [(self._table[i:i + 1], self._start[i:i + 1]) for i in range(layers)]

    def get_seq_length(self, layer_idx: int = 0) -> int:
        """``seen``, for every layer: callers count positions on from it."""
        return self.seen

    def __len__(self) -> int:
        return len(self.lengths)

    @property
    def is_compileable(self):
        """What transformers' ``generate`` asks first."""
        raise NotImplementedError("model.generate does not take a ReducedCache (it passes an attention_mask and drives the cache by one length for all layers): "
                                  "call the model once for the prompt and once for each token, or leave past_key_values to generate")

    def _room(self, layer, count):
        """Pages for `count` tokens of a layer."""
        if count > self.max_tokens:
            raise FrameFusionHipError(f"ReducedCache: {count} tokens in layer {layer}, max_tokens is {self.max_tokens}")
        have = self._pages[layer]
        more = -(-count // self.page_size) - len(have)
        if more > 0:
            if more > len(self._free):
                raise FrameFusionHipError(f"ReducedCache: layer {layer} needs {more} more pages, {len(self._free)} of {self.tensors.keys.shape[0]} are free")
            new = [self._free.pop() for _ in range(more)]
            self._table[layer, len(have):len(have) + more] = torch.tensor(new, dtype=torch.int32)
            have += new

    def update(self, *args, **kwargs):
        """What a layer that does not know this class would call."""
        raise FrameFusionHipError("a ReducedCache serves Qwen2 / Qwen2-VL models patched by apply_framefusion; this layer expects a transformers cache")

    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor) -> None:
        """Writes key and value [1, kv_heads, n, head_dim] behind the layer's tokens; they count once ``advance`` or ``keep`` is called."""
        if key.ndim != 4 or key.shape[0] != 1:
            raise FrameFusionHipError(f"ReducedCache: one sequence, keys [1, kv_heads, n, head_dim], got {tuple(key.shape)}")
        if self.pending[layer]:
            raise FrameFusionHipError("ReducedCache: tokens of the last step are pending; call advance() or keep() first")
        self._room(layer, self.lengths[layer] + key.shape[2])
        cache_write(self.tensors, key, value, *self._rows[layer])
        self.pending[layer] = key.shape[2]

    def attend(self, layer: int, query: torch.Tensor, mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
        """``cache_attention`` of the layer's pending tokens."""
        if query.ndim != 4 or query.shape[2] != self.pending[layer]:
            raise FrameFusionHipError(f"ReducedCache: {self.pending[layer]} tokens are pending in layer {layer}, query is {tuple(query.shape)}")
        return cache_attention(query, self.tensors, *self._rows[layer], mask=mask, scale=scale)

    def _count(self, added, tokens):
        """The pending tokens of every layer become `added` held ones, `tokens` of the model's."""
        self.seen += tokens
        self.lengths = [n + a for n, a in zip(self.lengths, added)]
        self.pending = [0] * len(added)
        if min(added) == max(added):
            if added[0]:
                self._start += added[0]
        else:
            self._start.copy_(torch.tensor(self.lengths, dtype=torch.int32))

    def advance(self, tokens: Optional[int] = None) -> None:
        """Every pending token counts from now on.  ``tokens``: how many the model was given, where layers were written fewer (a reduced
        prefill); by default as many as the fullest layer was written."""
        most = max(self.pending)
        if tokens is not None and tokens < most:
            raise FrameFusionHipError(f"ReducedCache: {most} tokens are pending in a layer, the model cannot have been given {tokens}")
        self._count(self.pending, most if tokens is None else tokens)

    def keep(self, accepted) -> None:
        """Of the pending drafted tokens the ``accepted`` ones (increasing indices, the same in every layer) stay, in one launch for all
        layers; the others are forgotten."""
        accepted = [int(x) for x in accepted]
        n = self.pending[0]
        if min(self.pending) != max(self.pending) or any(a >= b for a, b in zip(accepted, accepted[1:])) \
                or (accepted and not 0 <= accepted[0] <= accepted[-1] < n):
            raise FrameFusionHipError(f"ReducedCache: accepted must be increasing indices of the {n} pending tokens, got {accepted}")
        if accepted and accepted != list(range(len(accepted))):
            lists = torch.tensor(accepted, dtype=torch.int32, device=self._table.device).expand(len(self.lengths), -1).contiguous()
            cache_keep(self.tensors, self._table, self._start, lists)
        self._count([len(accepted)] * len(self.lengths), len(accepted))

    def dense(self, layer: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """The layer's keys and values [1, kv_heads, length, head_dim], read back."""
        return cache_read(self.tensors, self._rows[layer][0], torch.zeros_like(self._rows[layer][1]), self.lengths[layer], dtype=self.dtype)

    def reset(self) -> None:
        """Empty again; every page is free."""
        for have in self._pages:
            self._free += have
            have.clear()
        self._table.fill_(-1)
        self._start.zero_()
        self.seen, self.lengths, self.pending = 0, [0] * len(self.lengths), [0] * len(self.lengths)
