"""What the Qwen2 and Qwen2-VL adapters do differently with a ``ReducedCache``: rotation, cache and decoding attention by this
package's kernels.  The prefill's own attention (and the importance hook) stay as they are; its keys and values are written to the cache
as they come, reduced, one layer shorter than the one before."""
from __future__ import annotations

import torch

from ..cache import ReducedCache
from ..rotary import apply_rotary, rotary_tables


def continues(past_key_values, layer_idx) -> bool:
    """Whether a layer's call is a step behind a prefill (nothing is reduced then)."""
    return isinstance(past_key_values, ReducedCache) and past_key_values.lengths[layer_idx] > 0


def default_positions(past_key_values, count, device, tree_mask):
    """[1, count]: what a call without ``position_ids`` means.  Behind a ``ReducedCache`` the tokens that the model was given count, not
    those that a layer has left, and a drafted token stands as far behind them as it has ancestors."""
    seen = past_key_values.get_seq_length() if past_key_values is not None else 0
    if isinstance(past_key_values, ReducedCache) and tree_mask is not None:
        if tuple(tree_mask.shape) not in ((count, count), (1, count, count)):
            raise ValueError(f"tree_mask must be bool [{count}, {count}], got {tuple(tree_mask.shape)}")
        return (seen + tree_mask.reshape(count, count).sum(-1) - 1).clamp(min=seen).to(device).unsqueeze(0)
    return (torch.arange(count, device=device) + seen).unsqueeze(0)


def position_tables(model, cache, hidden_states, position_ids, attention_mask, tree_mask):
    """[cos, sin] of the step's positions, formed in 64 bits from the model's own frequencies."""
    if attention_mask is not None:
        raise NotImplementedError("a ReducedCache serves one unpadded sequence: run with attention_mask=None (drafted trees: tree_mask)")
    if hidden_states.shape[0] != 1:
        raise NotImplementedError("a ReducedCache serves one sequence (FrameFusion reduces one sample a prefill)")
    if any(cache.pending):
        raise RuntimeError("drafted tokens are pending: call cache.keep(accepted) before the next step")
    if tree_mask is not None and not cache.seen:
        raise ValueError("tree_mask needs a prefilled cache")
    rotary = model.rotary_emb
    if getattr(rotary, "rope_type", "default") in ("dynamic", "longrope"):      # (frequencies that follow the length)
        return list(rotary(hidden_states, position_ids))
    if not position_ids.is_floating_point():
        position_ids = position_ids.long()
    return list(rotary_tables(position_ids.contiguous(), rotary.inv_freq.double(), dtype=hidden_states.dtype, factor=rotary.attention_scaling))


def prefill_mask(model, cache, hidden_states):
    """The causal mask of a prefill's own attention, in the form that the configured attention asks for (None where it is causal by
    itself).  A step has none: ``cache_attention`` masks by position or by ``tree_mask``."""
    from transformers.masking_utils import create_causal_mask
    if cache.seen:
        return None
    return create_causal_mask(config=model.config, inputs_embeds=hidden_states, attention_mask=None, past_key_values=None, position_ids=None)


def rotate(query_states, key_states, cos, sin, sections=None):
    return apply_rotary(query_states, key_states, cos, sin, sections=sections)


def cached_attention(attention, cache, query_states, key_states, value_states, attention_mask, tree_mask):
    """Writes the step's keys and values; the attention output [1, n, H, dh] of a step behind a prefill, None for a prefill."""
    step = cache.lengths[attention.layer_idx] > 0
    if step and (attention_mask is not None or getattr(attention, "sliding_window", None) is not None):
        raise NotImplementedError("a step over a ReducedCache takes neither an attention_mask nor a sliding window")
    cache.append(attention.layer_idx, key_states, value_states)
    if not step:
        return None
    return cache.attend(attention.layer_idx, query_states, mask=tree_mask, scale=attention.scaling).transpose(1, 2)


def finish_step(cache, tree_mask, count) -> None:
    """The `count` tokens of a step count at its end; drafted ones wait for ``cache.keep``."""
    if isinstance(cache, ReducedCache) and tree_mask is None:
        cache.advance(count)
