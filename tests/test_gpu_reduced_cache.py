"""GPU: the adapters over a ReducedCache - prefill with reductions, single tokens, a drafted tree, accepted drafts - against the same
models over transformers' DynamicCache.  fp32 models: the two differ by rounding alone (attention order, 64-bit against fp32 angles at
positions below 2^12: 2^12 * 2^-24 radians of phase), so outputs agree to a small part of their largest value."""
import pytest
import torch

import framefusion_amd as ffa
from framefusion_amd.synth import video_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F_, P, PRE, POST, D = 12, 24, 5, 7, 256
# 4 layers of fp32 sums over 256-512 terms (2^-24 * 512 = 3e-5 of a sum's terms), phases off by 2^-12: an order of magnitude above both
TOL = 2e-3


def qwen2(dtype=torch.float32):
    from transformers import Qwen2Config, Qwen2ForCausalLM
    from framefusion_amd.models.qwen2 import register_hf_qwen2
    torch.manual_seed(0)
    cfg = Qwen2Config(vocab_size=128, hidden_size=D, intermediate_size=512, num_hidden_layers=4, num_attention_heads=8, num_key_value_heads=2,
                      max_position_embeddings=4096)
    cfg._attn_implementation = "sdpa"
    model = Qwen2ForCausalLM(cfg).to(DEV).to(dtype).eval()
    register_hf_qwen2()
    ffa.apply_framefusion(model, cost=0.3, similarity_lower_bound=0.6, ratio_lower_bound=0.1)
    return model, cfg


def qwen2_vl(dtype=torch.float32):
    from transformers.models.qwen2_vl.modeling_qwen2_vl import Qwen2VLTextConfig, Qwen2VLTextModel
    from framefusion_amd.models.qwen2_vl import register_hf_qwen2_vl
    torch.manual_seed(0)
    cfg = Qwen2VLTextConfig(vocab_size=128, hidden_size=D, intermediate_size=512, num_hidden_layers=4, num_attention_heads=8, num_key_value_heads=2,
                            max_position_embeddings=4096, rope_parameters={"rope_type": "default", "rope_theta": 1e6, "mrope_section": [4, 6, 6]})
    cfg._attn_implementation = "sdpa"

    class Holder(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.model = Qwen2VLTextModel(cfg)
    model = Holder().to(DEV).to(dtype).eval()
    register_hf_qwen2_vl()
    ffa.apply_framefusion(model, cost=0.3, similarity_lower_bound=0.5, ratio_lower_bound=0.1)
    return model, cfg


def prefill(model, cache, emb, pt):
    L = emb.shape[1]
    model.framefusion.prepare(pt.to(DEV), P, PRE, PRE + F_ * P, F_ * P, L)
    return model.model(inputs_embeds=emb, past_key_values=cache, use_cache=True).last_hidden_state


def positions(family, at):
    pos = torch.tensor([at], device=DEV)
    return pos if family == "qwen2" else pos[None].expand(3, 1, -1)


def close(got, want):
    assert got.shape == want.shape and torch.isfinite(got).all()
    off = float((got.float() - want.float()).abs().max() / want.float().abs().max())
    assert off <= TOL, off


@pytest.mark.parametrize("family", ["qwen2", "qwen2_vl"])
def test_prefill_tokens_and_trees(family):
    from transformers.cache_utils import DynamicCache
    model, cfg = (qwen2 if family == "qwen2" else qwen2_vl)()
    emb, pt = video_tokens(F_, P, D, p_change=0.5, sigma=0.3, sigma_hi=1.2, seed=11, pre=PRE, post=POST, dtype=torch.float32)
    emb = emb.to(DEV)
    L = emb.shape[1]
    old, new = DynamicCache(config=cfg), ffa.ReducedCache(4, 2, 32, 512, dtype=torch.float32, page_size=16, pages=60, device=DEV)
    with torch.no_grad():
        want = prefill(model, old, emb, pt)
        got = prefill(model, new, emb, pt)
        close(got, want)
        kv = [old.layers[i].keys.shape[2] for i in range(4)]
        assert new.lengths == kv and len(set(kv)) > 1                                  # another length in every layer
        for i in range(4):
            k, v = new.dense(i)
            close(k, old.layers[i].keys), close(v, old.layers[i].values)
        gen = torch.Generator(device=DEV).manual_seed(1)
        tok = torch.randn(1, 12, D, generator=gen, device=DEV)

        def step(cache, x, at, **kw):
            return model.model(inputs_embeds=x, past_key_values=cache, use_cache=True, position_ids=positions(family, at), **kw).last_hidden_state
        for i in range(3):                                                             # single tokens
            close(step(new, tok[:, i:i + 1], [L + i]), step(old, tok[:, i:i + 1], [L + i]))
        # a tree behind them: 0 - 2 - 4 is what the sequential model sees, 1 and 3 are other drafts
        path, at = [0, 2, 4], L + 3
        want = torch.cat([step(old, tok[:, 3 + i:4 + i], [at + i]) for i in range(3)], 1)
        drafts = torch.randn(1, 5, D, generator=gen, device=DEV)
        drafts[:, path] = tok[:, 3:6]
        mask = torch.eye(5, dtype=torch.bool, device=DEV)
        mask[2, 0] = mask[4, 0] = mask[4, 2] = mask[3, 1] = True
        got = step(new, drafts, [at, at, at + 1, at + 1, at + 2], tree_mask=mask)
        close(got[:, path], want)
        with pytest.raises(RuntimeError, match="pending"):
            step(new, tok[:, :1], [at])
        new.keep(path)
        assert new.lengths == [n + 6 for n in kv]
        close(step(new, tok[:, 6:7], [at + 3]), step(old, tok[:, 6:7], [at + 3]))
        # a chunk of several tokens, causal
        want = torch.cat([step(old, tok[:, 7 + i:8 + i], [at + 4 + i]) for i in range(4)], 1)
        close(step(new, tok[:, 7:11], [at + 4 + i for i in range(4)]), want)
        # drafts of which nothing is accepted leave no trace
        step(new, drafts, [at + 8] * 5, tree_mask=torch.eye(5, dtype=torch.bool, device=DEV))
        new.keep([])
        close(step(new, tok[:, 11:12], [at + 8]), step(old, tok[:, 11:12], [at + 8]))
        # the instance again, for another sample
        new.reset()
        assert new.lengths == [0] * 4 and len(new._free) == 60
        close(prefill(model, new, emb, pt), prefill(model, DynamicCache(config=cfg), emb, pt))


@pytest.mark.parametrize("family", ["qwen2", "qwen2_vl"])
def test_attention_that_needs_a_mask(family):
    """Eager attention is causal only by its mask: the prefill gets one, with a ReducedCache as with a DynamicCache."""
    from transformers.cache_utils import DynamicCache
    model, cfg = (qwen2 if family == "qwen2" else qwen2_vl)()
    emb, pt = video_tokens(F_, P, D, p_change=0.5, sigma=0.3, sigma_hi=1.2, seed=11, pre=PRE, post=POST, dtype=torch.float32)
    emb = emb.to(DEV)
    L = emb.shape[1]
    cfg._attn_implementation = "eager"
    old, new = DynamicCache(config=cfg), ffa.ReducedCache(4, 2, 32, 512, dtype=torch.float32, device=DEV)
    with torch.no_grad():
        close(prefill(model, new, emb, pt), prefill(model, old, emb, pt))
        x = torch.randn(1, 1, D, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
        step = [dict(inputs_embeds=x, past_key_values=c, use_cache=True, position_ids=positions(family, [L])) for c in (new, old)]
        got = model.model(**step[0]).last_hidden_state
        cfg._attn_implementation = "sdpa"              # (a step's eager mask has layer 0's length, a DynamicCache another in every layer)
        close(got, model.model(**step[1]).last_hidden_state)


@pytest.mark.parametrize("store", ["fp8", "fp4", None])
def test_quantised_cache_runs(store):
    """bf16 model, keys and values in 8 and 4 bits: what is stored is the rounding of what a cache in bf16 holds (fp32 of it against the
    block's own half step: 2^-4 and 2^-2 of a value, or of the block's largest over 2^8 for what is small in it)."""
    model, cfg = qwen2(torch.bfloat16)
    emb, pt = video_tokens(F_, P, D, p_change=0.5, sigma=0.3, sigma_hi=1.2, seed=11, pre=PRE, post=POST)
    emb = emb.to(DEV)
    whole, cache = (ffa.ReducedCache(4, 2, 32, 512, store=s, device=DEV) for s in (None, store))
    with torch.no_grad():
        a, b = prefill(model, whole, emb, pt), prefill(model, cache, emb, pt)
        assert torch.equal(a, b) and whole.lengths == cache.lengths                    # the prefill's own attention does not read the cache
        for i in range(4):
            for x, y in zip(whole.dense(i), cache.dense(i)):
                x, y = x.float().unflatten(-1, (-1, 32)), y.float().unflatten(-1, (-1, 32))
                part, floor = {"fp8": (2.0 ** -4, 2.0 ** -9), "fp4": (2.0 ** -2, 2.0 ** -2), None: (0, 0)}[store]
                assert ((x - y).abs() <= part * x.abs() + floor * x.abs().amax(-1, keepdim=True)).all()
        for i in range(3):
            out = model.model(inputs_embeds=torch.randn(1, 1, D, device=DEV).bfloat16(), past_key_values=cache, use_cache=True,
                              position_ids=positions("qwen2", [emb.shape[1] + i])).last_hidden_state
            assert torch.isfinite(out).all()


def test_refusals():
    model, cfg = qwen2()
    emb, pt = video_tokens(F_, P, D, p_change=0.5, sigma=0.3, sigma_hi=1.2, seed=11, pre=PRE, post=POST, dtype=torch.float32)
    emb = emb.to(DEV)
    with torch.no_grad():
        with pytest.raises(NotImplementedError, match="attention_mask"):
            model.model(inputs_embeds=emb, past_key_values=ffa.ReducedCache(4, 2, 32, 512, dtype=torch.float32, device=DEV),
                        attention_mask=torch.ones(1, emb.shape[1], dtype=torch.long, device=DEV))
        with pytest.raises(NotImplementedError, match="one sequence"):
            model.model(inputs_embeds=emb.expand(2, -1, -1), past_key_values=ffa.ReducedCache(4, 2, 32, 512, dtype=torch.float32, device=DEV))
        with pytest.raises(ValueError, match="prefilled"):
            model.model(inputs_embeds=emb[:, :3], past_key_values=ffa.ReducedCache(4, 2, 32, 512, dtype=torch.float32, device=DEV),
                        tree_mask=torch.eye(3, dtype=torch.bool, device=DEV))
    cache = ffa.ReducedCache(2, 2, 32, 40, page_size=16, pages=4, device=DEV)
    x = torch.randn(1, 2, 20, 32, device=DEV).bfloat16()
    with pytest.raises(ffa.FrameFusionHipError, match="max_tokens"):
        cache.append(0, x.repeat(1, 1, 3, 1), x.repeat(1, 1, 3, 1))
    cache.append(0, x, x)
    with pytest.raises(ffa.FrameFusionHipError, match="pending"):
        cache.append(0, x, x)
    with pytest.raises(ffa.FrameFusionHipError, match="accepted"):
        cache.keep([0])                                                                # layer 1 has no pending tokens
    cache.append(1, x, x)
    for bad in ([1, 0], [0, 0], [-1], [20]):
        with pytest.raises(ffa.FrameFusionHipError, match="accepted"):
            cache.keep(bad)
    with pytest.raises(ffa.FrameFusionHipError, match="query"):
        cache.attend(0, x[:, :, :3])
    cache.advance()
    with pytest.raises(ffa.FrameFusionHipError, match="more pages"):
        cache.append(0, x[:, :, :13], x[:, :, :13])
    assert cache.lengths == [20, 20]
    with pytest.raises(ffa.FrameFusionHipError):
        ffa.ReducedCache(0, 2, 32, 40, device=DEV)
