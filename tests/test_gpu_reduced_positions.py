"""GPU: steps over a ReducedCache without position_ids stand where the unreduced sequence says."""
import pytest
import torch

import framefusion_amd as ffa
from framefusion_amd.synth import video_tokens
from tests.test_gpu_reduced_cache import D, DEV, F_, P, POST, PRE, positions, prefill, qwen2, qwen2_vl

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("family", ["qwen2", "qwen2_vl"])
def test_default_positions(family):
    """Bit for bit what the same calls with position_ids give: tokens, a chunk, a tree of which some are kept, a token behind them."""
    model, cfg = (qwen2 if family == "qwen2" else qwen2_vl)()
    emb, pt = video_tokens(F_, P, D, p_change=0.5, sigma=0.3, sigma_hi=1.2, seed=11, pre=PRE, post=POST, dtype=torch.float32)
    emb = emb.to(DEV)
    L = emb.shape[1]
    told, left = (ffa.ReducedCache(4, 2, 32, 512, dtype=torch.float32, page_size=16, device=DEV) for _ in range(2))
    mask = torch.eye(5, dtype=torch.bool, device=DEV)
    mask[2, 0] = mask[4, 0] = mask[4, 2] = mask[3, 1] = True
    gen = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(1, 12, D, generator=gen, device=DEV)
    with torch.no_grad():
        assert torch.equal(prefill(model, told, emb, pt), prefill(model, left, emb, pt))
        assert left.seen == L and max(left.lengths) < L
        at = 0
        for n, where, tree in ((1, [L], None), (1, [L + 1], None), (3, [L + 2, L + 3, L + 4], None), (5, [L + 5, L + 5, L + 6, L + 6, L + 7], mask), (1, [L + 8], None)):
            how = dict(inputs_embeds=x[:, at:at + n], use_cache=True, **({} if tree is None else {"tree_mask": tree}))
            want = model.model(past_key_values=told, position_ids=positions(family, where), **how).last_hidden_state
            got = model.model(past_key_values=left, **how).last_hidden_state
            assert torch.equal(got, want)
            if tree is not None:
                told.keep([0, 2, 4]), left.keep([0, 2, 4])
            at += n


def test_positions_of_other_integer_types():
    model, cfg = qwen2()
    emb, pt = video_tokens(F_, P, D, p_change=0.5, sigma=0.3, sigma_hi=1.2, seed=11, pre=PRE, post=POST, dtype=torch.float32)
    emb = emb.to(DEV)
    caches = [ffa.ReducedCache(4, 2, 32, 512, dtype=torch.float32, page_size=16, device=DEV) for _ in range(2)]
    x = torch.randn(1, 2, D, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV)
    with torch.no_grad():
        for c in caches:
            prefill(model, c, emb, pt)
        got, want = (model.model(inputs_embeds=x, past_key_values=c, use_cache=True, position_ids=positions("qwen2", [310, 311]).to(t)).last_hidden_state
                     for c, t in zip(caches, (torch.int32, torch.int64)))
        assert torch.equal(got, want)


def test_the_full_qwen2_vl_model_counts_on_from_the_unreduced_prompt():
    """Its own positions are (tokens seen) + (the prompt's M-RoPE offset): they need the unreduced count."""
    from transformers import Qwen2VLConfig, Qwen2VLForConditionalGeneration
    from transformers.cache_utils import DynamicCache
    from framefusion_amd.models.qwen2_vl import register_hf_qwen2_vl
    from tests.test_gpu_reduced_cache import close
    torch.manual_seed(0)
    VID = 151
    cfg = Qwen2VLConfig(
        text_config=dict(vocab_size=160, hidden_size=256, intermediate_size=512, num_hidden_layers=4, num_attention_heads=8, num_key_value_heads=2,
                         max_position_embeddings=4096, bos_token_id=None, eos_token_id=None,
                         rope_parameters={"rope_type": "default", "rope_theta": 1e6, "mrope_section": [4, 6, 6]}),
        vision_config=dict(depth=1, embed_dim=32, hidden_size=256, num_heads=2, mlp_ratio=2, in_channels=3, patch_size=14, spatial_merge_size=2, temporal_patch_size=2),
        image_token_id=150, video_token_id=VID, vision_start_token_id=152, vision_end_token_id=153)
    cfg._attn_implementation = "sdpa"
    model = Qwen2VLForConditionalGeneration(cfg).to(DEV).eval()
    register_hf_qwen2_vl()
    ffa.apply_framefusion(model, cost=0.3, similarity_lower_bound=0.5, ratio_lower_bound=0.1)
    T, H, W = 12, 8, 12
    n = T * H * W // 4
    ids = torch.tensor([[1, 2, 3, 4, 152] + [VID] * n + [153, 5, 6, 7, 8, 9, 10]], device=DEV)
    frame = torch.randn(H * W, 3 * 2 * 14 * 14)
    frames = [frame]
    for t in range(1, T):
        frames.append(torch.randn_like(frame) if t in (5, 9) else frames[-1] + 0.05 * torch.randn_like(frame))
    video = dict(pixel_values_videos=torch.cat(frames).to(DEV), video_grid_thw=torch.tensor([[T, H, W]], device=DEV), mm_token_type_ids=(ids == VID).int() * 2)
    left, told = (ffa.ReducedCache(4, 2, 32, 512, dtype=torch.float32, device=DEV) for _ in range(2))
    old = DynamicCache(config=cfg.text_config)
    token = torch.tensor([[11]], device=DEV)
    with torch.no_grad():
        for cache in (left, told, old):
            model.model(input_ids=ids, past_key_values=cache, use_cache=True, **video)
        L, delta = ids.shape[1], int(model.model.rope_deltas)
        assert left.seen == L and left.lengths[0] < L and delta != 0
        for i in range(2):
            at = torch.full((3, 1, 1), L + i + delta, device=DEV)
            got = model.model(input_ids=token, past_key_values=left, use_cache=True).last_hidden_state
            assert torch.equal(got, model.model(input_ids=token, past_key_values=told, use_cache=True, position_ids=at).last_hidden_state)
            close(got, model.model(input_ids=token, past_key_values=old, use_cache=True, position_ids=at).last_hidden_state)
