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
