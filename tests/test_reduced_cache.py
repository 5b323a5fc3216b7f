"""CPU: what a ReducedCache counts, and the positions that follow from it.  The calls that would reach a kernel are left out."""
import pytest
import torch

import framefusion_amd as ffa
from framefusion_amd import _lib
from framefusion_amd.models.cached import default_positions


@pytest.fixture
def cache(monkeypatch):
    class Nothing:
        def write(self, *a):
            pass

        def keep(self, *a):
            pass
    monkeypatch.setattr(_lib, "host", lambda: Nothing())
    return ffa.ReducedCache(3, 2, 32, 400, page_size=16, device="cpu")


def written(cache, counts):
    for i, n in enumerate(counts):
        x = torch.zeros(1, 2, n, 32, dtype=torch.bfloat16)
        cache.append(i, x, x)


# ---- positions follow on from what the model was given
def test_positions_follow_on_from_the_unreduced_tokens(cache):
    at = lambda n, mask=None: default_positions(cache, n, torch.device("cpu"), mask).tolist()
    assert at(3) == [[0, 1, 2]]
    written(cache, [150, 90, 60])
    assert cache.get_seq_length() == 0                       # (a step's tokens count at its end)
    cache.advance(300)
    assert cache.lengths == [150, 90, 60] and cache.seen == 300 and [cache.get_seq_length(i) for i in range(3)] == [300] * 3
    assert at(2) == [[300, 301]]
    written(cache, [1, 1, 1])
    cache.advance(1)
    assert at(1) == [[301]] and cache.lengths == [151, 91, 61]
    # a tree: a token stands behind its ancestors, siblings side by side; a row that sees nothing of the drafts stands first
    mask = torch.eye(6, dtype=torch.bool)
    mask[2, 0] = mask[3, 0] = mask[4, 0] = mask[4, 2] = True
    mask[5, 5] = False
    assert at(6, mask) == at(6, mask[None]) == [[301, 301, 302, 302, 303, 301]]
    with pytest.raises(ValueError, match="tree_mask"):
        at(5, mask)
    written(cache, [6, 6, 6])
    cache.keep([0, 2, 4])
    assert cache.seen == 304 and cache.lengths == [154, 94, 64]
    written(cache, [6, 6, 6])
    cache.keep([])
    assert cache.seen == 304
    written(cache, [2, 3, 1])
    with pytest.raises(ffa.FrameFusionHipError, match="pending"):
        cache.advance(2)
    cache.advance()
    assert cache.seen == 307
    cache.reset()
    assert cache.seen == cache.get_seq_length() == 0 and cache.lengths == [0, 0, 0]


def test_other_caches_count_as_before():
    class Other:
        def get_seq_length(self, layer_idx=0):
            return 7
    assert default_positions(None, 2, torch.device("cpu"), None).tolist() == [[0, 1]]
    assert default_positions(Other(), 2, torch.device("cpu"), None).tolist() == [[7, 8]]


# ---- transformers' generate
def test_generate_says_that_it_does_not_take_one():
    from transformers import Qwen2Config, Qwen2ForCausalLM
    from framefusion_amd.models.qwen2 import register_hf_qwen2
    cfg = Qwen2Config(vocab_size=128, hidden_size=64, intermediate_size=64, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=2,
                      max_position_embeddings=128, bos_token_id=0, eos_token_id=1, pad_token_id=2)
    model = Qwen2ForCausalLM(cfg).eval()
    register_hf_qwen2()
    ffa.apply_framefusion(model, cost=0.3, similarity_lower_bound=0.6, ratio_lower_bound=0.1)
    with pytest.raises(NotImplementedError, match="generate does not take a ReducedCache"):
        model.generate(torch.arange(3, 9)[None], past_key_values=ffa.ReducedCache(2, 2, 32, 100, dtype=torch.float32, device="cpu"), max_new_tokens=3)
