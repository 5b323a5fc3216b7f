"""CPU: every entry of a scaling dictionary counts or is refused."""
import pytest
import torch

import framefusion_amd as ffa

YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}
LLAMA = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}


@pytest.mark.parametrize("extra", [
    {}, {"mscale": 1.0, "mscale_all_dim": 1.0}, {"mscale": 1.0, "mscale_all_dim": 0.707}, {"mscale": 0.707, "mscale_all_dim": 1.0}, {"mscale": 0.707}, {"mscale_all_dim": 0.707},
    {"mscale": 0.0, "mscale_all_dim": 1.0}, {"mscale": 0.7, "mscale_all_dim": 0.9, "attention_factor": 1.5}, {"truncate": False}, {"truncate": True},
    {"truncate": False, "beta_fast": 24, "beta_slow": 2}, {"attention_factor": None, "beta_fast": None}])
@pytest.mark.parametrize("dim,base", [(128, 1e6), (64, 1e4)])
def test_yarn_entries_against_transformers(extra, dim, base):
    """Pair for pair within float32's rounding there: powers to ln(1e6) = 14 carry 14 * 2^-24, and the blend's unrounded ends (in 64 bits
    there too) its own 2^-24 a step."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    scaling = {**YARN, **extra}
    cfg = LlamaConfig(hidden_size=dim * 2, num_attention_heads=2, head_dim=dim, max_position_embeddings=4096 * 40, rope_parameters={**scaling, "rope_theta": base})
    want, want_factor = ROPE_INIT_FUNCTIONS["yarn"](cfg, "cpu")
    for inv, factor in (ffa.rotary_frequencies(dim, base, scaling), ffa.rotary_frequencies(dim, scaling={**scaling, "rope_theta": base})):
        assert torch.allclose(inv, want.double(), rtol=2e-5, atol=0)
        assert abs(factor - want_factor) < 1e-6


def test_the_base_comes_from_either_place():
    want = ffa.rotary_frequencies(64, 1e6)[0]
    assert torch.equal(ffa.rotary_frequencies(64, scaling={"rope_type": "default", "rope_theta": 1e6, "mrope_section": [8, 12, 12]})[0], want)
    assert torch.equal(ffa.rotary_frequencies(64, 1e6, {"rope_theta": 1000000})[0], want)
    assert torch.equal(ffa.rotary_frequencies(64)[0], ffa.rotary_frequencies(64, 1e4)[0])
    assert torch.equal(ffa.rotary_frequencies(64, 1e6, {"type": "linear", "factor": 2.0})[0], want / 2)


@pytest.mark.parametrize("dim,base,scaling,match", [
    (64, 1e4, {"rope_theta": 1e6}, "differ"), (64, 0.0, None, "positive"), (64, None, {"rope_type": "linear", "factor": 2.0, "beta_fast": 3}, "beta_fast"),
    (64, None, {"rope_type": "default", "factor": 2.0}, "factor"), (64, None, {"rope_type": "linear"}, "needs factor"), (64, None, {**YARN, "short_factor": [1.0]}, "short_factor"),
    (64, None, {"rope_type": "yarn", "factor": 4.0}, "original_max_position_embeddings"), (64, None, {**LLAMA, "attention_factor": 2.0}, "attention_factor"),
    (64, None, {**LLAMA, "high_freq_factor": 1.0}, "above"), (64, None, {**YARN, "original_max_position_embeddings": 0}, "positive"), (64, 1.0, YARN, "above 1"),
    (64, None, {**YARN, "beta_fast": -1}, "positive"), (64, None, {"rope_type": "longrope", "factor": 2.0}, "not one of"), (64, None, {"partial_rotary_factor": 0.5}, "rotated channels"),
    (64, None, {"mrope_interleaved": True}, "mrope_interleaved"), (64, None, {"rope_type": "linear", "factor": float("nan")}, "positive")])
def test_what_is_not_known_is_refused(dim, base, scaling, match):
    with pytest.raises(ffa.FrameFusionHipError, match=match):
        ffa.rotary_frequencies(dim, base, scaling)


def test_the_dictionary_is_left_as_it_was():
    scaling = {**YARN, "rope_theta": 1e6, "mrope_section": [8, 12, 12]}
    before = dict(scaling)
    ffa.rotary_frequencies(64, scaling=scaling)
    assert scaling == before
