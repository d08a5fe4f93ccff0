"""Without a GPU: what a model's configuration says of norms and rotary positions, and what cannot be taken from it."""

import pytest

from insitu_amd import ModelConfig

BASE = {"hidden_size": 2048, "num_attention_heads": 32, "num_key_value_heads": 8, "rope_theta": 10000.0}


@pytest.mark.parametrize("eps", [0.0, 0, -1e-6, float("nan")])
def test_a_models_eps_matters_where_heads_are_normed(eps):
    """rms_norm_eps belongs to the model's other norms too: no value of it keeps a model without norms of queries
    and keys from being read."""
    m = ModelConfig.from_hf(dict(BASE, rms_norm_eps=eps))
    assert m.qk_norm_eps is None and m.head_dim == 64
    with pytest.raises(ValueError, match="qk_norm_eps"):
        ModelConfig(hidden_size=256, num_heads=4, num_kv_heads=2, qk_norm_eps=eps)


@pytest.mark.parametrize("eps,want", [(None, 1e-6), (1e-5, 1e-5), (5e-324, 5e-324)])
def test_a_models_eps_is_read(eps, want):
    assert ModelConfig.from_hf(dict(BASE, rms_norm_eps=eps)).qk_norm_eps == want


@pytest.mark.parametrize("part", [0.3, 1 / 64, 0.0, 1.5, -0.5])
def test_parts_of_a_head_that_have_no_pairs(part):
    """Refused as what is not modelled (a whole head turned instead would be another model)."""
    with pytest.raises(NotImplementedError, match="channels"):
        ModelConfig.from_hf(dict(BASE, partial_rotary_factor=part))


@pytest.mark.parametrize("part,want", [(None, 64), (1.0, 64), (1, 64), (0.5, 32), (0.25, 16), (1 / 32, 2)])
def test_parts_of_a_head(part, want):
    assert ModelConfig.from_hf(dict(BASE, partial_rotary_factor=part)).rotary_dim == want
    assert ModelConfig.from_hf(dict(BASE, rope_parameters={"rope_theta": 1e4, "partial_rotary_factor": part})).rotary_dim == want
