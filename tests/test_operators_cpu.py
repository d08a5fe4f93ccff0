"""Without a GPU: what the drafts', forks' and seam's entry points refuse before any device work, the scaled
rotary frequencies, and the configurations that name them."""

import ctypes

import numpy as np
import pytest

from insitu_amd import ModelConfig


def _lib():
    from insitu_amd import _lib as m
    return m, m.load()


def test_null_arguments_are_refused():
    m, lib = _lib()
    assert lib.insitu_attend_tree(None, 1, None, 0, None, None, 0, None) == m.EINVAL
    assert lib.insitu_cache_fork(None, 0, None, None, 0, None, 0, None) == m.EINVAL
    assert lib.insitu_cache_keep(None, 0, None, 0, None) == m.EINVAL
    d = m.SeamDesc()
    assert lib.insitu_seam_heads(None, ctypes.byref(d), None, 0, None, 0, None, None, None, None) == m.EINVAL


def test_seam_desc_is_the_headers():
    """The C struct's size: seven int32, padding to eight bytes, two doubles, five pointers, an int64."""
    m, _ = _lib()
    assert ctypes.sizeof(m.SeamDesc) == 32 + 16 + 40 + 8
    assert m.SeamDesc.attn_scale.offset == 32 and m.SeamDesc.max_pos.offset == 88


def _hf(kind, **kw):
    import torch
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    params = {"rope_type": kind, "rope_theta": 10000.0, **kw}
    cfg = LlamaConfig(hidden_size=512, num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=4096,
                      rope_theta=10000.0, rope_scaling=dict(params))
    if getattr(cfg, "rope_parameters", None) is None:
        cfg.rope_parameters = dict(params)
    inv, factor = ROPE_INIT_FUNCTIONS[kind](cfg, torch.device("cpu"))
    return inv.double().numpy(), float(factor), params


@pytest.mark.parametrize("kw", [dict(factor=4.0), dict(factor=40.0, beta_fast=16.0, beta_slow=2.0), dict(factor=8.0, attention_factor=1.0)])
def test_yarn_frequencies_are_transformers(kw):
    """To float32's rounding of a few steps, in which transformers computes them."""
    from insitu_amd import YarnScaling
    inv, factor, params = _hf("yarn", original_max_position_embeddings=1024, **kw)
    y = YarnScaling.from_hf(params)
    plain = 1.0 / 10000.0 ** (np.arange(64) / 64)
    np.testing.assert_allclose(y.apply(plain), inv, rtol=16 * 2.0 ** -24)
    assert y.attention_factor == pytest.approx(factor, rel=2.0 ** -23)


def test_linear_frequencies_are_transformers():
    from insitu_amd import LinearScaling
    inv, factor, _ = _hf("linear", factor=8.0)
    plain = 1.0 / 10000.0 ** (np.arange(64) / 64)
    np.testing.assert_allclose(LinearScaling(8.0).apply(plain), inv, rtol=16 * 2.0 ** -24)
    assert factor == 1.0


def test_tables_of_part_of_a_head_and_of_stretched_positions():
    from insitu_amd import LinearScaling, RoPE, YarnScaling
    whole, part = RoPE.build(64, 100), RoPE.build(16, 100)
    assert part.cos.shape == (100, 8)
    np.testing.assert_array_equal(part.cos, whole.cos[:, ::4])        # theta^(2 j / 16) is theta^(8 j / 64)
    np.testing.assert_array_equal(RoPE.build(64, 400, scaling=LinearScaling(4.0)).sin[::4], whole.sin)
    y = YarnScaling(4.0, 256)
    t = RoPE.build(64, 10, scaling=y)
    assert t.cos[0, 0] == round(32768 * y.attention_factor) and y.attention_factor > 1


def test_scalings_refuse():
    from insitu_amd import LinearScaling, YarnScaling
    for make in (lambda: LinearScaling(0.0), lambda: YarnScaling(0.0, 100), lambda: YarnScaling(2.0, 0),
                 lambda: YarnScaling(2.0, 100, beta_fast=1.0, beta_slow=1.0), lambda: YarnScaling(2.0, 100, beta_slow=0.0)):
        with pytest.raises(ValueError):
            make()


def test_from_hf_reads_the_forms():
    from insitu_amd import LinearScaling, YarnScaling
    base = {"hidden_size": 2048, "num_attention_heads": 32, "num_key_value_heads": 8, "rope_theta": 10000.0}
    m = ModelConfig.from_hf(dict(base, rope_scaling={"type": "linear", "factor": 2.0}))
    assert m.rope_scaling == LinearScaling(2.0) and m.rotary_dim == 64 and not m.rope_interleaved
    m = ModelConfig.from_hf(dict(base, rope_scaling={"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096},
                                 partial_rotary_factor=0.5, rms_norm_eps=1e-5))
    assert m.rope_scaling == YarnScaling(4.0, 4096) and m.rotary_dim == 32 and m.qk_norm_eps == 1e-5
    for bad in ({"rope_type": "dynamic", "factor": 2.0}, {"rope_type": "yarn", "factor": 2.0}, {"rope_type": "longrope"}):
        with pytest.raises(NotImplementedError):
            ModelConfig.from_hf(dict(base, rope_scaling=bad))


@pytest.mark.parametrize("kw", [dict(rotary_dim=0), dict(rotary_dim=3), dict(rotary_dim=66), dict(qk_norm_eps=0.0),
                                dict(qk_norm_eps=-1.0), dict(qk_norm_eps=float("nan"))])
def test_model_config_refuses(kw):
    with pytest.raises(ValueError):
        ModelConfig(hidden_size=256, num_heads=4, num_kv_heads=2, **kw)


def test_a_replaced_head_is_rotated_whole():
    import dataclasses
    from insitu_amd import ModelConfig
    m = ModelConfig(hidden_size=256, num_heads=4, num_kv_heads=2)
    for d in (32, 128):
        r = dataclasses.replace(m, head_dim=d)
        assert r.rotary_dim == d and dataclasses.replace(r, head_dim=64).rotary_dim == 64
    part = dataclasses.replace(m, rotary_dim=32)
    assert dataclasses.replace(part, head_dim=128).rotary_dim == 32
    assert dataclasses.replace(part, rotary_dim=None).rotary_dim == 64 and m == dataclasses.replace(m)
