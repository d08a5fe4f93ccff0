"""Without a GPU: which channels a layer's rotary positions pair up, as its own file shows it."""

import sys
import types

import pytest
import torch

from insitu_amd import ModelConfig
from insitu_amd.adapters.torch_llama import _interleaved


def _half(x):
    a, b = x.chunk(2, -1)
    return torch.cat([-b, a], -1)


def _pairs(x):
    return torch.stack([-x[..., 1::2], x[..., 0::2]], -1).flatten(-2)


def whole_half(q, k, cos, sin, unsqueeze_dim=1):
    cos, sin = cos.unsqueeze(unsqueeze_dim), sin.unsqueeze(unsqueeze_dim)
    return q * cos + _half(q) * sin, k * cos + _half(k) * sin


def whole_interleaved(q, k, cos, sin, unsqueeze_dim=1):
    cos, sin = cos.unsqueeze(unsqueeze_dim), sin.unsqueeze(unsqueeze_dim)
    return q * cos + _pairs(q) * sin, k * cos + _pairs(k) * sin


def part_interleaved(q, k, cos, sin, unsqueeze_dim=1):
    """Of the table's width, half of which is used for the pairs; the channels behind it pass."""
    r = cos.shape[-1]
    cos, sin = (t[..., : r // 2].repeat_interleave(2, -1).unsqueeze(unsqueeze_dim) for t in (cos, sin))
    return tuple(torch.cat([x[..., :r] * cos + _pairs(x[..., :r]) * sin, x[..., r:]], -1) for x in (q, k))


def an_angle_a_pair(q, k, cos, sin, unsqueeze_dim=1):
    cos, sin = cos.unsqueeze(unsqueeze_dim), sin.unsqueeze(unsqueeze_dim)

    def turn(x):
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return turn(q), turn(k)


def another_call(x, sin, cos):
    return x * cos + _half(x) * sin


def another_order(q, k, cos, sin, unsqueeze_dim=1):
    return q.roll(3, -1), k.roll(3, -1)


def _layer(fn, name="a_models_file"):
    mod = types.ModuleType(name)
    if fn is not None:
        mod.apply_rotary_pos_emb = fn
    sys.modules[name] = mod
    return type("Attention", (torch.nn.Module,), {"__module__": name})()


@pytest.fixture(autouse=True)
def _forget():
    yield
    sys.modules.pop("a_models_file", None)


@pytest.mark.parametrize("r", [4, 16, 32, 64, 128])
@pytest.mark.parametrize("fn,want", [(whole_half, False), (whole_interleaved, True), (part_interleaved, True),
                                     (an_angle_a_pair, False), (None, False)])
def test_a_layer_shows_its_pairs(fn, want, r):
    assert _interleaved(_layer(fn), r) is want


@pytest.mark.parametrize("fn", [another_call, another_order])
def test_what_cannot_be_seen_is_refused(fn):
    with pytest.raises(NotImplementedError, match="rope_interleaved"):
        _interleaved(_layer(fn), 64)


def test_transformers_llama_layers_pair_halves():
    from transformers import LlamaConfig
    from transformers.models.llama.modeling_llama import LlamaAttention
    c = LlamaConfig(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64)
    assert _interleaved(LlamaAttention(c, 0), 64) is False


def test_a_configuration_is_told_its_pairs():
    base = {"hidden_size": 256, "num_attention_heads": 4, "num_key_value_heads": 2, "rope_theta": 10000.0,
            "partial_rotary_factor": 0.5}
    assert ModelConfig.from_hf(base).rope_interleaved is False
    m = ModelConfig.from_hf(base, rope_interleaved=True)
    assert m.rope_interleaved is True and m.rotary_dim == 32
