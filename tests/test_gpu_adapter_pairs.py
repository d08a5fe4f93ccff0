"""GPU: a grafted layer whose file turns part of each head in interleaved pairs: its wire rows against the formula on
the block's own projections; and pairs given by the caller."""

import sys
import types

import pytest

pytestmark = pytest.mark.gpu

CONFIG = {"hidden_size": 256, "num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 64, "rope_theta": 10000.0,
          "max_position_embeddings": 256, "partial_rotary_factor": 0.5}


def _turn(q, k, cos, sin, unsqueeze_dim=1):
    import torch
    r = cos.shape[-1]
    cos, sin = (t[..., : r // 2].repeat_interleave(2, -1).unsqueeze(unsqueeze_dim) for t in (cos, sin))

    def one(x):
        y = torch.stack([-x[..., 1:r:2], x[..., 0:r:2]], -1).flatten(-2)
        return torch.cat([x[..., :r] * cos + y * sin, x[..., r:]], -1)
    return one(q), one(k)


@pytest.fixture
def layer():
    import torch
    import torch.nn as nn
    mod = types.ModuleType("a_models_file")
    mod.apply_rotary_pos_emb = _turn
    sys.modules["a_models_file"] = mod

    class Attention(nn.Module):
        __module__ = "a_models_file"

        def __init__(self):
            super().__init__()
            torch.manual_seed(0)
            for name, a, b in (("q", 256, 512), ("k", 256, 128), ("v", 256, 128), ("o", 512, 256)):
                setattr(self, f"{name}_proj", nn.Linear(a, b, bias=False))

    yield Attention()
    del sys.modules["a_models_file"]


@pytest.mark.parametrize("given", [None, True, False])
def test_pairs(ctx, layer, given):
    import torch
    from insitu_amd.adapters.torch_llama import build_from_layer
    a = build_from_layer(layer, CONFIG, rope_interleaved=given, ctx=ctx)
    m = a.kernel.model
    assert m.rotary_dim == 32 and m.rope_interleaved is (given is not False)
    x = torch.randn(1, 12, 256)
    a(x)
    p = a.kernel.host.project_qkv(x[0]).cpu().double().reshape(12, 12, 64)
    inv = 1.0 / 10000.0 ** (torch.arange(16, dtype=torch.float64) / 16)
    ang = torch.arange(12, dtype=torch.float64)[:, None, None] * inv
    c, s = (torch.round(f(ang) * 32768) / 32768 for f in (torch.cos, torch.sin))
    for name, rows in (("q", p[:, :8] / 8.0), ("k", p[:, 8:10])):
        if m.rope_interleaved:
            want = _turn(rows, rows, torch.cat([c, c], -1)[:, 0], torch.cat([s, s], -1)[:, 0])[0]
        else:
            u, v = rows[..., :16], rows[..., 16:32]
            want = torch.cat([u * c - v * s, u * s + v * c, rows[..., 32:]], -1)
        got = a.kernel.taps[f"wire.{name}"].cpu().double()
        assert (got - want * 65536).abs().max() <= 0.5 + 1e-6      # (the cast's half, and float64 on both sides)
