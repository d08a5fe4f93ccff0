"""GPU: the seam of models whose configuration gives no eps."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

BASE = {"hidden_size": 256, "num_attention_heads": 4, "num_key_value_heads": 2, "rope_theta": 10000.0,
        "max_position_embeddings": 64, "rms_norm_eps": 0.0}


def test_a_seam_without_eps(ctx):
    import torch
    from insitu_amd import ModelConfig, Seam
    m, plain = ModelConfig.from_hf(BASE), ModelConfig.from_hf(dict(BASE, rms_norm_eps=1e-6))
    p = np.random.default_rng(0).standard_normal((3, 8 * 64)).astype(np.float32)
    for a, b in zip(Seam(m, ctx=ctx).wire(p, 0), Seam(plain, ctx=ctx).wire(p, 0)):
        assert torch.equal(a, b)
    for kw in (dict(q_norm=np.ones(64, np.float32)), dict(k_norm=np.ones(64, np.float32))):
        with pytest.raises(ValueError, match="qk_norm_eps"):
            Seam(m, ctx=ctx, **kw)
