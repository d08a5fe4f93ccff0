"""GPU: a draft's keys and values in another order of sequences and nodes are no draft."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_step_tree_takes_rows_by_sequence(ctx):
    from insitu_amd import AttentionBlock, ModelConfig, QuantConfig
    m = ModelConfig(hidden_size=256, num_heads=8, num_kv_heads=2, head_dim=64)
    blk = AttentionBlock(m, QuantConfig(key_bits=4, value_bits=2), capacity=20, batch=3, ctx=ctx)
    rng = np.random.default_rng(0)
    q, k, v = (np.rint(rng.standard_normal((3, 4, h, 64)) * 32768).astype(np.int32) for h in (8, 2, 2))
    for bad in ((q, k.swapaxes(0, 1), v), (q, k, v.swapaxes(0, 1)), (q, k[:, :, ::-1].swapaxes(2, 3), v),
                (q, k.reshape(3, 8, 1, 64), v), (q, k, v.reshape(-1))):
        with pytest.raises(ValueError, match="must be"):
            blk.step_tree(*bad, [-1, 0, 1, 1])
    assert blk.cache.lengths() == [0, 0, 0]
    blk.step_tree(q, k, v, [-1, 0, 1, 1])
    assert blk.cache.lengths() == [4, 4, 4]
