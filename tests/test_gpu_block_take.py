"""GPU: positions of hidden states behind rows that AttentionBlock.take took over. forward without positions goes by the
cache's first row; emptied by any call, the cache begins at position 0 again."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

EMPTIED = {"cache.reset": lambda b: b.cache.reset(), "block.reset": lambda b: b.reset(),
           "set_length": lambda b: b.cache.set_length(0), "accept": lambda b: b.accept(b.cache.length)}


def _blocks(ctx, n):
    from insitu_amd import QuantConfig
    from insitu_amd.block import AttentionBlock
    from insitu_amd.config import ModelConfig
    from insitu_amd.host import Weights
    m = ModelConfig(hidden_size=256, num_heads=8, num_kv_heads=2, head_dim=64)
    blocks = [AttentionBlock(m, QuantConfig(key_bits=4, value_bits=2), capacity=80, window=9, ctx=ctx) for _ in range(n)]
    for b in blocks:
        b.weights = Weights.random(m, b.rotation, ctx=ctx)
    return blocks


@pytest.mark.parametrize("again", [None, 0, 40])
@pytest.mark.parametrize("how", list(EMPTIED))
def test_positions_after_an_emptied_cache(ctx, how, again):
    """Rows of position 22 on, dropped; others of position `again` on (or none): forward and forward_tree are those with
    the positions given."""
    import torch
    rng = np.random.default_rng(0)
    a, b = _blocks(ctx, 2)
    k, v = (torch.from_numpy(rng.standard_normal((12, 2, 64))).float().to(ctx.torch_device) for _ in "kv")
    a.take(k[:5], v[:5], first=22)
    a.forward(rng.standard_normal((3, 256)).astype(np.float32))
    EMPTIED[how](a)
    rows = 0
    if again is not None:
        rows = 12
        a.take(k, v, first=again)
        b.take(k, v)
    for n in (4, 1):
        x = rng.standard_normal((n, 256)).astype(np.float32)
        got = a.forward(x)[0]
        want = b.forward(x, np.arange(rows, rows + n) + (again or 0))[0]
        assert all(torch.equal(a.taps[t], b.taps[t]) for t in a.taps) and torch.equal(got, want)
        rows += n
