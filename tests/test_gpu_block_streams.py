"""GPU: AttentionBlock called with another current stream than its context's: inputs that come late on that stream are
waited for, and its later work finds the results."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _block(ctx, window):
    from insitu_amd import QuantConfig
    from insitu_amd.block import AttentionBlock
    from insitu_amd.config import ModelConfig
    from insitu_amd.host import Weights
    m = ModelConfig(hidden_size=256, num_heads=8, num_kv_heads=2, head_dim=64)
    b = AttentionBlock(m, QuantConfig(key_bits=4, value_bits=2), capacity=300, window=window, ctx=ctx)
    b.weights = Weights.random(m, b.rotation, ctx=ctx)
    return b


def _calls(block, k, v, wire, x, late):
    """Rows taken, a prompt, a token, hidden states, a token of them, the rows read: what a user's stream gets of each."""
    out = []
    block.take(late(k), late(v))
    for rows in wire:
        rows = [late(r) for r in rows]
        out.append((block.prefill if len(rows[0]) > 1 else block.step)(*rows, stats=False) + 0)
    for h in (x, x[:1]):
        out.append(block.forward(late(h), stats=False)[0] * 1.0)
    out += [r * 1.0 for r in block.cache.read_float(seq=0)]
    return out


@pytest.mark.parametrize("window", [None, 20])
def test_a_caller_on_another_stream(ctx, window):
    import torch
    rng = np.random.default_rng(0)
    dev = ctx.torch_device
    k, v = (torch.from_numpy(rng.standard_normal((30, 2, 64))).float().to(dev) for _ in "kv")
    wire = [[torch.from_numpy(np.rint(rng.standard_normal((n, h, 64)) * 65536).astype(np.int32)).to(dev) for h in (8, 2, 2)]
            for n in (40, 1, 1)]
    x = torch.from_numpy(rng.standard_normal((33, 256)).astype(np.float32)).to(dev)
    a, b = _block(ctx, window), _block(ctx, window)
    want = _calls(a, k, v, wire, x, lambda t: t)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(dev)
    with torch.cuda.stream(side):
        big = torch.randn(1024, 1024, device=dev)

        def late(t):                                  # the same values behind some milliseconds of work
            y = big
            for _ in range(20):
                y = y @ big * 1e-3
            return t + (y[0, 0] * 0).nan_to_num(0.0).to(t.dtype)
        got = _calls(b, k, v, wire, x, late)
    side.synchronize()
    assert len(got) == len(want) and all(torch.equal(g, w) for g, w in zip(got, want))
