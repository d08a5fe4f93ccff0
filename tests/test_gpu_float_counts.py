"""GPU: the count of values beyond Q8.16 of keys and values that differ, exactly; and the scale of rows that a block
appended, read back: centroid times norm / 2^24."""

import numpy as np
import pytest

from oracle.quantize import Cache, Format
from oracle.rotate import rotate, signs_from_seed

pytestmark = pytest.mark.gpu

N_KV = 3
EDGES = [128.0, -128.0, 127.99998, -128.00001, 1e4, -1e4, float("inf"), -float("inf"), float("nan"), 0.0, -0.0, 2.0 ** -17,
         127.0, -127.5, 1.0]


def _lost(x):
    """Elements whose value times 2^16, rounded half to even, is no number of 24 bits (NaN is none)."""
    r = np.rint(x.double().numpy() * 65536)
    return int((~((r >= -2 ** 23) & (r <= 2 ** 23 - 1))).sum())


@pytest.mark.parametrize("type", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("d,kb,vb,rounds", [(64, 4, 2, 1), (128, 3, 3, 1), (64, 4, 2, 2), (64, 8, 8, 1)])
def test_counts(ctx, d, kb, vb, rounds, type):
    import torch
    from insitu_amd import QuantConfig
    from insitu_amd.cache import CompressedCache
    c = CompressedCache(N_KV, d, 40, QuantConfig(key_bits=kb, value_bits=vb, rot_rounds=rounds), n_q_heads=N_KV, ctx=ctx)
    n = 19
    x = torch.tensor(EDGES * (n * N_KV * d // len(EDGES) + 1))[:n * N_KV * d].reshape(n, N_KV, d).to(getattr(torch, type))
    y = (x * 0 + 1).to(x.dtype)                       # ones, and NaN in the place of infinities and NaN
    fits = torch.ones_like(x)
    assert 0 < _lost(y) < _lost(x)
    for k, v in ((y, x), (x, y), (x, fits), (fits, x), (fits, y), (fits, fits)):
        c.reset()
        assert c.append_float(k.to(ctx.torch_device), v.to(ctx.torch_device), counts=True) == _lost(k) + _lost(v)


@pytest.mark.parametrize("type", ["float32", "float16", "bfloat16"])
def test_a_blocks_rows_have_their_scale(ctx, type):
    """Rows taken, a turn and a token behind them, read as they are held: the oracle's codes and norms over 2^24."""
    import torch
    from insitu_amd import QuantConfig
    from insitu_amd.block import AttentionBlock
    from insitu_amd.config import ModelConfig
    t, dev = getattr(torch, type), ctx.torch_device
    rng = np.random.default_rng(1)
    m = ModelConfig(hidden_size=256, num_heads=8, num_kv_heads=2, head_dim=64)
    blk = AttentionBlock(m, QuantConfig(key_bits=4, value_bits=2), capacity=60, window=24, sinks=4, ctx=ctx)
    f, sg = Format(d=64, key_bits=4, value_bits=2), signs_from_seed(64, 0, 1)
    host = Cache(2, 60, f)
    dense = [torch.from_numpy(rng.standard_normal((31, 2, 64))).to(t) for _ in "kv"]
    blk.take(*(x.to(dev) for x in dense))
    host.append_rotated(*(rotate(np.rint(x.double().numpy() * 65536).astype(np.int64), sg) for x in dense))
    for n in (20, 1):
        q, k, v = (np.rint(rng.standard_normal((n, h, 64)) * 65536).astype(np.int64) for h in (8, 2, 2))
        host.append_rotated(rotate(k, sg), rotate(v, sg))
        blk.forward_seam(q, k, v)
    kc, _, vc = f.codebooks()[:3]
    got = blk.cache.read_float(seq=0, dtype=t, rotated=True)
    for h in range(2):
        kv = host.view(h)
        for x, idx, norm, c in ((got[0], kv.k_idx, kv.k_norm, kc), (got[1], kv.v_idx, kv.v_norm, vc)):
            want = np.asarray(c)[idx].astype(np.float64) * np.asarray(norm, np.float64)[:, None] / 2.0 ** 24
            # a whole number below 2^24 times a scale of 16 bits: one rounding to 32 bits and one to the type
            np.testing.assert_allclose(x[:, h].double().cpu().numpy(), want, rtol=torch.finfo(t).eps / 2 + 3 * 2.0 ** -24, atol=0)
