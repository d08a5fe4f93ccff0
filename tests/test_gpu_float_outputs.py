"""GPU: CompressedCache.read_float into two tensors of one storage: refused where an element is both's, and nothing
written; right where they lie side by side."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _cache(ctx):
    from insitu_amd import QuantConfig
    from insitu_amd.cache import CompressedCache
    c = CompressedCache(2, 64, 40, QuantConfig(key_bits=4, value_bits=2), n_q_heads=2, ctx=ctx)
    rng = np.random.default_rng(0)
    c.append_wire(*(np.rint(rng.standard_normal((30, 2, 64)) * 65536).astype(np.int32) for _ in "kv"))
    return c


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("views,apart", [
    (lambda z: (z[:30], z[15:45]), False), (lambda z: (z[15:45], z[:30]), False), (lambda z: (z[:30], z[29:59]), False),
    (lambda z: (z[:60:2], z[2:62:2]), False), (lambda z: (z[:30], z[30:60]), True), (lambda z: (z[30:60], z[:30]), True),
    (lambda z: (z[:60:2], z[1:61:2]), True)])
def test_two_outputs_of_one_storage(ctx, dtype, views, apart):
    import torch
    c = _cache(ctx)
    z = torch.full((64, 2, 64), 7.0, dtype=getattr(torch, dtype), device=ctx.torch_device)
    out = views(z)
    if not apart:
        with pytest.raises(ValueError, match="one place"):
            c.read_float(seq=0, out=out)
        assert bool((z == 7).all())
        return
    c.read_float(seq=0, out=out)
    for x, want in zip(out, c.read_float(seq=0, dtype=z.dtype)):
        assert torch.equal(x, want)
