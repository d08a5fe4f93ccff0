"""GPU: a context that ends before its caches, as a garbage collector may have it: a cycle's objects are finalised
in any order."""

import gc
import weakref

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _cache(ctx):
    from insitu_amd import QuantConfig
    from insitu_amd.cache import CompressedCache
    return CompressedCache(2, 64, 100, QuantConfig(key_bits=4, value_bits=2), batch=2, n_q_heads=8, ctx=ctx)


def test_a_context_closed_before_its_caches(ctx):
    from insitu_amd.attention import CompressedAttention
    from insitu_amd.runtime import Context
    rng = np.random.default_rng(0)
    rows = [np.rint(rng.standard_normal((2, 9, 2, 64)) * 65536).astype(np.int32) for _ in "kv"]
    q = np.rint(rng.standard_normal((2, 8, 64)) * 16384).astype(np.int32)
    own = Context(ctx.device)
    a, b = _cache(own), _cache(own)
    own.close()
    own.close()
    # the caches live on: the context is there until the last of them goes
    a.append_rotated(*rows)
    got, _ = CompressedAttention(a).attend(q)
    a.close()
    b.append_rotated(*rows)
    again, _ = CompressedAttention(b).attend(q)
    assert np.array_equal(got.cpu().numpy(), again.cpu().numpy())
    b.close()
    b.close()


def test_a_cycle_of_contexts_and_caches(ctx):
    from insitu_amd.runtime import Context

    class Holder:
        pass

    gone = []
    for _ in range(8):
        own = Context(ctx.device)
        h = Holder()
        h.ctx, h.me, h.caches = own, h, [_cache(own), _cache(own)]
        own.holder = h                                  # a cycle through all of them
        gone.append(weakref.ref(own))
    del own, h
    gc.collect()
    assert all(r() is None for r in gone)
    c = _cache(ctx)
    assert c.lengths() == [0, 0]
