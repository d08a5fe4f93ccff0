"""CompressedCache.append_float's arguments, without a GPU: what reaches the library."""

import contextlib

import pytest
import torch

from insitu_amd._lib import CapacityError
from insitu_amd.cache import CompressedCache


class _Calls(list):
    def insitu_append_float(self, handle, seq, k, v, type, n, lost):
        self.append((seq, n))
        return 0

    def insitu_cache_destroy(self, handle):
        return 0


class _Context:
    torch_device = torch.device("cpu")

    def __init__(self):
        self.lib = _Calls()

    def ordered(self, *tensors):
        return contextlib.nullcontext()


def _cache(batch=1):
    c = object.__new__(CompressedCache)
    c.n_kv_heads, c.head_dim, c.capacity, c.batch, c.ctx, c.handle, c.first = 2, 64, 1000, batch, _Context(), 1, 0
    return c


@pytest.mark.parametrize("n", [1001, 2 ** 31, 2 ** 32 - 1, 2 ** 32, 2 ** 32 + 3])
def test_more_tokens_than_there_is_room_for(n):
    """A row repeated (stride 0): its number of tokens is refused and not cut off to 32 bits."""
    for c, shape, kw in ((_cache(), (n, 2, 64), {}), (_cache(3), (n, 2, 64), {"seq": 1}), (_cache(3), (3, n, 2, 64), {})):
        x = torch.zeros(1, 2, 64).expand(shape)
        with pytest.raises(CapacityError):
            c.append_float(x, x, **kw)
        assert c.ctx.lib == []
    c = _cache()
    x = torch.zeros(1, 2, 64).expand(1000, 2, 64)
    c.append_float(x, x)
    assert c.ctx.lib == [(0, 1000)]
