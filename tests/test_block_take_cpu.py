"""AttentionBlock.take and the position of a cache's row 0, on the CPU: the Python calls against a stand-in for the
library that keeps lengths alone. On the GPU: tests/test_gpu_block_take.py."""

import contextlib
import ctypes

import pytest
import torch

from insitu_amd.block import AttentionBlock
from insitu_amd.cache import CompressedCache


class _Lengths:
    """The library's calls that change or tell lengths."""

    def __init__(self, batch, capacity):
        self.n, self.capacity = [0] * batch, capacity

    def insitu_cache_length(self, handle, b, out):
        ctypes.cast(out, ctypes.POINTER(ctypes.c_int64))[0] = self.n[b]
        return 0

    def insitu_cache_set_length(self, handle, seq, n):
        self.n[seq] = n
        return 0

    def insitu_cache_reset(self, handle):
        self.n = [0] * len(self.n)
        return 0

    def insitu_append_float(self, handle, seq, k, v, type, n, lost):
        for b in range(len(self.n)) if seq < 0 else [seq]:
            self.n[b] += n
        return 0

    def insitu_cache_keep(self, handle, n, rows, stride, counts):
        self.n = [m - n + c for m, c in zip(self.n, counts)]
        return 0

    def insitu_cache_fork(self, handle, copies, src, dst, n, rows, stride, counts):
        for i in range(copies):
            self.n[dst[i]] = self.n[src[i]]
        return 0

    def insitu_cache_destroy(self, handle):
        return 0


class _Context:
    torch_device = torch.device("cpu")

    def __init__(self, lib):
        self.lib = lib

    def ordered(self, *tensors):
        return contextlib.nullcontext()


def _block(batch=1, capacity=100):
    cache = object.__new__(CompressedCache)
    cache.n_kv_heads, cache.head_dim, cache.capacity, cache.batch = 2, 64, capacity, batch
    cache.ctx, cache.handle, cache.first = _Context(_Lengths(batch, capacity)), 1, 0
    block = object.__new__(AttentionBlock)
    block.cache, block.ctx, block.window, block.sinks = cache, cache.ctx, 8, 0
    return block


def _rows(n):
    return torch.zeros(n, 2, 64)


EMPTIED = {"cache.reset": lambda b: b.cache.reset(), "block.reset": lambda b: b.reset(),
           "set_length": lambda b: b.cache.set_length(0), "accept": lambda b: b.accept(b.cache.length),
           "keep": lambda b: b.cache.keep(b.cache.length)}


@pytest.mark.parametrize("again", [0, 40])
@pytest.mark.parametrize("how", list(EMPTIED))
def test_an_emptied_caches_rows_begin_anew(how, again):
    b = _block()
    b.take(_rows(5), _rows(5), first=22)
    assert b.first == 22
    EMPTIED[how](b)
    assert b.cache.length == 0 and b.first == 0
    b.take(_rows(3), _rows(3), first=again)
    assert b.first == again
    b.take(_rows(4), _rows(4))                        # behind them
    assert b.first == again and b.cache.length == 7


def test_rows_that_stay_keep_their_position():
    b = _block()
    b.take(_rows(9), _rows(9), first=22)
    b.cache.set_length(4)
    b.accept(3)
    assert b.cache.length == 1 and b.first == 22
    with pytest.raises(ValueError, match="empty cache"):
        b.take(_rows(1), _rows(1), first=23)


def test_no_rows_have_no_position():
    b = _block()
    b.take(_rows(0), _rows(0), first=22)
    assert b.first == 0 and b.cache.length == 0
    b.take(_rows(2), _rows(2))
    assert b.first == 0


def test_a_batch_is_empty_when_every_sequence_is():
    b = _block(batch=2)
    b.take(_rows(5), _rows(5), first=7, seq=0)
    b.take(_rows(3), _rows(3), seq=1)
    assert b.first == 7
    b.cache.set_length(0, 0)
    assert b.first == 7
    b.cache.set_length(0, 1)
    assert b.first == 0
    b.take(_rows(5), _rows(5), first=7, seq=0)
    b.cache.fork(1, [0])                              # the empty sequence over the one with rows
    assert b.cache.lengths() == [0, 0] and b.first == 0


def test_a_position_that_is_set():
    """Of rows that came another way: until they are dropped."""
    b = _block()
    b.cache.append_float(_rows(3), _rows(3))
    b.first = 30
    b.take(_rows(2), _rows(2))
    assert b.first == 30
    b.cache.reset()
    assert b.first == 0
