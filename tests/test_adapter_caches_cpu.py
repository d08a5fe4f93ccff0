"""The adapter's exchange with dense caches, on the CPU: which of a transformers cache's layouts KernelAttention.take
and give handle, and where the rows go. The block is a stand-in that keeps floating rows as they are."""

import types

import pytest
import torch
from transformers import DynamicCache, LlamaConfig, MistralConfig, StaticCache

from insitu_amd.adapters.torch_llama import KernelAttention, ungraft

N_KV, D = 2, 64


class _Rows:
    """CompressedCache of one sequence, uncompressed."""

    def __init__(self):
        self.k = self.v = torch.zeros(0, N_KV, D)

    @property
    def length(self):
        return self.k.shape[0]

    def read_float(self, t0, n, *, seq, dtype):
        assert seq == 0 and 0 <= t0 and t0 + n <= self.length
        return self.k[t0:t0 + n].to(dtype), self.v[t0:t0 + n].to(dtype)


class _Block:
    def __init__(self, window=None, sinks=0):
        self.model = types.SimpleNamespace(num_kv_heads=N_KV, head_dim=D)
        self.cache, self.first, self.window, self.sinks = _Rows(), 0, window, sinks

    def take(self, k, v, *, first=0, seq=None):
        assert not self.cache.length
        self.append(k, v)
        self.first = first

    def append(self, k, v):
        self.cache.k, self.cache.v = torch.cat([self.cache.k, k]), torch.cat([self.cache.v, v])


def _config(window=None):
    kw = dict(hidden_size=128, num_attention_heads=2, num_key_value_heads=N_KV, head_dim=D, num_hidden_layers=2,
              intermediate_size=64)
    return LlamaConfig(**kw) if window is None else MistralConfig(sliding_window=window, **kw)


CACHES = {"dynamic": lambda: DynamicCache(), "dynamic_window": lambda: DynamicCache(config=_config(6)),
          "static": lambda: StaticCache(config=_config(), max_cache_len=16),
          "static_window": lambda: StaticCache(config=_config(6), max_cache_len=16)}


def _rows(lo, hi):
    """Rows lo .. hi - 1 of a sequence, (n, heads, d): each its number, from 1."""
    return (torch.arange(lo, hi) + 1.0)[:, None, None].expand(hi - lo, N_KV, D).contiguous()


def _grown(cache, n, layer=0):
    """An adapter whose block holds a sequence's rows 0 .. n - 1 and has advanced the dense cache by them."""
    a = KernelAttention(_Block(), layer_idx=layer)
    a.kernel.append(_rows(0, n), -_rows(0, n))
    a._advance_hf_cache(cache, torch.zeros(1, n, 128))
    return a


def _held(cache, layer=0):
    return cache.layers[layer].keys[0, 0, :, 0].tolist(), cache.layers[layer].values[0, 1, :, 3].tolist()


@pytest.mark.parametrize("n", [1, 5, 6, 9, 16])
@pytest.mark.parametrize("kind", list(CACHES))
def test_rows_are_given_to_where_they_belong_or_not_at_all(kind, n):
    """A tensor that ends with the sequence takes its last rows; one with room behind it is refused and stays."""
    cache = CACHES[kind]()
    a = _grown(cache, n)
    room = {"static": 16, "static_window": 6}.get(kind, 0)
    if n < room:
        with pytest.raises(NotImplementedError, match="room for"):
            a.give(cache)
        assert not any(_held(cache)[0]) and not any(_held(cache)[1])
        return
    kept = {"dynamic_window": 5, "static_window": 6}.get(kind, n)
    assert a.give(cache) == min(n, kept)
    want = _rows(0, n)[-kept:, 0, 0].tolist()
    assert _held(cache) == (want, [-x for x in want])


class _Residual:
    """A cache with a layer that holds its last rows alone in its tensors, the others elsewhere (quantised, say)."""

    def __init__(self, rows, written):
        x = torch.zeros(1, N_KV, rows, D)
        self.layers, self.written = [types.SimpleNamespace(keys=x, values=x.clone())], written

    def get_seq_length(self, layer_idx=0):
        return self.written


@pytest.mark.parametrize("rows", [0, 3])
def test_rows_that_the_tensors_do_not_hold_are_not_given(rows):
    a = KernelAttention(_Block())
    a.kernel.append(_rows(0, 27), _rows(0, 27))
    with pytest.raises(NotImplementedError, match=f"{rows} of 27 rows"):
        a.give(_Residual(rows, 27))


def test_another_sequences_cache_is_not_given_to():
    a = KernelAttention(_Block())
    assert a.give(DynamicCache()) == 0                # (neither holds a row)
    a.kernel.append(_rows(0, 4), _rows(0, 4))
    with pytest.raises(ValueError, match="not of the block's sequence"):
        a.give(DynamicCache())


def test_layers_are_put_back_all_or_none():
    """The second layer's tensors have room left: the first one's stay as they were, and both stay grafted."""
    cache = DynamicCache()
    blocks = [_grown(cache, 5, layer) for layer in (0, 1)]
    cache.layers[1].keys = torch.cat([cache.layers[1].keys] * 2, 2)
    cache.layers[1].values = cache.layers[1].keys.clone()
    cache.layers[1].get_seq_length = lambda: 5
    model = types.SimpleNamespace(model=types.SimpleNamespace(layers=[types.SimpleNamespace(self_attn=b) for b in blocks]))
    with pytest.raises(NotImplementedError):
        ungraft(model, {0: "own 0", 1: "own 1"}, past_key_values=cache)
    assert not any(_held(cache)[0]) and [x.self_attn for x in model.model.layers] == blocks


@pytest.mark.parametrize("n", [1, 4, 5, 6, 9, 16])
@pytest.mark.parametrize("window", [None, 1, 6, 7, 40])
@pytest.mark.parametrize("kind", list(CACHES))
def test_rows_are_taken_where_the_block_needs_no_others(kind, window, n):
    """A block without a window needs every row, one with a window the last window - 1 of them (and the query's own)."""
    cache = CACHES[kind]()
    x = _rows(0, n).transpose(0, 1)[None]
    cache.update(x, -x, 0)
    a = KernelAttention(_Block(window))
    room = {"static": 16, "static_window": 6}.get(kind, 0)
    there = min(n, {"dynamic_window": 5, "static_window": 6}.get(kind, n))
    if n < room or (there < n and (window is None or there < window - 1)):
        with pytest.raises(NotImplementedError, match="room for" if n < room else f"{there} of {n} rows"):
            a.take(cache)
        assert not a.kernel.cache.length and a.kernel.first == 0
        return
    assert a.take(cache) == there and a.kernel.first == n - there
    assert torch.equal(a.kernel.cache.k, _rows(n - there, n)) and torch.equal(a.kernel.cache.v, -_rows(n - there, n))


@pytest.mark.parametrize("window", [None, 2, 3])
@pytest.mark.parametrize("rows", [0, 3])
def test_rows_that_the_tensors_do_not_hold_are_not_taken(rows, window):
    """Few rows of a long sequence in a layer that is not a window's, or none of them."""
    a = KernelAttention(_Block(window))
    with pytest.raises(NotImplementedError, match=f"{rows} of 27 rows"):
        a.take(_Residual(rows, 27))
    assert not a.kernel.cache.length and a.kernel.first == 0
    assert a.take(_Residual(0, 0)) == 0 and a.take(DynamicCache()) == 0
