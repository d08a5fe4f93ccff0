"""AttentionBlock's calls and the caller's stream, on the CPU: every library call of step, prefill and forward lies between
the two waits of Context.ordered (the library's stream waits for the caller's, the caller's for the library's), with
the tensors that the caller made. On the GPU: tests/test_gpu_block_streams.py."""

import contextlib
import ctypes
import types

import numpy as np
import pytest
import torch

from insitu_amd.attention import CompressedAttention
from insitu_amd.block import AttentionBlock
from insitu_amd.cache import CompressedCache
from insitu_amd.rotate import Rotation

H, N_KV, D, HIDDEN = 4, 2, 64, 96


class _Lib:
    """Records each call, whether it is between the waits, and of which tensors."""

    def __init__(self):
        self.inside, self.calls, self.length = [], [], 0

    def __getattr__(self, name):
        def call(*args):
            if name == "insitu_cache_length":
                ctypes.cast(args[2], ctypes.POINTER(ctypes.c_int64))[0] = self.length
            elif name != "insitu_cache_destroy":
                self.calls.append((name, bool(self.inside)))
            return 0
        return call


class _Context:
    torch_device = torch.device("cpu")

    def __init__(self):
        self.lib, self.handle, self.tensors = _Lib(), 1, []

    @contextlib.contextmanager
    def ordered(self, *tensors):
        self.tensors += [t.data_ptr() for t in tensors]
        self.lib.inside.append(1)
        yield
        self.lib.inside.pop()

    def to_device(self, a, dtype=None):
        return torch.as_tensor(a, dtype=dtype).contiguous()


class _Host:
    cast_after_rope, last_saturated = True, 0

    def __init__(self, ctx):
        self.ctx = ctx

    def wire(self, x, positions, *, counts):
        self.ctx.lib.insitu_project_seam()
        return tuple(torch.zeros(len(x), h, D, dtype=torch.int32) for h in (H, N_KV, N_KV))

    def output(self, out):
        self.ctx.lib.insitu_output_projection()
        return torch.zeros(len(out), HIDDEN)


def _block(window, length):
    ctx = _Context()
    ctx.lib.length = length
    cache = object.__new__(CompressedCache)
    cache.n_kv_heads, cache.n_q_heads, cache.head_dim, cache.capacity, cache.batch = N_KV, H, D, 1000, 1
    cache.ctx, cache.handle, cache.first = ctx, 1, 0
    b = object.__new__(AttentionBlock)
    b.ctx, b.cache, b.attn, b.rotation = ctx, cache, CompressedAttention(cache), Rotation.from_seed(D, 0)
    b.window, b.sinks, b.softmax, b.force_token_loop, b.cast_after_rope = window, 0, "online", False, True
    b.model = types.SimpleNamespace(num_heads=H, num_kv_heads=N_KV, head_dim=D, hidden_size=HIDDEN)
    b.weights, b._host, b.taps = object(), _Host(ctx), {}
    return b


@pytest.mark.parametrize("window,length", [(None, 0), (None, 50), (8, 0), (8, 50)])
@pytest.mark.parametrize("call", ["step", "prefill", "forward 1", "forward 5", "token loop"])
def test_every_call_is_between_the_waits(call, window, length):
    b = _block(window, length)
    rows = [torch.zeros(5, h, D, dtype=torch.int32) for h in (H, N_KV, N_KV)]
    x = torch.zeros(int(call[-1]) if call.startswith("forward") else 3, HIDDEN)
    if call == "step":
        rows = [r[:1] for r in rows]
        b.step(*rows)
    elif call == "prefill":
        b.prefill(*rows)
    else:
        rows = [x]
        b.force_token_loop = call == "token loop"
        b.forward(x, np.arange(len(x)))
    calls = b.ctx.lib.calls
    assert calls and all(inside for _, inside in calls), calls
    assert {r.data_ptr() for r in rows} <= set(b.ctx.tensors)
    if call == "step":
        assert [n for n, _ in calls] == ["insitu_step" if window is None else "insitu_step_window"]
