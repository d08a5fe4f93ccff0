"""Device context and the glue between torch device memory and the C ABI.

PyTorch supplies device memory and the stream; the work is done by
libinsitu_hip.so. A Context binds the library to torch's current stream on a
device, so library kernels and torch copies are ordered on one stream.
"""

from __future__ import annotations

import ctypes
import threading

import numpy as np

from . import _lib

_contexts: dict = {}
_lock = threading.Lock()


def _torch():
    import torch
    return torch


class Context:
    """insitu_ctx_create/destroy (include/insitu.h) on one device and stream."""

    def __init__(self, device: int = 0, stream=None) -> None:
        torch = _torch()
        if not torch.cuda.is_available():
            raise RuntimeError("insitu_amd needs a ROCm GPU; there is no CPU fallback")
        self.lib = _lib.load()
        self.device = device
        self.torch_device = torch.device("cuda", device)
        with torch.cuda.device(device):
            s = stream if stream is not None else torch.cuda.current_stream(device)
        self.stream = s
        self._raw = s.cuda_stream
        h = ctypes.c_void_p()
        _lib.check(self.lib.insitu_ctx_create(device, ctypes.c_void_p(s.cuda_stream),
                                              ctypes.byref(h)))
        self.handle = h

    def sync(self) -> None:
        _lib.check(self.lib.insitu_ctx_sync(self.handle))

    def close(self) -> None:
        if self.handle:
            self.lib.insitu_ctx_destroy(self.handle)
            self.handle = None

    def __del__(self) -> None:
        try:
            self.close()
        except Exception:
            pass

    # -- streams --------------------------------------------------------------

    def ordered(self, *tensors) -> "_Ordered":
        """With this, library calls come after what the caller's current stream holds so far, and
        what it gets later comes after them, where that stream is not the context's own; `tensors`
        (used by the calls, perhaps from the other stream's pool) then stay in memory until they
        are through. Nothing waits on the host."""
        return _Ordered(self, tensors)

    # -- tensors --------------------------------------------------------------

    def to_device(self, a, dtype=None):
        """numpy/torch -> contiguous torch tensor on this device (int32 by default)."""
        torch = _torch()
        if isinstance(a, torch.Tensor):
            if a.device == self.torch_device and (dtype is None or a.dtype == dtype) and a.is_contiguous():
                return a
            t = a.to(self.torch_device, non_blocking=False)
        else:
            t = torch.from_numpy(np.ascontiguousarray(a)).to(self.torch_device)
        if dtype is not None:
            t = t.to(dtype)
        return t.contiguous()

    def numbers(self, a, lo: int, hi: int):
        """to_device(a, int32) of numbers of lo .. hi, without making such a number of one that is not."""
        torch = _torch()
        if isinstance(a, torch.Tensor) and (a.dtype == torch.int64 or a.is_floating_point()):
            a = a.clamp(lo - 1, hi + 1)
        return self.to_device(a, torch.int32)


class _Ordered:
    def __init__(self, ctx: Context, tensors) -> None:
        self.ctx, self.tensors, self.other = ctx, tensors, None

    def __enter__(self) -> None:
        if _raw_stream(self.ctx.device) != self.ctx._raw:
            self.other = _torch().cuda.current_stream(self.ctx.device)
            self.ctx.stream.wait_stream(self.other)

    def __exit__(self, *exc) -> None:
        if self.other is not None:
            self.other.wait_stream(self.ctx.stream)
            for t in self.tensors:
                if t is not None:
                    t.record_stream(self.ctx.stream)


def _raw_stream(device: int) -> int:
    """The handle of torch's current stream (without the Stream object around it, 2 us, where torch gives it)."""
    torch = _torch()
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(device) if raw is not None else torch.cuda.current_stream(device).cuda_stream


def default_context(device: int = 0) -> Context:
    with _lock:
        ctx = _contexts.get(device)
        if ctx is None:
            ctx = Context(device)
            _contexts[device] = ctx
        return ctx


def ptr(t) -> ctypes.c_void_p:
    return ctypes.c_void_p(t.data_ptr())


def i64p(a: np.ndarray):
    return a.ctypes.data_as(ctypes.POINTER(ctypes.c_int64))
