"""Without a GPU: what the entry points of windows and floating rows refuse before any device work, and the
struct they take."""

import ctypes

import pytest


def _lib():
    from insitu_amd import _lib as m
    return m, m.load()


def test_null_arguments_are_refused():
    m, lib = _lib()
    r = m.FloatRows()
    assert lib.insitu_attend_window(None, -1, 1, 1, 0, None, None, 0, None) == m.EINVAL
    assert lib.insitu_append_float(None, -1, ctypes.byref(r), ctypes.byref(r), 0, 1, None) == m.EINVAL
    assert lib.insitu_read_float(None, -1, 0, 1, 0, ctypes.byref(r), ctypes.byref(r), 0) == m.EINVAL


def test_float_rows_are_the_headers():
    """The C struct's size: a pointer and three int64."""
    m, _ = _lib()
    assert ctypes.sizeof(m.FloatRows) == 32 and m.FloatRows.head_stride.offset == 24


def test_numbers_that_64_bits_do_not_hold():
    m, _ = _lib()
    assert m.int64(-(1 << 63), "x") == -(1 << 63) and m.int64(True, "x") == 1
    for bad in (1 << 63, -(1 << 63) - 1):
        with pytest.raises(ValueError):
            m.int64(bad, "x")
    with pytest.raises(TypeError):
        m.int64(1.0, "x")


@pytest.mark.parametrize("make,bad", [
    (lambda t: t.zeros(2, 3, 4), False), (lambda t: t.zeros(2, 3, 8)[..., :4], False), (lambda t: t.zeros(3, 2, 4).transpose(0, 1), False),
    (lambda t: t.zeros(2, 1, 4).expand(2, 3, 4), True), (lambda t: t.zeros(2, 3, 8)[..., ::2], True), (lambda t: t.zeros(0, 3, 4), False),
    (lambda t: t.zeros(40).as_strided((2, 3, 4), (6, 3, 1)), True), (lambda t: t.zeros(1, 1, 1).expand(1, 1, 1), False)])
def test_outputs_in_one_place(make, bad):
    import torch
    from insitu_amd.cache import _overlaps
    assert _overlaps(make(torch)) is bad


class _Names:
    def __init__(self, **kw):
        self.__dict__.update(kw)


@pytest.mark.parametrize("module,config,want", [
    (dict(), dict(), None),
    (dict(), dict(sliding_window=4096), 4096),
    (dict(), dict(sliding_window=None), None),
    (dict(), dict(sliding_window=512, use_sliding_window=False), None),
    (dict(), dict(sliding_window=512, layer_types=["full_attention", "sliding_attention"]), 512),
    (dict(), dict(sliding_window=512, layer_types=["sliding_attention", "full_attention"]), None),
    (dict(sliding_window=None), dict(sliding_window=512), None),
    (dict(sliding_window=128), dict(), 128),
    (dict(sliding_window=-1), dict(), None),
])
def test_a_layers_own_window(module, config, want):
    """Of layer 1: the module's word before the configuration's, given as attributes or as a dictionary."""
    from insitu_amd.adapters.torch_llama import _window
    assert _window(_Names(**module), _Names(**config), 1) == want
    assert _window(_Names(**module), config, 1) == want
