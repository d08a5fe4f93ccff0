"""GPU: the two kernels of the window attends, each pinned (INSITU_DEBUG_WINDOW) on calls that the automatic choice would
give the other: prompts over workgroups of one tile, and few queries over waves of 16 rows, with the masks, events,
digits and clamps where they differ; several launches of one call; a cache of more rows than the prompts' kernel
counts. Against oracle/c, as the calls of the automatic choice."""

import numpy as np
import pytest

import test_gpu_window as w

pytestmark = pytest.mark.gpu

FEW, PROMPTS = 1, 2


@pytest.fixture(params=[FEW, PROMPTS], ids=["few", "prompts"])
def pinned(request, monkeypatch):
    """Caches of the helpers of test_gpu_window, on one kernel."""
    from insitu_amd import _lib
    make = w._cache

    def cache(ctx, *args, **kw):
        c = make(ctx, *args, **kw)
        _lib.check(ctx.lib.insitu_cache_debug(c.handle, _lib.DEBUG_WINDOW, request.param))
        return c
    monkeypatch.setattr(w, "_cache", cache)
    return request.param


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("fmt", w.FORMATS)
def test_formats(ctx, pinned, fmt, mode):
    for lens, n, window, sinks in (((40, 17, 33), 17, 16, 3), ((300,), 1, 128, 4), ((700, 650), 650, 200, 30)):
        w._run(ctx, fmt, lens, n, window, sinks, mode, seed=n, queries=sorted({0, n // 3, n - 1}))


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 33, 64, 65, 100, 10 ** 12])
@pytest.mark.parametrize("sinks", [0, 1, 16, 17, 33, 64, 250, 10 ** 12])
def test_windows_and_sinks(ctx, pinned, window, sinks, mode):
    for n in (1, 90, 250):
        w._run(ctx, w.FORMATS[0], (250,), n, window, sinks, mode, seed=window % 1000 + sinks % 1000, queries=sorted({0, n // 2, n - 1}))


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("fmt", [w.FORMATS[0], w.FORMATS[4], w.FORMATS[5]])
def test_statistics(ctx, pinned, fmt, mode):
    w._run(ctx, fmt, (333, 270), 70, 50, 3, mode, serial=None)


@pytest.mark.parametrize("fmt", [w.FORMATS[0], w.FORMATS[1], w.FORMATS[5], w.FORMATS[7]])
@pytest.mark.parametrize("T,n,window", [(60, 3, 50), (900, 1, 700), (700, 400, 600)])
def test_every_row_an_event(ctx, pinned, fmt, T, n, window):
    w.test_every_row_an_event(ctx, fmt, T, n, window)


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("n", [4, 200])
def test_past_three_digits_32_bits_and_the_clamp(ctx, pinned, n, mode):
    w.test_long_runs_of_wide_values(ctx, w.FORMATS[5], n, mode)
    w.test_queries_past_three_digits(ctx, n, mode)
    w.test_scores_past_32_bits(ctx, min(n, 150), mode)
    w.test_values_that_clamp(ctx, n, mode)


@pytest.mark.parametrize("n", [1, 300])
def test_unaligned_streams_and_one_sequence(ctx, pinned, n):
    w.test_unaligned_tensors_and_in_place(ctx, n)
    w.test_another_stream_and_its_own(ctx, n)
    w.test_one_sequence_of_a_batch(ctx, min(n, 200))


@pytest.mark.parametrize("mode", ["online", "two_pass"])
def test_more_tiles_than_a_launch(ctx, pinned, mode):
    """2 KV heads x 600 tiles of 16 rows: the few queries' kernel in two launches, its scratch used twice."""
    rng = np.random.default_rng(0)
    n = 2400
    w._run(ctx, w.FORMATS[0], (n + 3,), n, 90, 5, mode, queries=sorted({0, 5, 2047, 2048, 2049, n - 1} | set(rng.integers(0, n, 8).tolist())))


@pytest.mark.parametrize("mode", ["online", "two_pass"])
def test_a_batch_of_decode_tokens_past_a_launch(ctx, mode):
    """600 sequences x 2 KV heads of one tile each, lengths 1 to 60."""
    lens = [1 + i * 7 % 60 for i in range(600)]
    w._run(ctx, w.FORMATS[0], lens, 1, 9, 2, mode)


def test_the_rule_at_its_edges(ctx):
    """Calls just inside and outside what either kernel is chosen for: the same integers."""
    from insitu_amd import _lib
    from insitu_amd.attention import CompressedAttention
    rng = np.random.default_rng(1)
    c = w._cache(ctx, w.FORMATS[0], [4200])
    w._fill(c, w.FORMATS[0], [4200], *(w._draw(rng, 65536, 1, 4200, w.N_KV, 64) for _ in "kv"))
    a = CompressedAttention(c)
    for n, window in ((1024, 100), (1025, 100), (1024, 1024), (1025, 1023), (2048, 1024), (2049, 1024)):
        q = w._draw(rng, 1 << 14, n, w.N_KV * 4, 64)
        got = []
        for kernel in (0, FEW, PROMPTS):
            _lib.check(ctx.lib.insitu_cache_debug(c.handle, _lib.DEBUG_WINDOW, kernel))
            out, st = a.attend_window(q, window, 4)
            got.append((out.cpu().numpy(), st.rescale_events, st.max_abs_score, st.max_abs_acc, st.n_tokens))
        for other in got[1:]:
            np.testing.assert_array_equal(other[0], got[0][0])
            assert other[1:] == got[0][1:]


def test_more_rows_than_the_prompts_kernel_counts(ctx):
    """A capacity past 2^27 rows (8.6 GB of 1 KV head): the few queries' kernel takes calls of any size."""
    from insitu_amd import QuantConfig, _lib
    from insitu_amd.attention import CompressedAttention
    from insitu_amd.cache import CompressedCache
    rng = np.random.default_rng(2)
    n, G = 2100, 8
    big, small = (CompressedCache(1, 64, cap, QuantConfig(key_bits=4, value_bits=2), n_q_heads=G, ctx=ctx)
                  for cap in ((1 << 27) + 8, n))
    with pytest.raises(ValueError):
        _lib.check(ctx.lib.insitu_cache_debug(big.handle, _lib.DEBUG_WINDOW, PROMPTS))
    k, v = (w._draw(rng, 65536, n, 1, 64) for _ in "kv")
    q = w._draw(rng, 1 << 14, n, G, 64)
    outs = []
    for c in (big, small):
        c.append_rotated(k, v)
        outs.append(CompressedAttention(c).attend_window(q, 150, 4, stats=False)[0].cpu().numpy())
    np.testing.assert_array_equal(*outs)


def test_pinning_refusals(ctx):
    from insitu_amd import _lib
    c = w._cache(ctx, (64, 8, 8, 2), [5])
    for value in (FEW, PROMPTS, 3, -1):
        with pytest.raises(ValueError):
            _lib.check(ctx.lib.insitu_cache_debug(c.handle, _lib.DEBUG_WINDOW, value))
