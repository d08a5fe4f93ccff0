"""GPU: attends of a sliding window with first rows that stay visible (attend_window.hip): every query against
oracle/c over the rows it sees. Windows from one row to more than there is, around tiles of 16 rows; sinks from
none to overlapping the window; decode steps, chunks and prompts; every group, key and value width; ragged
batches and single sequences of one; peaked and flat weights; events in every row; rows that need the
token-by-token path; formats that only it takes; streams, graphs, repeated calls and refusals. All results are
integers: equality."""

import numpy as np
import pytest

from oracle import native
from oracle.quantize import Cache, CompressedKV, Format

pytestmark = pytest.mark.gpu

N_KV = 2
FORMATS = [(64, 4, 2, 4), (64, 3, 2, 8), (64, 2, 3, 1), (64, 4, 1, 5), (64, 3, 3, 3), (128, 3, 3, 4), (128, 4, 2, 2),
           (128, 2, 1, 8)]


def _draw(rng, scale, *shape):
    return np.rint(rng.standard_normal(shape) * scale).astype(np.int64)


def _cache(ctx, fmt, lens, room=2, **kw):
    from insitu_amd import QuantConfig
    from insitu_amd.cache import CompressedCache
    d, kb, vb, G = fmt
    return CompressedCache(N_KV, d, max(lens) + room, QuantConfig(key_bits=kb, value_bits=vb), batch=len(lens),
                           n_q_heads=N_KV * G, ctx=ctx, **kw)


def _fill(c, fmt, lens, k, v):
    """Sequence b holds the first lens[b] rows of k, v (batch, rows, N_KV, d), on the device and the host."""
    d, kb, vb, _ = fmt
    f = Format(d=d, key_bits=kb, value_bits=vb)
    hosts = []
    for b, n in enumerate(lens):
        c.append_rotated(k[b, :n], v[b, :n], seq=b)
        host = Cache(N_KV, n, f)
        host.append_rotated(k[b, :n], v[b, :n])
        hosts.append(host)
    return hosts, f


def _seen(p, window, sinks):
    """The rows that the query at row p attends."""
    t = np.arange(p + 1)
    return t[(t < sinks) | (t > p - window)]


def _check(out, st, q, hosts, f, G, lens, n, window, sinks, mode, serial=0, queries=None):
    """out (sequences, n, heads, d). queries: those to look at (all), and then no statistics."""
    attend = native.attend_two_pass if mode == "two_pass" else native.attend_online
    sts = []
    for b, T in enumerate(lens):
        views = [hosts[b].view(h) for h in range(N_KV)]
        for i in range(n) if queries is None else queries:
            idx = _seen(T - n + i, window, sinks)
            for h, kv in enumerate(views):
                sl = slice(G * h, G * h + G)
                want, s = attend(q[b, i, sl], CompressedKV(kv.k_idx[idx], kv.k_norm[idx], kv.v_idx[idx], kv.v_norm[idx]), f)
                np.testing.assert_array_equal(out[b, i, sl], want, err_msg=f"sequence {b} query {i} head {h}")
                sts.append(s)
    if st is None or queries is not None:
        return
    assert st.n_tokens == max(s.n_tokens for s in sts)
    assert st.max_abs_score == max(s.max_abs_score for s in sts)
    assert st.max_abs_acc == max(s.max_abs_acc for s in sts)
    assert st.acc_overflows == sum(s.acc_overflows for s in sts)
    assert st.rescale_events == sum(s.rescale_events for s in sts)
    assert st.score_overflows == 0
    if serial is not None:
        assert st.serial_fallbacks == serial


def _run(ctx, fmt, lens, n, window, sinks, mode, q_scale=1 << 14, seed=0, serial=0, queries=None, kv_scale=65536, k=None,
         v=None, q=None):
    from insitu_amd.attention import CompressedAttention
    d, _, _, G = fmt
    rng = np.random.default_rng(seed)
    c = _cache(ctx, fmt, lens)
    k = _draw(rng, kv_scale, len(lens), max(lens), N_KV, d) if k is None else k
    v = _draw(rng, kv_scale, len(lens), max(lens), N_KV, d) if v is None else v
    hosts, f = _fill(c, fmt, lens, k, v)
    q = _draw(rng, q_scale, len(lens), n, N_KV * G, d) if q is None else q
    out, st = CompressedAttention(c).attend_window(q, window, sinks, mode)
    _check(out.cpu().numpy(), st, q, hosts, f, G, lens, n, window, sinks, mode, serial, queries)
    return c, st


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens,n,window,sinks", [((1,), 1, 1, 0), ((300,), 1, 128, 4), ((40, 17, 33), 17, 16, 3),
                                                 ((95, 130, 6), 5, 60, 20)])
def test_formats(ctx, fmt, lens, n, window, sinks, mode):
    for q_scale in (1 << 13, 1 << 17):
        _run(ctx, fmt, lens, n, window, sinks, mode, q_scale, seed=n)


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 31, 63, 64, 100, 250, 251, 10 ** 12])
@pytest.mark.parametrize("sinks", [0, 1, 16, 17, 64, 250, 10 ** 12])
def test_windows_and_sinks(ctx, window, sinks, mode):
    """One query and a few, in a context of 250 rows."""
    for n in (1, 4, 7):
        _run(ctx, FORMATS[0], (250,), n, window, sinks, mode, seed=window % 1000 + sinks % 1000)


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("fmt", [FORMATS[0], FORMATS[1], FORMATS[5]])
@pytest.mark.parametrize("n", [1, 2, 3, 16, 100])
@pytest.mark.parametrize("window,sinks", [(1024, 4), (700, 0), (2000, 70)])
def test_long_contexts(ctx, fmt, n, window, sinks, mode):
    """Flat weights (every token counts), a model's, and peaked ones, behind thousands of rows, ragged."""
    for q_scale in (1 << 10, 1 << 14, 1 << 17):
        _run(ctx, fmt, (4100, 137, 2500), n, window, sinks, mode, q_scale, queries=sorted({0, n // 2, n - 1}))


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("fmt", [FORMATS[0], FORMATS[1], FORMATS[4], FORMATS[6]])
@pytest.mark.parametrize("n,window,sinks", [(600, 100, 4), (513, 1, 0), (700, 64, 100), (1000, 10 ** 6, 0)])
def test_prompts(ctx, fmt, n, window, sinks, mode):
    """Prompts from an empty cache and behind a few rows."""
    rng = np.random.default_rng(n)
    look = sorted({0, 1, 15, 16, 63, 64, n - 17, n - 1} | set(rng.integers(0, n, 8).tolist()))
    _run(ctx, fmt, (n, n + 37), n, window, sinks, mode, queries=look)


@pytest.mark.parametrize("mode", ["online", "two_pass"])
def test_a_prompts_statistics(ctx, mode):
    _run(ctx, FORMATS[0], (333,), 333, 50, 3, mode, serial=None)


def test_a_window_of_everything_is_a_prompt(ctx):
    from insitu_amd.attention import CompressedAttention
    fmt, n, T = FORMATS[0], 40, 700
    rng = np.random.default_rng(5)
    c = _cache(ctx, fmt, [T])
    _fill(c, fmt, [T], *(_draw(rng, 65536, 1, T, N_KV, 64) for _ in "kv"))
    q = _draw(rng, 1 << 14, n, N_KV * 4, 64)
    a = CompressedAttention(c)
    for mode in ("online", "two_pass", "split", "serial"):
        got, st = a.attend_window(q, T, mode=mode)
        assert got.shape == (n, N_KV * 4, 64)
        want, st2 = a.attend_prefill(q, T - n, "online" if mode == "split" else mode)
        np.testing.assert_array_equal(got.cpu().numpy(), want.cpu().numpy())
        assert st.max_abs_score == st2.max_abs_score and st.n_tokens == st2.n_tokens == T


@pytest.mark.parametrize("n", [1, 5, 200])
def test_one_sequence_of_a_batch(ctx, n):
    from insitu_amd.attention import CompressedAttention
    fmt, lens = FORMATS[1], [400, 250, 333]
    rng = np.random.default_rng(n)
    c = _cache(ctx, fmt, lens)
    hosts, f = _fill(c, fmt, lens, *(_draw(rng, 65536, 3, 400, N_KV, 64) for _ in "kv"))
    q = _draw(rng, 1 << 14, 1, n, N_KV * 8, 64)
    for b in range(3):
        for mode in ("online", "two_pass"):
            out, st = CompressedAttention(c).attend_window(q[0], 70, 5, mode, seq=b)
            _check(out.cpu().numpy()[None], st, q, [hosts[b]], f, 8, [lens[b]], n, 70, 5, mode)


def _rising(d, T, step):
    """Keys along one direction, longer and longer: every score of a query along it is an event."""
    u = np.where(np.arange(d) % 3 == 0, -65536.0, 65536.0)
    k = u * (0.25 + step * np.arange(T))[:, None]
    return np.rint(np.stack([k] * N_KV, 1)[None]).astype(np.int64), u


@pytest.mark.parametrize("fmt", [FORMATS[0], FORMATS[1], FORMATS[5], FORMATS[7]])
@pytest.mark.parametrize("T,n,window", [(60, 3, 50), (900, 3, 800), (900, 1, 700), (700, 400, 600), (2500, 1, 2000)])
def test_every_row_an_event(ctx, fmt, T, n, window):
    """Events in every row: all that a kernel holds, and more."""
    d, _, _, G = fmt
    rng = np.random.default_rng(1)
    k, u = _rising(d, T, 0.02)
    q = np.rint(np.broadcast_to(u / 32, (1, n, N_KV * G, d))).astype(np.int64)
    v = _draw(rng, 65536, 1, T, N_KV, d)
    _run(ctx, fmt, (T,), n, window, 6, "online", serial=None, k=k, v=v, q=q, queries=sorted({0, n // 2, n - 1}))


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("fmt", [FORMATS[1], FORMATS[5]])
@pytest.mark.parametrize("n", [1, 200])
def test_long_runs_of_wide_values(ctx, fmt, n, mode):
    """Flat weights over thousands of tokens, values of norm 40: a term is up to 20480 x 32768 x 70498 / 2^23
    = 5.6 M, so that 384 of them could pass 2^31."""
    d, _, _, G = fmt
    _, st = _run(ctx, fmt, (5600, 3000), n, 4000, 4, mode, q_scale=1 << 4, queries=sorted({0, n // 2, n - 1}), serial=None,
                 kv_scale=40 / d ** 0.5 * 65536)
    assert st.acc_overflows == 0


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("n", [4, 300])
def test_queries_past_three_digits(ctx, n, mode):
    """Values of 2^23 and more, up to the seam's range and beyond it (range errors)."""
    rng = np.random.default_rng(2)
    q = _draw(rng, 1 << 14, 1, n, N_KV * 4, 64)
    q[0, 1, 2, 7] = (1 << 23) + 5
    q[0, 2, 5, 63] = -(1 << 26)
    q[0, 3, 0, 0] = 0x7F7F7F
    _run(ctx, FORMATS[0], (430,), n, 90, 3, mode, serial=None, q=q)
    q[0, 0, 1, 1] = 1 << 27
    _, st = _run(ctx, FORMATS[0], (430,), n, 90, 3, mode, serial=None, q=q)
    assert st.range_errors == 1


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("n", [3, 150])
def test_scores_past_32_bits(ctx, n, mode):
    """Long queries against long keys: scores that only int64 holds."""
    T = 190
    rng = np.random.default_rng(3)
    k = _draw(rng, 40 * 65536, 1, T, N_KV, 128).clip(-(1 << 23), (1 << 23) - 1)
    q = _draw(rng, 40 * 65536, 1, n, N_KV * 4, 128).clip(-0x7F7F7F, 0x7F7F7F)
    _, st = _run(ctx, FORMATS[5], (T,), n, 77, 2, mode, serial=None, k=k, q=q)
    assert st.max_abs_score > 1 << 31


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("n", [1, 3, 150])
def test_values_that_clamp(ctx, n, mode):
    """Sums past 2^31: online they clamp after every token, two-pass once, at the end."""
    T = 3000
    rng = np.random.default_rng(4)
    v = np.abs(_draw(rng, 50 * 65536, 1, T, N_KV, 64)).clip(0, (1 << 23) - 1)
    _, st = _run(ctx, FORMATS[0], (T,), n, 2600, 9, mode, q_scale=1 << 6, serial=None, v=v, queries=[0, n - 1])
    assert st.acc_overflows > 0


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("kb,vb", [(5, 2), (4, 4), (1, 1), (8, 8)])
def test_other_widths_go_token_by_token(ctx, kb, vb, mode):
    _run(ctx, (64, kb, vb, 2), (120, 63), 6, 37, 5, mode, serial=0)


def test_serial_mode(ctx):
    from insitu_amd.attention import CompressedAttention
    fmt, n, T = FORMATS[5], 9, 450
    rng = np.random.default_rng(6)
    c = _cache(ctx, fmt, [T])
    hosts, f = _fill(c, fmt, [T], *(_draw(rng, 65536, 1, T, N_KV, 128) for _ in "kv"))
    q = _draw(rng, 1 << 14, n, N_KV * 4, 128)
    out, st = CompressedAttention(c).attend_window(q, 130, 70, "serial")
    _check(out.cpu().numpy()[None], st, q[None], hosts, f, 4, [T], n, 130, 70, "online")


@pytest.mark.parametrize("n", [1, 11, 300])
def test_unaligned_tensors_and_in_place(ctx, n):
    """Queries and outputs 4 bytes behind a boundary; outputs over the queries; rows behind the last left alone."""
    import torch
    from insitu_amd.attention import CompressedAttention
    fmt, T = FORMATS[5], 400
    rng = np.random.default_rng(17)
    c = _cache(ctx, fmt, [T, T - 30])
    _fill(c, fmt, [T, T - 30], *(_draw(rng, 65536, 2, T, N_KV, 128) for _ in "kv"))
    q = torch.from_numpy(_draw(rng, 1 << 14, 2, n, N_KV * 4, 128).astype(np.int32)).to(ctx.torch_device)
    q[1, n // 2, 2, 5] = (1 << 23) + 9                  # (a row of the token-by-token path)
    a = CompressedAttention(c)

    def behind(t):
        b = torch.full((t.numel() + 2,), 77, dtype=t.dtype, device=t.device)
        return b, b[1:-1].view(t.shape).copy_(t)
    for mode in ("online", "two_pass", "serial"):
        want = a.attend_window(q, 100, 20, mode, stats=False)[0]
        whole, out = behind(torch.zeros_like(q))
        assert a.attend_window(behind(q)[1], 100, 20, mode, out=out, stats=False)[0] is out and torch.equal(out, want)
        assert int(whole[0]) == 77 == int(whole[-1])
        x = q.clone()
        assert torch.equal(a.attend_window(x, 100, 20, mode, out=x, stats=False)[0], want)


def test_repeated_and_other_shapes_between(ctx):
    """The scratch is shared by calls of all shapes: results do not depend on what ran before."""
    from insitu_amd.attention import CompressedAttention
    fmt, T = FORMATS[0], 2000
    rng = np.random.default_rng(8)
    c = _cache(ctx, fmt, [T, 900])
    _fill(c, fmt, [T, 900], *(_draw(rng, 65536, 2, T, N_KV, 64) for _ in "kv"))
    a = CompressedAttention(c)
    calls = [(n, w, mode, _draw(rng, s, 2, n, N_KV * 4, 64))
             for n, w, mode, s in ((5, 90, "online", 1 << 14), (64, 700, "two_pass", 1 << 17), (1, 1500, "online", 1 << 10),
                                   (333, 100, "online", 1 << 17), (1, 64, "two_pass", 1 << 14))]
    first = [a.attend_window(q, w, 4, mode, stats=False)[0].cpu().numpy() for n, w, mode, q in calls]
    tree = a.attend_tree(calls[0][3], np.arange(5) - 1, stats=False)[0].cpu().numpy()
    for _ in range(2):
        for (n, w, mode, q), want in zip(calls[::-1], first[::-1]):
            np.testing.assert_array_equal(a.attend_window(q, w, 4, mode, stats=False)[0].cpu().numpy(), want)
        np.testing.assert_array_equal(a.attend_tree(calls[0][3], np.arange(5) - 1, stats=False)[0].cpu().numpy(), tree)


@pytest.mark.parametrize("n", [1, 16, 256])
def test_another_stream_and_its_own(ctx, n):
    """Inputs made on a stream that is not the context's, outputs used there, no synchronisation between."""
    import torch
    from insitu_amd.attention import CompressedAttention
    fmt, T = FORMATS[0], 1500
    rng = np.random.default_rng(9)
    c = _cache(ctx, fmt, [T])
    _fill(c, fmt, [T], *(_draw(rng, 65536, 1, T, N_KV, 64) for _ in "kv"))
    q = torch.from_numpy(_draw(rng, 1 << 14, n, N_KV * 4, 64).astype(np.int32)).to(ctx.torch_device)
    a = CompressedAttention(c)
    want = a.attend_window(q, 500, 4, stats=False)[0].clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream(ctx.torch_device)
    with torch.cuda.stream(side):
        big = torch.randn(2048, 2048, device=ctx.torch_device)
        for _ in range(20):
            big = big @ big * 1e-3                      # the queries come late
        q2 = q + (big[0, 0] * 0).to(torch.int32)
        got = a.attend_window(q2, 500, 4, stats=False)[0] + 0
    side.synchronize()
    assert torch.equal(got, want)


def test_captured_and_replayed(ctx):
    """Calls of several shapes in one graph, on a context of the capturing stream, replayed with new queries and
    with lengths that changed since, eager calls of the same cache between."""
    import torch
    from insitu_amd.attention import CompressedAttention
    from insitu_amd.runtime import Context
    fmt, T = FORMATS[0], 3000
    side = torch.cuda.Stream(ctx.torch_device)
    own = Context(ctx.device, stream=side)
    rng = np.random.default_rng(10)
    shapes = [(1, 128, 4, "online"), (1, 2000, 4, "online"), (1, 900, 0, "two_pass"), (40, 700, 20, "online"),
              (300, 100, 3, "two_pass"), (2, 50, 1, "serial")]
    with torch.cuda.stream(side):
        c = _cache(own, fmt, [T], room=100)
        _fill(c, fmt, [T], *(_draw(rng, 65536, 1, T, N_KV, 64) for _ in "kv"))
        c.set_length(400)
        a = CompressedAttention(c)
        qs = [torch.zeros((n, N_KV * 4, 64), dtype=torch.int32, device=own.torch_device) for n, *_ in shapes]
        outs = [torch.zeros_like(q) for q in qs]

        def all_of(qs, outs):
            for q, o, (n, w, s, mode) in zip(qs, outs, shapes):
                a.attend_window(q, w, s, mode, out=o, stats=False)
        all_of(qs, outs)                                # (the scratch is allocated before the capture)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            all_of(qs, outs)
        for r, now in enumerate((400, 1000, 3000, 2345, 300, 2999)):
            c.set_length(now)
            new = [torch.from_numpy(_draw(rng, 1 << 14, *q.shape).astype(np.int32)).to(own.torch_device) for q in qs]
            for q, x in zip(qs, new):
                q.copy_(x)
            for o in outs:
                o.zero_()
            g.replay()
            got = [o.clone() for o in outs]
            side.synchronize()
            eager = [torch.zeros_like(q) for q in qs]
            all_of(new, eager)
            side.synchronize()
            for i, (x, y) in enumerate(zip(got, eager)):
                assert torch.equal(x, y), f"replay {r} call {shapes[i]}"


def test_captured_without_scratch(ctx):
    """A capture allocates nothing: a call whose scratch is not there yet says so."""
    import torch
    from insitu_amd import _lib
    from insitu_amd.attention import CompressedAttention
    from insitu_amd.runtime import Context
    side = torch.cuda.Stream(ctx.torch_device)
    own = Context(ctx.device, stream=side)
    rng = np.random.default_rng(14)
    with torch.cuda.stream(side):
        c = _cache(own, FORMATS[0], [900])
        _fill(c, FORMATS[0], [900], *(_draw(rng, 65536, 1, 900, N_KV, 64) for _ in "kv"))
        a = CompressedAttention(c)
        q = torch.from_numpy(_draw(rng, 1 << 14, 3, N_KV * 4, 64).astype(np.int32)).to(own.torch_device)
        out = torch.zeros_like(q)
        side.synchronize()
        with pytest.raises(_lib.InsituError, match="before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                a.attend_window(q, 700, 4, out=out, stats=False)
        want = a.attend_window(q, 700, 4, stats=False)[0]
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            a.attend_window(q, 700, 4, out=out, stats=False)
        for _ in range(3):
            out.zero_()
            g.replay()
            side.synchronize()
            assert torch.equal(out, want)


def test_refusals(ctx):
    import torch
    from insitu_amd import _lib
    from insitu_amd.attention import CompressedAttention
    c = _cache(ctx, FORMATS[0], [20, 9])
    rng = np.random.default_rng(0)
    _fill(c, FORMATS[0], [20, 9], *(_draw(rng, 65536, 2, 20, N_KV, 64) for _ in "kv"))
    a = CompressedAttention(c)
    q = np.zeros((2, 3, N_KV * 4, 64), dtype=np.int32)
    for bad in (dict(window=0), dict(window=-5), dict(window=4, sinks=-1), dict(window=4, seq=2), dict(window=4, seq=-1),
                dict(window=1 << 70)):
        with pytest.raises(ValueError):
            a.attend_window(q if "seq" not in bad else q[0], **bad)
    with pytest.raises(TypeError):
        a.attend_window(q, 2.5)
    for shape in ((2, 3, 8, 32), (3, 3, 8, 64), (2, 3, 4, 64), (3, 8, 64), (2, 8, 64), (2, 1, 3, 8, 64)):
        with pytest.raises(ValueError):
            a.attend_window(np.zeros(shape, dtype=np.int32), 4)
    with pytest.raises(ValueError):
        a.attend_window(q, 4, seq=0)
    with pytest.raises(_lib.InsituError):               # more queries than rows
        a.attend_window(np.zeros((2, 10, 8, 64), dtype=np.int32), 4)
    with pytest.raises(_lib.InsituError):               # no query
        a.attend_window(np.zeros((2, 0, 8, 64), dtype=np.int32), 4)
    with pytest.raises(KeyError):
        a.attend_window(q, 4, mode="sliding")
    dev = ctx.torch_device
    for out in (torch.zeros((2, 3, 8, 64), device=dev), torch.zeros((2, 3, 8, 65), dtype=torch.int32, device=dev)[..., :64],
                torch.zeros((3, 8, 64), dtype=torch.int32, device=dev), torch.zeros((2, 3, 8, 64), dtype=torch.int32)):
        with pytest.raises(ValueError):
            a.attend_window(q, 4, out=out)
    a.attend_window(np.zeros((10, 8, 64), dtype=np.int32), 4, seq=0)
    ctx.sync()
