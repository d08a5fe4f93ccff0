"""GPU: attends of trees of drafted tokens (attend_tree.hip): every node against oracle/c over the context,
the node's ancestors and itself. Contexts from none to several spans, around tiles of 16 tokens; trees of 1
to 256 nodes, as chains, stars and in between; every group, key and value width; ragged batches; peaked and
flat weights; events in every row; rows that need the token-by-token path; formats that only it takes;
streams, graphs, repeated calls and refusals. All results are integers: equality."""

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


def _tree(kind, n, rng):
    i = np.arange(n)
    if kind == "chain":
        return i - 1
    if kind == "star":
        return np.full(n, -1)
    if kind == "binary":
        return np.maximum((i - 1) // 2, np.where(i > 0, 0, -1))
    return np.array([rng.integers(-1, x) if x else -1 for x in i])


def _path(parents, i):
    p = []
    while i >= 0:
        p.append(i)
        i = int(parents[i])
    return p[::-1]


def _cache(ctx, fmt, lens, **kw):
    from insitu_amd import QuantConfig
    from insitu_amd.cache import CompressedCache
    d, kb, vb, G = fmt
    return CompressedCache(N_KV, d, max(lens) + 2, QuantConfig(key_bits=kb, value_bits=vb), batch=len(lens),
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


def _rows(kv, idx):
    return CompressedKV(kv.k_idx[idx], kv.k_norm[idx], kv.v_idx[idx], kv.v_norm[idx])


def _check(out, st, q, hosts, f, G, lens, parents, n, mode, serial=0, nodes=None):
    """out (batch, n, heads, d); parents (batch, n). nodes: those to look at (all), and then no statistics."""
    attend = native.attend_two_pass if mode == "two_pass" else native.attend_online
    sts = []
    for b, T in enumerate(lens):
        base = T - n
        for i in range(n) if nodes is None else nodes:
            idx = np.concatenate([np.arange(base), base + np.array(_path(parents[b], i))]).astype(np.int64)
            for h in range(N_KV):
                sl = slice(G * h, G * h + G)
                want, s = attend(q[b, i, sl], _rows(hosts[b].view(h), idx), f)
                np.testing.assert_array_equal(out[b, i, sl], want, err_msg=f"sequence {b} node {i} head {h}")
                sts.append(s)
    if st is None or nodes is not None:
        return
    assert st.n_tokens == max(lens)
    assert st.max_abs_score == max(s.max_abs_score for s in sts)
    assert st.max_abs_acc == max(s.max_abs_acc for s in sts)
    assert st.acc_overflows == sum(s.acc_overflows for s in sts)
    assert st.rescale_events == sum(s.rescale_events for s in sts)
    assert st.score_overflows == 0
    if serial is not None:
        assert st.serial_fallbacks == serial


def _run(ctx, fmt, bases, n, kind, mode, q_scale=1 << 14, seed=0, serial=0, nodes=None, kv_scale=65536, k=None, v=None, q=None):
    from insitu_amd.attention import CompressedAttention
    d, _, _, G = fmt
    rng = np.random.default_rng(seed)
    lens = [x + n for x in bases]
    c = _cache(ctx, fmt, lens)
    k = _draw(rng, kv_scale, len(lens), max(lens), N_KV, d) if k is None else k
    v = _draw(rng, kv_scale, len(lens), max(lens), N_KV, d) if v is None else v
    hosts, f = _fill(c, fmt, lens, k, v)
    q = _draw(rng, q_scale, len(lens), n, N_KV * G, d) if q is None else q
    parents = np.stack([_tree(kind, n, rng) for _ in lens])
    out, st = CompressedAttention(c).attend_tree(q, parents, mode)
    _check(out.cpu().numpy(), st, q, hosts, f, G, lens, parents, n, mode, serial, nodes)
    return c, st


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bases,n", [((0,), 1), ((100,), 5), ((1, 0, 15), 17), ((16, 47, 300), 3)])
def test_formats(ctx, fmt, bases, n, mode):
    for q_scale in (1 << 13, 1 << 17):
        _run(ctx, fmt, bases, n, "random", mode, q_scale, seed=n)


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("kind", ["chain", "star", "binary", "random"])
@pytest.mark.parametrize("base,n", [(0, 33), (31, 32), (63, 64), (5, 65), (200, 100)])
def test_trees(ctx, kind, base, n, mode):
    _run(ctx, FORMATS[0], (base,), n, kind, mode, seed=base + n)


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("kind", ["chain", "random", "star"])
def test_largest_tree(ctx, kind, mode):
    _run(ctx, FORMATS[0], (77,), 256, kind, mode, nodes=[0, 1, 31, 32, 63, 64, 127, 128, 200, 254, 255])


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("fmt", [FORMATS[0], FORMATS[1], FORMATS[5]])
@pytest.mark.parametrize("q_scale", [1 << 10, 1 << 14, 1 << 17])
def test_long_contexts(ctx, fmt, q_scale, mode):
    """Many spans, ragged: flat weights (every token counts), a model's, and peaked ones."""
    _run(ctx, fmt, (4100, 37, 2500), 7, "random", mode, q_scale)


@pytest.mark.parametrize("mode", ["online", "two_pass"])
def test_context_of_the_benchmark(ctx, mode):
    _run(ctx, FORMATS[0], (32768 - 4,), 6, "binary", mode, 1 << 16)


def test_a_chain_is_a_prompts_last_tokens(ctx):
    from insitu_amd.attention import CompressedAttention
    fmt, n, T = FORMATS[0], 40, 700
    rng = np.random.default_rng(5)
    c = _cache(ctx, fmt, [T])
    _fill(c, fmt, [T], *(_draw(rng, 65536, 1, T, N_KV, 64) for _ in "kv"))
    q = _draw(rng, 1 << 14, n, N_KV * 4, 64)
    a = CompressedAttention(c)
    for mode in ("online", "two_pass", "split"):
        tree, _ = a.attend_tree(q, np.arange(n) - 1, mode)
        assert tree.shape == (n, N_KV * 4, 64)
        prompt, _ = a.attend_prefill(q, T - n, "online" if mode == "split" else mode)
        np.testing.assert_array_equal(tree.cpu().numpy(), prompt.cpu().numpy())


def _rising(d, T, step):
    """Keys along one direction, longer and longer: every score of a query along it is an event."""
    u = np.where(np.arange(d) % 3 == 0, -65536.0, 65536.0)
    k = u * (0.25 + step * np.arange(T))[:, None]
    return np.rint(np.stack([k] * N_KV, 1)[None]).astype(np.int64), u


@pytest.mark.parametrize("T,serial", [(60, False), (900, None)])
def test_every_row_an_event(ctx, T, serial):
    """Events in every row: more runs than a tile holds send rows to the token-by-token path."""
    fmt = FORMATS[0]
    rng = np.random.default_rng(1)
    k, u = _rising(64, T, 0.02)
    n = 3
    q = np.rint(np.broadcast_to(u / 32, (1, n, N_KV * 4, 64))).astype(np.int64)
    v = _draw(rng, 65536, 1, T, N_KV, 64)
    _, st = _run(ctx, fmt, (T - n,), n, "chain", "online", serial=None, k=k, v=v, q=q)
    assert st.serial_fallbacks == 0 if serial is False else st.serial_fallbacks > 0


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("fmt", [FORMATS[0], FORMATS[4], FORMATS[5]])
def test_around_the_longest_context_of_one_launch(ctx, fmt, mode):
    """The longest sequence decides between one launch and three: 511 to 514 rows, with shorter ones beside."""
    for rows in (511, 512, 513, 514):
        _run(ctx, fmt, (rows - 5, 60, 0), 5, "random", mode, seed=rows)


@pytest.mark.parametrize("fmt", [FORMATS[0], FORMATS[5]])
def test_every_row_an_event_in_one_launch(ctx, fmt):
    """A context of one launch whose events are more than shared memory and the scratch hold together."""
    d, n, T = fmt[0], 5, 500
    rng = np.random.default_rng(13)
    k, u = _rising(d, T, 0.02)
    q = np.rint(np.broadcast_to(u / 32, (1, n, N_KV * 4, d))).astype(np.int64)
    v = _draw(rng, 65536, 1, T, N_KV, d)
    _, st = _run(ctx, fmt, (T - n,), n, "chain", "online", serial=None, k=k, v=v, q=q)
    assert st.serial_fallbacks > 0


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("fmt", [FORMATS[1], FORMATS[5]])
def test_long_runs_of_wide_values(ctx, fmt, mode):
    """Flat weights over spans of hundreds of tokens, values of norm 40: a term is up to
    20480 x 32768 x 70498 / 2^23 = 5.6 M, so that 384 of them could pass 2^31, and runs end before."""
    d, _, _, G = fmt
    _, st = _run(ctx, fmt, (5600, 3000), 256, "random", mode, q_scale=1 << 4, nodes=[0, 130, 255], serial=None,
                 kv_scale=40 / d ** 0.5 * 65536)
    assert st.serial_fallbacks == 0 and st.acc_overflows == 0


@pytest.mark.parametrize("base", [40, 400])
def test_batches_past_the_scratch(ctx, base):
    """16 sequences of 256 nodes and 16 heads: their runs take several launches, a part of the batch each."""
    _run(ctx, FORMATS[7], tuple(base + i for i in range(16)), 256, "random", "online", nodes=[0, 97, 255])


@pytest.mark.parametrize("mode", ["online", "two_pass"])
def test_queries_past_three_digits(ctx, mode):
    """Values of 2^23 and more, up to the seam's range and beyond it (range errors)."""
    fmt, n = FORMATS[0], 4
    rng = np.random.default_rng(2)
    q = _draw(rng, 1 << 14, 1, n, N_KV * 4, 64)
    q[0, 1, 2, 7] = (1 << 23) + 5
    q[0, 2, 5, 63] = -(1 << 26)
    q[0, 3, 0, 0] = 0x7F7F7F
    _run(ctx, fmt, (130,), n, "random", mode, serial=2, q=q)
    q[0, 0, 1, 1] = 1 << 27
    _, st = _run(ctx, fmt, (130,), n, "random", mode, serial=3, q=q)
    assert st.range_errors == 1


@pytest.mark.parametrize("mode", ["online", "two_pass"])
def test_scores_past_32_bits(ctx, mode):
    """Long queries against long keys: scores that only int64 holds."""
    fmt, n, T = FORMATS[5], 3, 90
    rng = np.random.default_rng(3)
    k = _draw(rng, 40 * 65536, 1, T, N_KV, 128).clip(-(1 << 23), (1 << 23) - 1)
    q = _draw(rng, 40 * 65536, 1, n, N_KV * 4, 128).clip(-0x7F7F7F, 0x7F7F7F)
    _, st = _run(ctx, fmt, (T - n,), n, "random", mode, serial=None, k=k, q=q)
    assert st.max_abs_score > 1 << 31 and st.serial_fallbacks > 0


@pytest.mark.parametrize("mode", ["online", "two_pass"])
def test_values_that_clamp(ctx, mode):
    """Sums past 2^31: online they clamp after every token, two-pass once, at the end."""
    fmt, n, T = FORMATS[0], 3, 3000
    rng = np.random.default_rng(4)
    v = np.abs(_draw(rng, 50 * 65536, 1, T, N_KV, 64)).clip(0, (1 << 23) - 1)
    _, st = _run(ctx, fmt, (T - n,), n, "random", mode, q_scale=1 << 6, serial=None, v=v)
    assert st.acc_overflows > 0


@pytest.mark.parametrize("mode", ["online", "two_pass"])
@pytest.mark.parametrize("kb,vb", [(5, 2), (4, 4), (1, 1), (8, 8)])
def test_other_widths_go_token_by_token(ctx, kb, vb, mode):
    _run(ctx, (64, kb, vb, 2), (20, 3), 6, "random", mode, serial=0)


def test_serial_mode(ctx):
    from insitu_amd.attention import CompressedAttention
    fmt, n, T = FORMATS[5], 9, 150
    rng = np.random.default_rng(6)
    c = _cache(ctx, fmt, [T])
    _fill(c, fmt, [T], *(_draw(rng, 65536, 1, T, N_KV, 128) for _ in "kv"))
    q = _draw(rng, 1 << 14, n, N_KV * 4, 128)
    parents = _tree("random", n, rng)
    a = CompressedAttention(c)
    np.testing.assert_array_equal(a.attend_tree(q, parents, "serial")[0].cpu().numpy(),
                                  a.attend_tree(q, parents, "online")[0].cpu().numpy())


def test_bad_parents_on_the_device_count_as_roots(ctx):
    import torch
    from insitu_amd.attention import CompressedAttention
    fmt, T = FORMATS[0], 300
    rng = np.random.default_rng(7)
    n = 6
    c = _cache(ctx, fmt, [T, T])
    hosts, f = _fill(c, fmt, [T, T], *(_draw(rng, 65536, 2, T, N_KV, 64) for _ in "kv"))
    q = _draw(rng, 1 << 14, 2, n, N_KV * 4, 64)
    bad = torch.tensor([[-1, 0, 2, 1 << 30, -7, 4], [-1, 0, 1, 2, 3, 4]], dtype=torch.int32, device=ctx.torch_device)
    good = np.array([[-1, 0, -1, -1, -1, 4], [-1, 0, 1, 2, 3, 4]])
    for mode in ("online", "serial"):
        out, st = CompressedAttention(c).attend_tree(q, bad, mode)
        _check(out.cpu().numpy(), None, q, hosts, f, 4, [T, T], good, n, "online")
        assert st.range_errors == 3


def test_bad_parents_past_32_bits(ctx):
    """A device tensor of 64-bit numbers: 2^32 + 1 is no node 1."""
    import torch
    from insitu_amd.attention import CompressedAttention
    fmt, T, n = FORMATS[0], 40, 4
    rng = np.random.default_rng(16)
    c = _cache(ctx, fmt, [T])
    hosts, f = _fill(c, fmt, [T], *(_draw(rng, 65536, 1, T, N_KV, 64) for _ in "kv"))
    q = _draw(rng, 1 << 14, 1, n, N_KV * 4, 64)
    bad = torch.tensor([-1, 0, (1 << 32) + 1, -(1 << 32)], device=ctx.torch_device)
    out, st = CompressedAttention(c).attend_tree(q, bad)
    _check(out.cpu().numpy(), None, q, hosts, f, 4, [T], np.array([[-1, 0, -1, -1]]), n, "online")
    assert st.range_errors == 2


@pytest.mark.parametrize("T", [90, 1300])
def test_unaligned_tensors_and_in_place(ctx, T):
    """Queries, parents and outputs 4 bytes behind a boundary; outputs over the queries."""
    import torch
    from insitu_amd.attention import CompressedAttention
    fmt, n = FORMATS[5], 11
    rng = np.random.default_rng(17)
    c = _cache(ctx, fmt, [T, T - 30])
    _fill(c, fmt, [T, T - 30], *(_draw(rng, 65536, 2, T, N_KV, 128) for _ in "kv"))
    q = torch.from_numpy(_draw(rng, 1 << 14, 2, n, N_KV * 4, 128).astype(np.int32)).to(ctx.torch_device)
    q[1, 3, 2, 5] = (1 << 23) + 9                       # (a row of the token-by-token path)
    par = torch.from_numpy(_tree("random", n, rng).astype(np.int32)).to(ctx.torch_device)
    a = CompressedAttention(c)

    def behind(t):
        b = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
        return b.copy_(t)
    for mode in ("online", "two_pass", "serial"):
        want = a.attend_tree(q, par, mode, stats=False)[0]
        out = behind(torch.zeros_like(q))
        assert a.attend_tree(behind(q), behind(par), mode, out=out, stats=False)[0] is out and torch.equal(out, want)
        x = q.clone()
        assert torch.equal(a.attend_tree(x, par, mode, out=x, stats=False)[0], want)


def test_repeated_and_other_shapes_between(ctx):
    """The scratch is shared by calls of all shapes: results do not depend on what ran before."""
    from insitu_amd.attention import CompressedAttention
    fmt, T = FORMATS[0], 2000
    rng = np.random.default_rng(8)
    c = _cache(ctx, fmt, [T, 900])
    _fill(c, fmt, [T, 900], *(_draw(rng, 65536, 2, T, N_KV, 64) for _ in "kv"))
    a = CompressedAttention(c)
    calls = [(n, mode, _draw(rng, s, 2, n, N_KV * 4, 64), _tree("random", n, rng))
             for n, mode, s in ((5, "online", 1 << 14), (64, "two_pass", 1 << 17), (1, "online", 1 << 10), (33, "online", 1 << 17))]
    first = [a.attend_tree(q, p, mode, stats=False)[0].cpu().numpy() for n, mode, q, p in calls]
    for _ in range(2):
        for (n, mode, q, p), want in zip(calls[::-1], first[::-1]):
            np.testing.assert_array_equal(a.attend_tree(q, p, mode, stats=False)[0].cpu().numpy(), want)


def test_another_stream_and_its_own(ctx):
    """Inputs made on a stream that is not the context's, outputs used there, no synchronisation between."""
    import torch
    from insitu_amd.attention import CompressedAttention
    fmt, n, T = FORMATS[0], 16, 1500
    rng = np.random.default_rng(9)
    c = _cache(ctx, fmt, [T])
    _fill(c, fmt, [T], *(_draw(rng, 65536, 1, T, N_KV, 64) for _ in "kv"))
    q = torch.from_numpy(_draw(rng, 1 << 14, n, N_KV * 4, 64).astype(np.int32)).to(ctx.torch_device)
    parents = torch.from_numpy(_tree("random", n, rng).astype(np.int32)).to(ctx.torch_device)
    a = CompressedAttention(c)
    want = a.attend_tree(q, parents, stats=False)[0].clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream(ctx.torch_device)
    with torch.cuda.stream(side):
        big = torch.randn(2048, 2048, device=ctx.torch_device)
        for _ in range(20):
            big = big @ big * 1e-3                      # the queries come late
        q2 = q + (big[0, 0] * 0).to(torch.int32)
        got = a.attend_tree(q2, parents, stats=False)[0] + 0
    side.synchronize()
    assert torch.equal(got, want)


def test_captured_and_replayed(ctx):
    """Two trees of different shapes in one graph, on a context of the capturing stream, replayed with
    new queries and eager calls of the same cache between."""
    import torch
    from insitu_amd.attention import CompressedAttention
    from insitu_amd.runtime import Context
    fmt, T = FORMATS[0], 1200
    side = torch.cuda.Stream(ctx.torch_device)
    own = Context(ctx.device, stream=side)
    rng = np.random.default_rng(10)
    with torch.cuda.stream(side):
        c = _cache(own, fmt, [T])
        _fill(c, fmt, [T], *(_draw(rng, 65536, 1, T, N_KV, 64) for _ in "kv"))
        a = CompressedAttention(c)
        qs = [torch.zeros((n, N_KV * 4, 64), dtype=torch.int32, device=own.torch_device) for n in (6, 40)]
        ps = [torch.from_numpy(_tree("random", n, rng).astype(np.int32)).to(own.torch_device) for n in (6, 40)]
        outs = [torch.zeros_like(q) for q in qs]
        for q, p, o in zip(qs, ps, outs):               # (the scratch is allocated before the capture)
            a.attend_tree(q, p, out=o, stats=False)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            for q, p, o in zip(qs, ps, outs):
                a.attend_tree(q, p, out=o, stats=False)
        for r in range(4):
            new = [torch.from_numpy(_draw(rng, 1 << 14, *q.shape).astype(np.int32)).to(own.torch_device) for q in qs]
            for q, x in zip(qs, new):
                q.copy_(x)
            g.replay()
            got = [o.clone() for o in outs]
            side.synchronize()
            for x, p, o in zip(new, ps, got):
                assert torch.equal(a.attend_tree(x, p, stats=False)[0], o), f"replay {r}"
            side.synchronize()


def test_captured_before_the_scratch_grew(ctx):
    """A graph keeps the scratch that it was captured with; and one captured without any is refused."""
    import torch
    from insitu_amd import _lib
    from insitu_amd.attention import CompressedAttention
    from insitu_amd.runtime import Context
    fmt, T, n = FORMATS[0], 2600, 5
    side = torch.cuda.Stream(ctx.torch_device)
    own = Context(ctx.device, stream=side)
    rng = np.random.default_rng(14)
    dev = own.torch_device
    with torch.cuda.stream(side):
        c = _cache(own, fmt, [T])
        _fill(c, fmt, [T], *(_draw(rng, 65536, 1, T, N_KV, 64) for _ in "kv"))
        a = CompressedAttention(c)
        q = torch.from_numpy(_draw(rng, 1 << 14, n, N_KV * 4, 64).astype(np.int32)).to(dev)
        p = torch.from_numpy(_tree("random", n, rng).astype(np.int32)).to(dev)
        out = torch.zeros_like(q)
        side.synchronize()
        with pytest.raises(_lib.InsituError, match="before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                a.attend_tree(q, p, out=out, stats=False)
        a.attend_tree(q, p, out=out, stats=False)
        side.synchronize()
        want = out.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            a.attend_tree(q, p, out=out, stats=False)
        big = torch.from_numpy(_draw(rng, 1 << 14, 256, N_KV * 4, 64).astype(np.int32)).to(dev)
        large = a.attend_tree(big, np.arange(256) - 1, stats=False)[0].clone()
        filler = [torch.full((1 << 22,), 77, dtype=torch.int32, device=dev) for _ in range(8)]
        for _ in range(3):
            out.zero_()
            g.replay()
            side.synchronize()
            assert torch.equal(out, want)
            assert torch.equal(a.attend_tree(big, np.arange(256) - 1, stats=False)[0], large)
        assert all(bool((x == 77).all()) for x in filler)


@pytest.mark.parametrize("T", [300, 2000])
def test_replayed_after_the_lengths_changed(ctx, T):
    """Shorter sequences are attended as they are, longer ones as far as the captured call's went."""
    import torch
    from insitu_amd.attention import CompressedAttention
    from insitu_amd.runtime import Context
    fmt, n = FORMATS[0], 6
    side = torch.cuda.Stream(ctx.torch_device)
    own = Context(ctx.device, stream=side)
    rng = np.random.default_rng(15)
    dev = own.torch_device
    with torch.cuda.stream(side):
        c = _cache(own, fmt, [2 * T])
        _fill(c, fmt, [2 * T], *(_draw(rng, 65536, 1, 2 * T, N_KV, 64) for _ in "kv"))
        a = CompressedAttention(c)
        q = torch.from_numpy(_draw(rng, 1 << 14, n, N_KV * 4, 64).astype(np.int32)).to(dev)
        p = torch.from_numpy(_tree("random", n, rng).astype(np.int32)).to(dev)
        graphs, want = {}, {}
        for mode in ("online", "two_pass", "serial"):
            out = torch.zeros_like(q)
            for m in (7, T // 2, T):
                c.set_length(m, 0)
                a.attend_tree(q, p, mode, out=out, stats=False)
                side.synchronize()
                want[mode, m] = out.clone()
            graphs[mode] = torch.cuda.CUDAGraph(), out
            with torch.cuda.graph(graphs[mode][0], stream=side):
                a.attend_tree(q, p, mode, out=out, stats=False)
        for now, as_if in ((7, 7), (T // 2, T // 2), (T, T), (T + 1, T), (2 * T, T)):
            c.set_length(now, 0)
            for mode, (g, out) in graphs.items():
                out.zero_()
                g.replay()
                side.synchronize()
                assert torch.equal(out, want[mode, as_if]), (mode, now)


def test_refusals(ctx):
    import torch
    from insitu_amd import _lib
    from insitu_amd.attention import CompressedAttention
    fmt = FORMATS[0]
    c = _cache(ctx, fmt, [20, 4])
    rng = np.random.default_rng(11)
    _fill(c, fmt, [20, 4], *(_draw(rng, 65536, 2, 20, N_KV, 64) for _ in "kv"))
    a = CompressedAttention(c)
    q = lambda n, heads=8, d=64: np.zeros((2, n, heads, d), dtype=np.int32)
    with pytest.raises(_lib.InsituError, match="fewer than"):
        a.attend_tree(q(5), np.arange(5) - 1)
    with pytest.raises(_lib.InsituError, match="1 to 256"):
        a.attend_tree(q(0), np.zeros(0, int))
    for bad in ([0, 0], [-1, 1], [-2, 0], [-1, 5]):
        with pytest.raises(ValueError, match="earlier node"):
            a.attend_tree(q(2), bad)
    for p in (np.zeros((3, 2), int) - 1, [-1], [[-1, 0]]):
        with pytest.raises(ValueError):
            a.attend_tree(q(2), p)
    for x in (q(2, 7), q(2, 8, 32), q(2)[0], np.zeros((2, 8, 64), np.int32)):
        with pytest.raises(ValueError):
            a.attend_tree(x, [-1, 0])
    for out in (torch.empty((2, 2, 8, 64), dtype=torch.int64, device=ctx.torch_device),
                torch.empty((2, 2, 8, 64), dtype=torch.int32),
                torch.empty((2, 2, 64, 8), dtype=torch.int32, device=ctx.torch_device).transpose(2, 3),
                torch.empty((2, 8, 64), dtype=torch.int32, device=ctx.torch_device)):
        with pytest.raises(ValueError, match="out must"):
            a.attend_tree(q(2), [-1, 0], out=out)
    big = _cache(ctx, fmt, [300])
    _fill(big, fmt, [300], *(_draw(rng, 65536, 1, 300, N_KV, 64) for _ in "kv"))
    with pytest.raises(_lib.InsituError, match="1 to 256"):
        CompressedAttention(big).attend_tree(np.zeros((257, 8, 64), np.int32), np.arange(257) - 1)
