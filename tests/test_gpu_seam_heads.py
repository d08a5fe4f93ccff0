"""GPU: the seam with norms of queries and keys and the other rotary forms (seam_heads.h) against float64
numpy, value by value. The rows are integers: a value whose exact image lies within the two sides' rounding
of a half may fall either way, so a difference of one is allowed there and nowhere else.

That rounding: float64 arithmetic of at most 2 log2(d) + 16 steps on each side, each off by half an ulp of
what it handles, whose size is at most four times the largest value of the head (a sum of two products, the
norm's weight and the reciprocal's factor included in it): with values below 2^7 in Q16 units of 2^23,
32 steps of 2^-53 on either side are 2^23 * 4 * 64 * 2^-53 = 2^-22. Far below it the test's 1e-6 (2^-20)."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

NEAR_HALF = 1e-6


def _exact(p, pos, cos, sin, n_q, n_kv, d, rotary, interleaved, wq, wk, bias, eps, cast_after):
    """Q16 images in float64 before the rounding (cast_after), or the rows themselves (integer rotation)."""
    x = p if bias is None else p + bias
    x = x.astype(np.float64).reshape(len(p), -1, d)
    out = []
    half = rotary // 2
    lo = 2 * np.arange(half) if interleaved else np.arange(half)
    hi = lo + 1 if interleaved else lo + half
    c, s = cos[pos][:, None].astype(np.float64), sin[pos][:, None].astype(np.float64)
    for kind, (a, b, w) in enumerate(((0, n_q, wq), (n_q, n_q + n_kv, wk), (n_q + n_kv, n_q + 2 * n_kv, None))):
        y = x[:, a:b].copy()
        if w is not None:
            y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
        if kind == 0:
            y = y * (1.0 / np.sqrt(d))
        if not cast_after:
            y = np.clip(np.rint(y * 65536), -(1 << 23), (1 << 23) - 1)
        if kind < 2:
            u, v = y[..., lo].copy(), y[..., hi].copy()
            if cast_after:
                y[..., lo], y[..., hi] = (u * c - v * s) / 32768, (u * s + v * c) / 32768
            else:
                u, v, ci, si = (t.astype(np.int64) for t in (u, v, c, s))
                y[..., lo], y[..., hi] = (u * ci - v * si) >> 15, (u * si + v * ci) >> 15
        out.append(y * 65536 if cast_after else y)
    return out


def _check(got, want, cast_after, near=NEAR_HALF):
    for g, w in zip(got, want):
        g = g.cpu().numpy().astype(np.int64)
        r = np.clip(np.rint(w), -(1 << 23), (1 << 23) - 1).astype(np.int64) if cast_after else w.astype(np.int64)
        off = g != r
        if off.any():
            assert cast_after, "the cast's neighbours differ in an integer rotation"
            assert np.abs(g - r).max() <= 1
            assert (np.abs(np.abs(w[off] - np.floor(w[off])) - 0.5) < near).all()


def _case(ctx, d=64, n_q=8, n_kv=2, n=5, rotary=None, interleaved=False, norm="qk", bias=False, cast_after=True, scale=1.0,
          seed=0, scaling=None, pos=None, counts=True):
    from insitu_amd import ModelConfig, Seam
    rotary = rotary or d
    m = ModelConfig(hidden_size=n_q * d, num_heads=n_q, num_kv_heads=n_kv, head_dim=d, rope_theta=10000.0, max_position=512,
                    rotary_dim=rotary, rope_interleaved=interleaved, rope_scaling=scaling, qk_norm_eps=1e-5)
    rng = np.random.default_rng(seed)
    heads = n_q + 2 * n_kv
    p = (rng.standard_normal((n, heads * d)) * scale).astype(np.float32)
    wq = (1 + 0.3 * rng.standard_normal(d)).astype(np.float32) if "q" in norm else None
    wk = (1 + 0.3 * rng.standard_normal(d)).astype(np.float32) if "k" in norm else None
    b = (0.3 * rng.standard_normal(heads * d)).astype(np.float32) if bias else None
    pos = rng.integers(0, 512, n) if pos is None else pos
    s = Seam(m, q_norm=wq, k_norm=wk, bias=b, cast_after_rope=cast_after, ctx=ctx)
    got = s.wire(p, pos, counts=counts)
    where = np.arange(pos, pos + n) if np.ndim(pos) == 0 else np.asarray(pos)
    want = _exact(p, where, s._cos.cpu().numpy(), s._sin.cpu().numpy(), n_q, n_kv, d, rotary, interleaved, wq, wk, b, 1e-5,
                  cast_after)
    _check(got, want, cast_after)
    return s, got


@pytest.mark.parametrize("d,rotary", [(64, 64), (64, 32), (64, 8), (128, 128), (128, 32), (64, 6), (128, 126), (16, 16),
                                      (32, 8), (16, 2)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("cast_after", [True, False])
def test_forms(ctx, d, rotary, interleaved, cast_after):
    for norm, bias in (("qk", False), ("", True)):
        _case(ctx, d=d, rotary=rotary, interleaved=interleaved, norm=norm, bias=bias, cast_after=cast_after, seed=rotary)


@pytest.mark.parametrize("n", [1, 2, 3, 17, 100, 1027])
@pytest.mark.parametrize("n_q,n_kv", [(32, 8), (3, 1), (7, 7), (1, 1)])
def test_tokens_and_heads(ctx, n, n_q, n_kv):
    _case(ctx, n=n, n_q=n_q, n_kv=n_kv, seed=n)
    _case(ctx, n=n, n_q=n_q, n_kv=n_kv, d=128, rotary=64, interleaved=True, bias=True, seed=n + 1)


@pytest.mark.parametrize("norm", ["q", "k"])
def test_one_of_the_norms(ctx, norm):
    _case(ctx, norm=norm, n=40)


@pytest.mark.parametrize("scale", [1e-20, 1e-3, 1e4, 1e15])
def test_sizes_of_values(ctx, scale):
    """Under the norm every size is the same but for eps; values saturate the cast, and zeros stay zeros."""
    s, (q, k, v) = _case(ctx, scale=scale, n=9)
    if scale > 1e3:
        assert s.last_saturated >= int((np.abs(v.cpu().numpy()) >= (1 << 23) - 1).sum()) > 0
    from insitu_amd import ModelConfig, Seam
    m = ModelConfig(hidden_size=256, num_heads=4, num_kv_heads=1, max_position=8)
    z = Seam(m, q_norm=np.ones(64, np.float32), k_norm=np.ones(64, np.float32), ctx=ctx).wire(np.zeros((2, 384), np.float32), 3)
    assert all(int(x.abs().max()) == 0 for x in z)


def test_without_norms_it_is_the_seam(ctx):
    """Bit for bit insitu_seam_wire's rows, in both cast orders, scaled frequencies and biases included."""
    from insitu_amd import HostHalf, ModelConfig, RopeScaling, Seam, Weights
    rng = np.random.default_rng(0)
    m = ModelConfig(hidden_size=256, num_heads=4, num_kv_heads=2, max_position=300, rope_scaling=RopeScaling(32.0, 1.0, 4.0, 64))
    x = rng.standard_normal((70, 256)).astype(np.float32)
    for after in (True, False):
        w = Weights.random(m, np.eye(64), ctx=ctx)
        h = HostHalf(m, w, cast_after_rope=after, ctx=ctx)
        pos = rng.integers(0, 300, 70)
        want = h.wire(x, pos)
        got = Seam(m, cast_after_rope=after, ctx=ctx).wire(h.project_qkv(x), pos)
        for a, b in zip(got, want):
            np.testing.assert_array_equal(a.cpu().numpy(), b.cpu().numpy())


def test_scaled_frequencies(ctx):
    from insitu_amd import LinearScaling, YarnScaling
    _case(ctx, n=60, scaling=YarnScaling(4.0, 128))
    _case(ctx, n=60, scaling=LinearScaling(8.0), rotary=32)


def test_positions(ctx):
    """Any order, the same one twice, a first one alone, device tensors; beyond the table an error, or an
    unwritten row where nothing is checked."""
    import torch
    from insitu_amd import _lib
    _case(ctx, pos=[5, 5, 511, 0, 4])
    _case(ctx, pos=507)
    s, _ = _case(ctx, pos=torch.tensor([3, 1, 4, 1, 5]).numpy())
    dev = lambda x: torch.tensor(x, device=ctx.torch_device)
    p = torch.randn((3, s.width), device=ctx.torch_device)
    a, b = s.wire(p, dev([7, 0, 9])), s.wire(p, [7, 0, 9])
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    for bad in ([0, 1, 512], [-1, 0, 1], 510, -1):
        with pytest.raises(_lib.FormatError):
            s.wire(p, bad)
    with pytest.raises(_lib.FormatError):
        s.wire(p, dev([7, 512, 9]))
    c = s.wire(p, dev([7, 512, 9]), counts=False)
    for x, y in zip(c, a):
        assert torch.equal(x[0], y[0])
    assert torch.equal(c[2], a[2])                      # values have no position
    for bad in ([1, 2], dev([1, 2])):
        with pytest.raises(ValueError):
            s.wire(p, bad)
    with pytest.raises(ValueError):
        s.wire(p[:, :-1], 0)
    assert all(x.shape[0] == 0 for x in s.wire(p[:0], 0))


def test_unaligned_rows(ctx):
    """A projection that is not 16-byte aligned takes single channels a lane."""
    import torch
    from insitu_amd import ModelConfig, Seam
    m = ModelConfig(hidden_size=256, num_heads=4, num_kv_heads=1, max_position=64)
    s = Seam(m, q_norm=np.ones(64, np.float32), k_norm=np.full(64, 0.5, np.float32), ctx=ctx)
    flat = torch.randn(10 * s.width + 1, device=ctx.torch_device)
    p = flat[1:].reshape(10, s.width)
    assert p.data_ptr() % 16 == 4 and p.is_contiguous()
    for a, b in zip(s.wire(p, 3), s.wire(p.clone(), 3)):
        assert torch.equal(a, b)


def test_refusals(ctx):
    from insitu_amd import ModelConfig, Seam
    m = ModelConfig(hidden_size=256, num_heads=4, num_kv_heads=1, max_position=64)
    with pytest.raises(ValueError):
        Seam(m, q_norm=np.ones(32, np.float32), ctx=ctx)
    with pytest.raises(ValueError):
        Seam(m, bias=np.ones(32, np.float32), ctx=ctx)
    for kw in (dict(rotary_dim=65), dict(rotary_dim=0), dict(rotary_dim=66), dict(qk_norm_eps=0.0)):
        with pytest.raises(ValueError):
            ModelConfig(hidden_size=256, num_heads=4, num_kv_heads=1, **kw)


def test_captured_and_replayed(ctx):
    import torch
    from insitu_amd import ModelConfig, Seam
    from insitu_amd.runtime import Context
    m = ModelConfig(hidden_size=256, num_heads=4, num_kv_heads=1, max_position=64)
    side = torch.cuda.Stream(ctx.torch_device)
    own = Context(ctx.device, stream=side)
    with torch.cuda.stream(side):
        s = Seam(m, q_norm=np.ones(64, np.float32), k_norm=np.ones(64, np.float32), ctx=own)
        p = torch.randn((6, s.width), device=ctx.torch_device)
        pos = torch.arange(6, device=ctx.torch_device)
        s.wire(p, pos, counts=False)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = s.wire(p, pos, counts=False)
        for _ in range(3):
            p.copy_(torch.randn_like(p))
            pos.copy_(torch.randint(0, 64, (6,), device=ctx.torch_device))
            g.replay()
            got = [x.clone() for x in out]
            side.synchronize()
            for a, b in zip(got, s.wire(p, pos, counts=False)):
                assert torch.equal(a, b)
            side.synchronize()


def test_refuses_other_tables(ctx):
    import torch
    from insitu_amd import ModelConfig, Seam
    from insitu_amd.host import RoPE
    m = ModelConfig(hidden_size=256, num_heads=4, num_kv_heads=1, max_position=64, rotary_dim=32)
    rope = RoPE.build(32, 64)
    good = [torch.from_numpy(t).to(ctx.torch_device) for t in (rope.cos, rope.sin)]
    assert Seam(m, ctx=ctx, tables=good).wire(np.zeros((2, 384), np.float32), 3)[0].shape == (2, 4, 64)
    short = [t[:63].contiguous() for t in good]
    wide = [torch.from_numpy(t).to(ctx.torch_device) for t in (RoPE.build(64, 64).cos, RoPE.build(64, 64).sin)]
    for bad in (short, wide, (good[0], short[1]), [t.to(torch.int32) for t in good], [t.cpu() for t in good],
                [t.t().contiguous().t() for t in good]):
        with pytest.raises(ValueError, match="tables"):
            Seam(m, ctx=ctx, tables=bad)


def test_on_another_stream(ctx):
    """Projections made late on a stream that is not the context's, rows used there without a synchronisation."""
    import torch
    from insitu_amd import ModelConfig, Seam
    m = ModelConfig(hidden_size=256, num_heads=4, num_kv_heads=1, max_position=64)
    s = Seam(m, q_norm=np.ones(64, np.float32), k_norm=np.ones(64, np.float32), ctx=ctx)
    p = torch.randn((40, s.width), device=ctx.torch_device)
    pos = torch.arange(40, device=ctx.torch_device)
    want = [x.clone() for x in s.wire(p, pos, counts=False)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream(ctx.torch_device)
    with torch.cuda.stream(side):
        big = torch.randn(2048, 2048, device=ctx.torch_device)
        for _ in range(20):
            big = big @ big * 1e-3
        late = p + (big[0, 0] * 0).nan_to_num()
        got = [x + 0 for x in s.wire(late, pos, counts=False)]
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
