"""GPU: drafted tokens through the whole block, as a serving program runs them: projections, norms of
queries and keys, rotary positions at the tree's depths, the rows appended, the tree attended, the taken path
kept, the next turn behind it. The seam's rows are integers of the same projections whichever way they go, so
where those agree, everything below the seam must: outputs, cache bytes and lengths."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

PARENTS = [-1, 0, 0, 1, 1, 2, -1, 6, 3]          # 0-1-3-8, 0-1-4, 0-2-5, 6-7
PATH = [0, 1, 3, 8]


def _model(**kw):
    from insitu_amd import ModelConfig
    return ModelConfig(hidden_size=256, num_heads=8, num_kv_heads=2, head_dim=64, max_position=512, **kw)


def _block(ctx, model, norms=True, batch=1, softmax="online", capacity=200, quant=None, **kw):
    from insitu_amd import AttentionBlock, QuantConfig, Weights
    b = AttentionBlock(model, quant or QuantConfig(key_bits=4, value_bits=2), capacity=capacity, batch=batch, softmax=softmax,
                       ctx=ctx, **kw)
    rng = np.random.default_rng(0)
    w = lambda *s: (rng.standard_normal(s) / 16).astype(np.float32)
    n = lambda: (1 + 0.2 * rng.standard_normal(64)).astype(np.float32)
    b.weights = Weights(w(512, 256), w(128, 256), w(128, 256), w(256, 512), model, b.rotation,
                        q_norm=n() if norms else None, k_norm=n() if norms else None, ctx=ctx)
    return b


def _wire(rng, batch, n, heads, d=64):
    return np.rint(rng.standard_normal((batch, n, heads, d)) * 32768).astype(np.int32)


@pytest.mark.parametrize("softmax", ["online", "two_pass"])
@pytest.mark.parametrize("batch", [1, 3])
@pytest.mark.parametrize("bits", [(4, 2), (3, 2), (5, 4)])
def test_a_draft_is_decode_steps_along_its_paths(ctx, softmax, batch, bits):
    """step_tree's rows against step() on a fork of the context for every path; then accept, and a decode
    step behind it against one behind the steps."""
    from insitu_amd import QuantConfig
    m = _model()
    rng = np.random.default_rng(1)
    mk = lambda: _block(ctx, m, batch=batch, softmax=softmax, quant=QuantConfig(key_bits=bits[0], value_bits=bits[1]))
    tree, line = mk(), mk()
    for blk in (tree, line):
        r = np.random.default_rng(2)
        for _ in range(23):
            blk.step(*(_wire(r, batch, 1, h)[:, 0] for h in (8, 2, 2)))
    n = len(PARENTS)
    q, k, v = _wire(rng, batch, n, 8), _wire(rng, batch, n, 2), _wire(rng, batch, n, 2)
    out = tree.step_tree(q, k, v, PARENTS).cpu().numpy()
    assert tree.cache.lengths() == [23 + n] * batch and tree.last_stats.n_tokens == 23 + n
    for leaf in (8, 4, 5, 7):
        path = []
        i = leaf
        while i >= 0:
            path.insert(0, i)
            i = PARENTS[i]
        for i in path:
            got = line.step(q[:, i], k[:, i], v[:, i]).cpu().numpy()
            np.testing.assert_array_equal(got, out[:, i], err_msg=f"node {i}")
        line.accept(len(path))                       # none of it: back to the context
    for i in PATH:
        line.step(q[:, i], k[:, i], v[:, i])
    tree.accept(n, PATH)
    assert tree.cache.lengths() == line.cache.lengths() == [27] * batch
    for b in range(batch):
        for h in range(2):
            np.testing.assert_array_equal(tree.cache.read_rows(h, 0, 27, b), line.cache.read_rows(h, 0, 27, b))
    nxt = [_wire(rng, batch, 1, h)[:, 0] for h in (8, 2, 2)]
    np.testing.assert_array_equal(tree.step(*nxt).cpu().numpy(), line.step(*nxt).cpu().numpy())


@pytest.mark.parametrize("softmax", ["online", "two_pass"])
@pytest.mark.parametrize("form", [dict(), dict(rotary_dim=32, rope_interleaved=True)])
def test_forward_tree(ctx, softmax, form):
    """Hidden states in and out: the taps of a draft are those of the wire rows attended by step_tree, at
    the context's length plus each node's depth; the next turn goes on behind the accepted path."""
    import torch
    m = _model(**form)
    a, b = _block(ctx, m, softmax=softmax), _block(ctx, m, softmax=softmax)
    rng = np.random.default_rng(3)
    x = lambda n: rng.standard_normal((n, 256)).astype(np.float32)
    prompt, draft, token = x(19), x(len(PARENTS)), x(1)
    ya, _ = a.forward(prompt)
    yb, _ = b.forward(prompt)
    assert torch.equal(ya, yb)
    y, report = a.forward_tree(draft, PARENTS)
    assert y.shape == (len(PARENTS), 256) and report.context == 19 + len(PARENTS) and report.n_tokens == len(PARENTS)
    depth = [0, 1, 1, 2, 2, 2, 0, 1, 3]
    wire = b.host.wire(draft, 19 + np.array(depth))
    for name, t in zip("qkv", wire):
        assert torch.equal(a.taps[f"wire.{name}"], t)
    out = b.step_tree(*(t[None] for t in wire), PARENTS)
    assert torch.equal(out[0], a.taps["out"]) and torch.equal(b.host.output(out[0]), y)
    for blk in (a, b):
        blk.accept(len(PARENTS), PATH)
        assert blk.cache.length == 23
    ya, ra = a.forward(token)
    yb, _ = b.forward(token)
    assert torch.equal(ya, yb) and ra.context == 24


def test_a_draft_on_another_stream(ctx):
    """Hidden states made late on a stream that is not the block's; the outputs used there."""
    import torch
    m = _model()
    a, b = _block(ctx, m), _block(ctx, m)
    rng = np.random.default_rng(6)
    x = torch.from_numpy(rng.standard_normal((len(PARENTS), 256)).astype(np.float32)).to(ctx.torch_device)
    prompt = rng.standard_normal((30, 256)).astype(np.float32)
    for blk in (a, b):
        blk.forward(prompt)
    want = a.forward_tree(x, PARENTS, stats=False)[0]
    rows = [_wire(rng, 1, len(PARENTS), h) for h in (8, 2, 2)]
    rows = [torch.as_tensor(np.asarray(r), dtype=torch.int32).to(ctx.torch_device) for r in rows]
    a.accept(len(PARENTS), PATH)
    want_step = a.step_tree(*rows, PARENTS, stats=False)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(ctx.torch_device)
    with torch.cuda.stream(side):
        big = torch.randn(2048, 2048, device=ctx.torch_device)
        for _ in range(20):
            big = big @ big * 1e-3
        zero = (big[0, 0] * 0).nan_to_num()
        got = b.forward_tree(x + zero, PARENTS, stats=False)[0] + 0
        b.accept(len(PARENTS), PATH)
        got_step = b.step_tree(*(r + zero.to(torch.int32) for r in rows), PARENTS, stats=False) + 0
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(got_step, want_step)


def test_branches_become_sequences(ctx):
    """Two branches of a draft go on as sequences of their own, each as if only its path had been decoded."""
    m = _model()
    blk, ref = _block(ctx, m, batch=3), _block(ctx, m, batch=3)
    rng = np.random.default_rng(4)
    for _ in range(9):
        rows = [_wire(rng, 3, 1, h)[:, 0] for h in (8, 2, 2)]
        blk.step(*rows)
        ref.step(*rows)
    n = len(PARENTS)
    q, k, v = (_wire(rng, 3, n, h) for h in (8, 2, 2))
    blk.step_tree(q, k, v, PARENTS)
    blk.cache.fork(0, [1, 2], n=n, rows=[[0, 1, 3, 8], [6, 7]])
    assert blk.cache.lengths() == [9 + n, 13, 11]
    ref.cache.fork(0, [1, 2])
    for i in (0, 1, 3, 8):
        ref.step(q[:, i], np.repeat(k[:1, i], 3, 0), np.repeat(v[:1, i], 3, 0))
    for h in range(2):
        np.testing.assert_array_equal(blk.cache.read_rows(h, 0, 13, 1), ref.cache.read_rows(h, 0, 13, 1))


def test_step_tree_refuses(ctx):
    m = _model()
    blk = _block(ctx, m, batch=2, capacity=10)
    rng = np.random.default_rng(5)
    w = lambda n: [_wire(rng, 2, n, h) for h in (8, 2, 2)]
    from insitu_amd import _lib
    with pytest.raises(_lib.CapacityError):
        blk.step_tree(*w(11), np.arange(11) - 1)
    with pytest.raises(ValueError):
        blk.step_tree(*w(3), [-1, 0, 2])             # before a row is written
    assert blk.cache.lengths() == [0, 0]
    with pytest.raises(ValueError):
        blk.step_tree(*(t[0] for t in w(3)), [-1, 0, 1])
    with pytest.raises(ValueError):
        blk.forward_tree(np.zeros((2, 256), np.float32), [-1, 0])


def _attention(d, cls=None):
    """A module as the adapter reads it, with norms of queries and keys."""
    import torch
    import torch.nn as nn

    class RMSNorm(nn.Module):
        def __init__(self, plus=0.0):
            super().__init__()
            self.weight = nn.Parameter(1 + 0.1 * torch.randn(d))
            self.variance_epsilon = 1e-6
            self.plus = plus

        def forward(self, x):
            v = x.float()
            return (self.weight + self.plus) * (v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + 1e-6)).to(x.dtype)

    class Attention(nn.Module):
        def __init__(self):
            super().__init__()
            self.q_proj = nn.Linear(256, 8 * d, bias=False)
            self.k_proj = nn.Linear(256, 2 * d, bias=False)
            self.v_proj = nn.Linear(256, 2 * d, bias=False)
            self.o_proj = nn.Linear(8 * d, 256, bias=False)
            self.q_norm, self.k_norm = (cls or RMSNorm)(), (cls or RMSNorm)()

    return Attention(), RMSNorm


_CONFIG = {"hidden_size": 256, "num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 64, "rope_theta": 10000.0,
           "max_position_embeddings": 256, "rms_norm_eps": 1e-6}


def test_adapter_takes_norms_of_queries_and_keys(ctx):
    import torch
    from insitu_amd.adapters.torch_llama import build_from_layer
    torch.manual_seed(0)
    attn, RMSNorm = _attention(64)
    a = build_from_layer(attn, _CONFIG, ctx=ctx)
    x = torch.randn(1, 12, 256)
    y, _ = a(x)
    assert y.shape == x.shape
    # the wire rows are the norm's, the rotation's and the scale's of the block's own projections
    p = a.kernel.host.project_qkv(x[0]).cpu().double().reshape(12, 12, 64)
    q = p[:, :8]
    q = q / (q.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * attn.q_norm.weight.detach().double() / 8.0
    inv = 1.0 / 10000.0 ** (torch.arange(32, dtype=torch.float64) / 32)
    ang = torch.arange(12, dtype=torch.float64)[:, None, None] * inv
    c, s = (torch.round(f(ang) * 32768) / 32768 for f in (torch.cos, torch.sin))
    want = torch.cat([q[..., :32] * c - q[..., 32:] * s, q[..., :32] * s + q[..., 32:] * c], -1) * 65536
    got = a.kernel.taps["wire.q"].cpu().double()
    assert (got - want).abs().max() <= 0.5 + 1e-6
    y2, _ = a(torch.randn(1, 1, 256))                # and a decode token behind them
    assert y2.shape == (1, 1, 256) and a.last_report.context == 13


def test_adapter_refuses_other_norms(ctx):
    import torch.nn as nn
    from insitu_amd.adapters.torch_llama import build_from_layer
    _, RMSNorm = _attention(64)
    for cls in (lambda: nn.LayerNorm(64), lambda: nn.LayerNorm(64, bias=False), lambda: RMSNorm(1.0), lambda: nn.Identity(),
                lambda: nn.RMSNorm(512, eps=1e-6)):
        attn, _ = _attention(64, cls)
        with pytest.raises(NotImplementedError, match="QK-norm"):
            build_from_layer(attn, _CONFIG, ctx=ctx)
    attn, _ = _attention(64)
    attn.k_norm.variance_epsilon = 1e-5
    with pytest.raises(NotImplementedError, match="QK-norm"):
        build_from_layer(attn, _CONFIG, ctx=ctx)
