"""GPU: layers with a sliding window as a user runs them. AttentionBlock(window=, sinks=): decode steps, prompts and
hidden states against oracle/c over the rows that each query sees; a window that no row has left is the block without
one. A dense cache's rows taken over, attended, and given back (append_float, attend_window and read_float
together). The adapter: the layer's own window, a graft in the middle of a sequence, and the model that goes on
without it. Integers: equality; models with 8-bit codes: cosines, as their ungrafted layers."""

import numpy as np
import pytest

from oracle import native
from oracle.quantize import Cache, CompressedKV, Format
from oracle.rotate import rotate, signs_from_seed

pytestmark = pytest.mark.gpu

N_KV = 2


def _block(ctx, G=4, d=64, **kw):
    from insitu_amd import QuantConfig
    from insitu_amd.block import AttentionBlock
    from insitu_amd.config import ModelConfig
    m = ModelConfig(hidden_size=256, num_heads=N_KV * G, num_kv_heads=N_KV, head_dim=d)
    kw.setdefault("quant", QuantConfig(key_bits=4, value_bits=2))
    kw.setdefault("capacity", 160)
    return AttentionBlock(m, ctx=ctx, **kw)


def _seen(p, window, sinks):
    t = np.arange(p + 1)
    return t[(t < sinks) | (t > p - window)]


def _draw(rng, *shape):
    return np.rint(rng.standard_normal(shape) * 65536).astype(np.int64)


def _want(host, f, q, p, window, sinks, softmax, sg):
    """A step's integers at row p: q (heads, d) off the wire."""
    fn = native.attend_two_pass if softmax == "two_pass" else native.attend_online
    idx, qr, G = _seen(p, window, sinks), rotate(q, sg), len(q) // N_KV
    out = []
    for h in range(N_KV):
        kv = host.view(h)
        out.append(fn(qr[G * h:G * h + G], CompressedKV(kv.k_idx[idx], kv.k_norm[idx], kv.v_idx[idx], kv.v_norm[idx]), f)[0])
    return np.concatenate(out).reshape(-1)


@pytest.mark.parametrize("softmax", ["online", "two_pass"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 2), (16, 4), (33, 0)])
@pytest.mark.parametrize("G,d", [(4, 64), (2, 128)])
def test_decode_steps(ctx, softmax, window, sinks, G, d):
    """A ragged batch from its first rows to far behind the window, token by token."""
    rng = np.random.default_rng(0)
    ahead, steps = [0, 11], 48
    blk = _block(ctx, G, d, batch=2, window=window, sinks=sinks, softmax=softmax)
    f, sg = Format(d=d, key_bits=4, value_bits=2), signs_from_seed(d, 0, 1)
    hosts = [Cache(N_KV, 160, f) for _ in ahead]
    k, v = _draw(rng, ahead[1], N_KV, d), _draw(rng, ahead[1], N_KV, d)
    blk.cache.append_wire(k, v, seq=1)
    hosts[1].append_rotated(rotate(k, sg), rotate(v, sg))
    for t in range(steps):
        q, k, v = _draw(rng, 2, N_KV * G, d), _draw(rng, 2, N_KV, d), _draw(rng, 2, N_KV, d)
        out = blk.step(q, k, v).cpu().numpy()
        assert blk.cache.lengths() == [t + 1, t + 12]
        assert blk.last_stats.n_tokens == max(len(_seen(t + a, window, sinks)) for a in ahead)
        for b in range(2):
            hosts[b].append_rotated(rotate(k[b][None], sg), rotate(v[b][None], sg))
            np.testing.assert_array_equal(out[b], _want(hosts[b], f, q[b], t + ahead[b], window, sinks, softmax, sg),
                                          err_msg=f"step {t} sequence {b}")


@pytest.mark.parametrize("softmax", ["online", "two_pass"])
@pytest.mark.parametrize("window,sinks", [(5, 1), (24, 4)])
def test_prompts_are_their_steps(ctx, softmax, window, sinks):
    """A prompt, another behind it, and a token: the block's integers are the token loop's and the oracle's."""
    rng = np.random.default_rng(1)
    a = _block(ctx, window=window, sinks=sinks, softmax=softmax)
    b = _block(ctx, window=window, sinks=sinks, softmax=softmax)
    f, sg = Format(d=64, key_bits=4, value_bits=2), signs_from_seed(64, 0, 1)
    host, p = Cache(N_KV, 160, f), 0
    for n in (3, 70, 1, 41):
        q, k, v = _draw(rng, n, 8, 64), _draw(rng, n, N_KV, 64), _draw(rng, n, N_KV, 64)
        host.append_rotated(rotate(k, sg), rotate(v, sg))
        got = a.forward_seam(q, k, v)
        np.testing.assert_array_equal(got, b.forward_seam(q, k, v, force_token_loop=True))
        for i in range(n):
            np.testing.assert_array_equal(got[i], _want(host, f, q[i], p + i, window, sinks, softmax, sg))
        p += n


def test_a_window_that_no_row_has_left(ctx):
    """... is the block without one, drafts too; behind it a draft is refused before its rows are written."""
    rng = np.random.default_rng(2)
    a, b = _block(ctx, window=20, sinks=3), _block(ctx)
    for n in (9, 1, 8):
        q, k, v = _draw(rng, n, 8, 64), _draw(rng, n, N_KV, 64), _draw(rng, n, N_KV, 64)
        np.testing.assert_array_equal(a.forward_seam(q, k, v), b.forward_seam(q, k, v))
    q, k, v = _draw(rng, 1, 5, 8, 64), _draw(rng, 1, 5, N_KV, 64), _draw(rng, 1, 5, N_KV, 64)
    parents = [-1, 0, 0, 1, 2]
    np.testing.assert_array_equal(a.step_tree(q, k, v, parents).cpu().numpy(), b.step_tree(q, k, v, parents).cpu().numpy())
    with pytest.raises(NotImplementedError, match="sliding window"):
        a.step_tree(q, k, v, parents)
    assert a.cache.length == 23


def test_refusals(ctx):
    for kw in (dict(window=0), dict(window=-4), dict(window=4, sinks=-1), dict(window=1 << 63)):
        with pytest.raises(ValueError):
            _block(ctx, **kw)
    with pytest.raises(TypeError):
        _block(ctx, window=2.5)
    from insitu_amd._lib import CapacityError
    rng = np.random.default_rng(3)
    blk = _block(ctx, window=4, sinks=1, capacity=12)
    row = [_draw(rng, 1, h, 64) for h in (8, N_KV, N_KV)]
    for _ in range(12):
        blk.step(*row)
    before = blk.cache.read_rows(0, 0, 12)
    with pytest.raises(CapacityError):
        blk.step(*row)
    assert blk.cache.length == 12
    np.testing.assert_array_equal(blk.cache.read_rows(0, 0, 12), before)
    k = np.zeros((3, N_KV, 64), np.float32)
    with pytest.raises(ValueError):
        blk.take(k, k, first=5)                       # it holds rows
    empty = _block(ctx, window=4, sinks=1)
    for first in (5, -1):
        with pytest.raises(ValueError):
            empty.take(k, k, first=first)             # without the rows that stay visible
    assert empty.cache.length == 0


@pytest.mark.parametrize("softmax", ["online", "two_pass"])
def test_forward(ctx, softmax):
    """Hidden states in and out, a prompt and tokens, with and without the token loop."""
    import torch
    from insitu_amd.host import Weights
    rng = np.random.default_rng(4)
    a, b = (_block(ctx, window=12, sinks=2, softmax=softmax) for _ in range(2))
    a.weights = b.weights = Weights.random(a.model, a.rotation, ctx=ctx)
    b.force_token_loop = True
    for n in (30, 1, 1):
        x = rng.standard_normal((n, 256)).astype(np.float32)
        (ya, ra), (yb, _) = a.forward(x), b.forward(x)
        # the projections of one row and of many are different products: compare below the seam where they agree
        same = all(torch.equal(a.taps[f"wire.{c}"], b.taps[f"wire.{c}"]) for c in "qkv")
        assert same and torch.equal(a.taps["out"], b.taps["out"]) and torch.equal(ya, yb)
        assert ra.attention.n_tokens == 14


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n", [1, 15, 65, 100])
def test_a_dense_cache_taken_over_attended_and_given_back(ctx, dtype, n):
    """The operators together: a dense cache's n rows are taken over, a turn of 20 tokens and three tokens
    attend a window with first rows, and all rows are read back."""
    import torch
    t = getattr(torch, dtype)
    rng = np.random.default_rng(5)
    dense = [torch.as_tensor(rng.standard_normal((1, N_KV, n, 64)), dtype=torch.float32).to(t).to(ctx.torch_device)
             for _ in range(2)]
    blk = _block(ctx, window=24, sinks=4)
    f, sg = Format(d=64, key_bits=4, value_bits=2), signs_from_seed(64, 0, 1)
    host = Cache(N_KV, 160, f)
    blk.take(dense[0].transpose(1, 2)[0], dense[1].transpose(1, 2)[0])
    fixed = [np.rint(x[0].transpose(0, 1).double().cpu().numpy() * 65536).astype(np.int64) for x in dense]
    host.append_rotated(*(rotate(x, sg) for x in fixed))
    p = n
    for m in (20, 1, 1, 1):
        q, k, v = _draw(rng, m, 8, 64), _draw(rng, m, N_KV, 64), _draw(rng, m, N_KV, 64)
        host.append_rotated(rotate(k, sg), rotate(v, sg))
        got = blk.forward_seam(q, k, v)
        for i in range(m):
            np.testing.assert_array_equal(got[i], _want(host, f, q[i], p + i, 24, 4, "online", sg))
        p += m
    k, v = blk.cache.read_float(dtype=t, rotated=True)
    assert k.shape == v.shape == (1, p, N_KV, 64) and k.dtype == t
    kc, _, vc = f.codebooks()[:3]
    for h in range(N_KV):
        kv = host.view(h)
        for got, idx, norm, c in ((k, kv.k_idx, kv.k_norm, kc), (v, kv.v_idx, kv.v_norm, vc)):
            want = np.asarray(c)[idx].astype(np.float64) * np.asarray(norm, np.float64)[:, None] / 2.0 ** 25
            got = got[0, :, h].double().cpu().numpy()
            # (the unit of a product of centroid and norm is the format's: taken from the largest element)
            i = np.unravel_index(np.abs(want).argmax(), want.shape)
            unit = 2.0 ** np.rint(np.log2(got[i] / want[i]))
            # one rounding of the product to 32 bits and one to the type
            np.testing.assert_allclose(got, want * unit, rtol=torch.finfo(t).eps / 2 + 3 * 2.0 ** -24, atol=0)


# -- the adapter ---------------------------------------------------------------------------

def _mistral(window, layers=2):
    import torch
    from transformers import MistralConfig, MistralForCausalLM
    torch.manual_seed(1)
    cfg = MistralConfig(hidden_size=512, intermediate_size=768, num_attention_heads=8, num_key_value_heads=2, head_dim=64,
                        num_hidden_layers=layers, vocab_size=256, max_position_embeddings=512, sliding_window=window)
    cfg._attn_implementation = "eager"
    return MistralForCausalLM(cfg).eval()


def _cos(a, b):
    return (a * b).sum(-1) / (np.linalg.norm(a, axis=-1) * np.linalg.norm(b, axis=-1))


IDS = [[5, 9, 200, 31, 77, 2, 140, 18, 66, 4, 91, 33, 250, 7, 12, 180, 99, 41, 3, 60, 61, 62, 201, 14, 15, 16, 120]]


def test_a_layers_own_window(ctx):
    """A prompt of 27 tokens and tokens behind it, window 6: the grafted model's logits are the model's to the codes'
    8 bits."""
    import torch
    from insitu_amd import QuantConfig
    from insitu_amd.adapters.torch_llama import graft
    from transformers import DynamicCache
    model = _mistral(6)
    ids = torch.tensor(IDS)
    more = torch.tensor([[8], [130], [44]])

    def run():
        cache, out = DynamicCache(config=model.config), []
        with torch.no_grad():
            out.append(model(input_ids=ids, past_key_values=cache, use_cache=True).logits[0])
            for t in more:
                out.append(model(input_ids=t[None], past_key_values=cache, use_cache=True).logits[0])
        return torch.cat(out).float().numpy()
    ref = run()
    graft(model, [0, 1], quant=QuantConfig(key_bits=8, value_bits=8), capacity=64, window="layer", ctx=ctx)
    assert [model.model.layers[i].self_attn.kernel.window for i in (0, 1)] == [6, 6]
    got = run()
    assert _cos(ref, got).min() > 0.99


@pytest.mark.parametrize("window", [None, 6])
def test_graft_in_the_middle_of_a_sequence_and_go_on_without(ctx, window):
    """The model reads a prompt, its layers are grafted with its dense cache, tokens, the layers are put back with it,
    tokens: the logits are those of the model alone to the codes' 8 bits. A dynamic cache of a window's layers
    keeps the last rows alone."""
    import torch
    from insitu_amd import QuantConfig
    from insitu_amd.adapters.torch_llama import graft, ungraft
    from transformers import DynamicCache
    model = _mistral(window)
    ids = torch.tensor(IDS)
    more = [torch.tensor([[t]]) for t in (8, 130, 44, 45, 99, 17)]

    def run(kernels):
        cache, out = DynamicCache(config=model.config), []
        with torch.no_grad():
            out.append(model(input_ids=ids, past_key_values=cache, use_cache=True).logits[0])
            if kernels:
                orig = graft(model, [0, 1], quant=QuantConfig(key_bits=8, value_bits=8), capacity=64, window="layer",
                             past_key_values=cache, ctx=ctx)
                blocks = [model.model.layers[i].self_attn.kernel for i in (0, 1)]
                rows = cache.layers[0].keys.shape[2]
                assert [b.cache.length for b in blocks] == [rows] * 2
                assert [b.first for b in blocks] == [27 - rows] * 2
            for t in more[:3]:
                out.append(model(input_ids=t, past_key_values=cache, use_cache=True).logits[0])
            if kernels:
                assert not cache.layers[0].keys[:, :, -3:].any()
                ungraft(model, orig, past_key_values=cache)
                assert cache.layers[1].keys[:, :, -3:].any()
            for t in more[3:]:
                out.append(model(input_ids=t, past_key_values=cache, use_cache=True).logits[0])
        return torch.cat(out).float().numpy()
    ref = run(False)
    got = run(True)
    np.testing.assert_array_equal(ref[:27], got[:27])
    assert _cos(ref, got).min() > 0.99


def test_take_and_give_refusals(ctx):
    import torch
    from insitu_amd.adapters.torch_llama import build_from_layer
    from transformers import DynamicCache
    model = _mistral(None)
    adapter = build_from_layer(model.model.layers[0].self_attn, model.config, capacity=64, ctx=ctx)
    assert adapter.take(DynamicCache()) == 0 and adapter.give(DynamicCache()) == 0
    two = DynamicCache()
    two.update(torch.zeros(2, 2, 5, 64), torch.zeros(2, 2, 5, 64), 0)
    with pytest.raises(NotImplementedError, match="batch of 2"):
        adapter.take(two)
    with pytest.raises(TypeError):
        adapter.take(object())
    one = DynamicCache()
    one.update(torch.randn(1, 2, 5, 64), torch.randn(1, 2, 5, 64), 0)
    assert adapter.take(one) == 5 and adapter.kernel.cache.length == 5
    with pytest.raises(ValueError, match="5 rows already"):
        adapter.take(one)
    one.update(torch.zeros(1, 2, 1, 64), torch.zeros(1, 2, 1, 64), 0)
    with pytest.raises(ValueError, match="not of the block's sequence"):
        adapter.give(one)


def test_a_graft_is_whole_or_not_at_all(ctx):
    """A cache that no block can take: the layers stay the model's own."""
    import torch
    from insitu_amd.adapters.torch_llama import graft, ungraft
    from transformers import DynamicCache
    model = _mistral(None)
    before = [layer.self_attn for layer in model.model.layers]
    cache = DynamicCache()
    cache.update(torch.randn(1, 2, 5, 64), torch.randn(1, 2, 5, 64), 0)
    cache.update(torch.randn(1, 2, 70, 64), torch.randn(1, 2, 70, 64), 1)     # more rows than there is room for
    with pytest.raises(ValueError):
        graft(model, [0, 1], capacity=64, past_key_values=cache, ctx=ctx)
    assert [layer.self_attn for layer in model.model.layers] == before
    orig = graft(model, [0, 0, 1], capacity=80, past_key_values=cache, ctx=ctx)
    assert [orig[0], orig[1]] == before
    ungraft(model, orig, past_key_values=cache)
    assert [layer.self_attn for layer in model.model.layers] == before


def test_a_window_step_is_its_parts(ctx):
    """insitu_step_window's statistics and appended rows against append_wire and attend_window."""
    import torch
    from insitu_amd.attention import CompressedAttention
    rng = np.random.default_rng(6)
    a, b = _block(ctx, batch=3, window=9, sinks=2), _block(ctx, batch=3)
    fill = _draw(rng, 3, 30, N_KV, 64), _draw(rng, 3, 30, N_KV, 64)
    for blk in (a, b):
        blk.cache.append_wire(*fill)
    for softmax in ("online", "two_pass", "serial"):
        a.softmax = softmax
        q, k, v = (torch.as_tensor(_draw(rng, 3, h, 64), dtype=torch.int32).to(ctx.torch_device) for h in (8, N_KV, N_KV))
        out = a.step(q, k, v)
        b.cache.append_wire(k[:, None].contiguous(), v[:, None].contiguous())
        want, st = CompressedAttention(b.cache).attend_window(b.rotation.apply(q, ctx).reshape(3, 1, 8, 64), 9, 2, softmax)
        assert torch.equal(out.reshape(want.shape), want)
        assert (a.last_stats.rescale_events, a.last_stats.max_abs_score, a.last_stats.max_abs_acc, a.last_stats.n_tokens) == \
            (st.rescale_events, st.max_abs_score, st.max_abs_acc, st.n_tokens)
        n = a.cache.lengths()[0]
        for s in range(3):
            for h in range(N_KV):
                np.testing.assert_array_equal(a.cache.read_rows(h, 0, n, s), b.cache.read_rows(h, 0, n, s))


def test_outputs_in_one_place(ctx):
    """Memory that two rows would be written to, or read from and written to."""
    import torch
    from insitu_amd.attention import CompressedAttention
    rng = np.random.default_rng(7)
    blk = _block(ctx)
    blk.cache.append_wire(_draw(rng, 30, N_KV, 64), _draw(rng, 30, N_KV, 64))
    whole = torch.zeros(6, 8, 64, dtype=torch.int32, device=ctx.torch_device)
    for q, out in ((whole[:5], whole[1:]), (whole[1:], whole[:5])):
        with pytest.raises(ValueError, match="part of it"):
            CompressedAttention(blk.cache).attend_window(q, 9, 2, out=out)
    x = torch.zeros(30, N_KV, 64, device=ctx.torch_device)
    with pytest.raises(ValueError, match="one place"):
        blk.cache.read_float(seq=0, out=(x, x))
    both = torch.zeros(30, N_KV, 2, 64, device=ctx.torch_device)              # (side by side is apart)
    blk.cache.read_float(seq=0, out=(both[:, :, 0], both[:, :, 1]))
    k, v = blk.cache.read_float(seq=0)
    assert torch.equal(both[:, :, 0], k) and torch.equal(both[:, :, 1], v)
