"""GPU: floating keys and values written to the compressed cache and read back (float_rows.hip). Written rows
are integers and equal the oracle's (to_fixed, rotate, encode, pack) byte for byte; rows read back are held to
the roundings of their type around the float64 value. Types, strides, alignments, formats, rotations of none to
two rounds, ragged batches, values beyond Q8.16, streams, graphs, refusals."""

import numpy as np
import pytest

from oracle.host import to_fixed
from oracle.quantize import Cache, Format, decode_plane
from oracle.rotate import rotate

pytestmark = pytest.mark.gpu

N_KV = 3
# (d, key bits, value bits, rounds)
FORMATS = [(64, 4, 2, 1), (64, 3, 2, 1), (64, 2, 2, 1), (64, 4, 1, 1), (64, 3, 3, 1), (128, 3, 3, 1), (128, 4, 2, 1), (128, 2, 1, 1),
           (64, 4, 2, 2), (64, 4, 2, 0), (128, 3, 3, 2), (64, 8, 5, 1), (64, 1, 7, 1), (64, 8, 8, 1), (128, 1, 7, 1)]
TYPES = ["float32", "float16", "bfloat16"]


def _cache(ctx, fmt, capacity, batch=1):
    from insitu_amd import QuantConfig
    from insitu_amd.cache import CompressedCache
    d, kb, vb, rounds = fmt
    return CompressedCache(N_KV, d, capacity, QuantConfig(key_bits=kb, value_bits=vb, rot_rounds=rounds), batch=batch,
                           n_q_heads=N_KV, ctx=ctx)


def _floats(rng, type, *shape, scale=1.0):
    """Values of a type, a few channels that stand out, as (torch tensor, float64 array)."""
    import torch
    x = rng.standard_normal(shape) * scale * np.where(rng.random(shape[-1]) < 0.06, 8.0, 1.0)
    t = torch.from_numpy(x).to(getattr(torch, type))
    return t, t.double().numpy()


def _rotated(c, x):
    """The oracle's rotated rows of float64 values that the type holds, and how many left Q8.16."""
    q, lost = to_fixed(x)
    return (rotate(q, c.rotation.signs) if c.rotation.rounds else q), lost


def _want(c, fmt, k, v):
    d, kb, vb, _ = fmt
    host = Cache(N_KV, k.shape[0], Format(d=d, key_bits=kb, value_bits=vb))
    host.append_rotated(_rotated(c, k)[0], _rotated(c, v)[0])
    return host.buf


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads_first", [False, True])
def test_written_rows_are_the_oracles(ctx, fmt, type, heads_first):
    import torch
    rng = np.random.default_rng(1)
    for n in (1, 5, 16, 33, 130):
        c = _cache(ctx, fmt, 200, batch=2)
        at = [0, 7]
        for b, m in enumerate(at):
            c.set_length(m, b)
        shape = (2, N_KV, n, fmt[0]) if heads_first else (2, n, N_KV, fmt[0])
        ts, xs = zip(*(_floats(rng, type, *shape) for _ in "kv"))
        ts = [t.to(ctx.torch_device) for t in ts]
        if heads_first:
            ts, xs = [t.transpose(1, 2) for t in ts], [x.transpose(0, 2, 1, 3) for x in xs]
        assert c.append_float(*ts) is None
        assert c.lengths() == [n, n + 7]
        for b, m in enumerate(at):
            want = _want(c, fmt, xs[0][b], xs[1][b])
            for h in range(N_KV):
                np.testing.assert_array_equal(c.read_rows(h, m, n, b), want[:, h], err_msg=f"{n} rows, sequence {b} head {h}")
                assert not c.read_rows(h, 0, m, b).any()
                assert not c.read_rows(h, m + n, 200 - m - n, b).any()


@pytest.mark.parametrize("fmt", [FORMATS[0], FORMATS[5], FORMATS[11]])
@pytest.mark.parametrize("type", TYPES)
def test_written_rows_anywhere_in_memory(ctx, fmt, type):
    """One sequence of a batch; rows off 16 bytes, with strides of their own, out of order, and repeated."""
    import torch
    d = fmt[0]
    rng = np.random.default_rng(2)
    n = 37
    c = _cache(ctx, fmt, 100, batch=3)
    wide, _ = _floats(rng, type, 2, n, N_KV, d + 3)
    flat, _ = _floats(rng, type, 2 * n * N_KV * d + 1)
    one, _ = _floats(rng, type, 2, 1, N_KV, d)
    views = [wide.to(ctx.torch_device)[..., 1:d + 1], flat.to(ctx.torch_device)[1:].view(2, n, N_KV, d),
             one.to(ctx.torch_device).expand(2, n, N_KV, d), wide.to(ctx.torch_device)[..., 3:].flip(1),
             flat.to(ctx.torch_device)[1:].view(2, N_KV, n, d).transpose(1, 2),
             flat.to(ctx.torch_device)[:-1].view(2, d, N_KV, n).transpose(1, 3)]
    for i, view in enumerate(views):
        c.reset()
        c.append_float(view[0], view[1], seq=1)
        x = view.double().cpu().numpy()
        want = _want(c, fmt, x[0], x[1])
        assert c.lengths() == [0, n, 0]
        for h in range(N_KV):
            np.testing.assert_array_equal(c.read_rows(h, 0, n, 1), want[:, h], err_msg=f"view {i} head {h}")
            assert not c.read_rows(h, 0, 100, 0).any() and not c.read_rows(h, 0, 100, 2).any()


@pytest.mark.parametrize("fmt", [FORMATS[0], FORMATS[5], FORMATS[8], FORMATS[9]])
@pytest.mark.parametrize("type", TYPES)
def test_values_beyond_q8_16(ctx, fmt, type):
    """The ends of 24 bits, halves, infinities; NaN is 0; the count of those that did not fit."""
    import torch
    d = fmt[0]
    edges = [128.0, -128.0, 127.99998, -128.00001, 1e4, -1e4, float("inf"), -float("inf"), float("nan"), 0.0, -0.0, 2.0 ** -17,
             3 * 2.0 ** -17, -(2.0 ** -17), 2.0 ** -24, 1.5 * 2.0 ** -16, 127.0, -127.5]
    x = torch.tensor(edges * (2 * N_KV * d // len(edges) + 1), dtype=torch.float32)[:2 * N_KV * d].reshape(2, N_KV, d)
    x = x.to(getattr(torch, type))
    c = _cache(ctx, fmt, 10)
    lost = c.append_float(x.to(ctx.torch_device), x.flip(0).to(ctx.torch_device), counts=True)
    f = x.double().numpy()
    r = np.rint(f * 65536)
    assert lost == 2 * int((~((r >= -2 ** 23) & (r <= 2 ** 23 - 1))).sum())
    f = np.nan_to_num(f, nan=0.0, posinf=1e9, neginf=-1e9)
    want = _want(c, fmt, f, f[::-1])
    for h in range(N_KV):
        np.testing.assert_array_equal(c.read_rows(h, 0, 2), want[:, h])
    assert c.append_float(x.to(ctx.torch_device) * 0.0 + 1, x.to(ctx.torch_device), counts=True) >= 0
    y = torch.ones(1, N_KV, d, dtype=x.dtype, device=ctx.torch_device)
    assert c.append_float(y, -y, counts=True) == 0


def test_a_wire_append_and_a_float_append_agree(ctx):
    """Thousands of rows, which the wire append's other kernel takes."""
    import torch
    fmt = FORMATS[0]
    rng = np.random.default_rng(3)
    n = 5000
    a, b = _cache(ctx, fmt, n), _cache(ctx, fmt, n)
    k, v = (_floats(rng, "bfloat16", n, N_KV, 64)[0].to(ctx.torch_device) for _ in "kv")
    a.append_float(k, v)
    b.append_wire(*((x.double() * 65536).round().clamp(-2 ** 23, 2 ** 23 - 1).to(torch.int32) for x in (k, v)))
    assert torch.equal(a.device_image(), b.device_image())


def _decoded(c, fmt, lens, rotated):
    """The rows as float64: centroid times norm / 2^24, and turned back; a list of (k, v) a sequence."""
    d, kb, vb, rounds = fmt
    f = Format(d=d, key_bits=kb, value_bits=vb)
    kc, _, vc, _ = f.codebooks()
    out = []
    for b, n in enumerate(lens):
        got = []
        for which, cent in (("k", kc), ("v", vc)):
            x = np.zeros((n, N_KV, d))
            for h in range(N_KV):
                kv = c.view_from_buffer(h, b)
                x[:, h] = cent[getattr(kv, which + "_idx")] * getattr(kv, which + "_norm")[:, None] / 2.0 ** 24
            got.append(x if rotated or not rounds else x @ c.rotation.matrix())
        out.append(got)
    return out


def _near(got, want, type, d, rounds):
    """A value is rounded once into float32 and once into its type, and its scale (norm / 2^24 / sqrt d) once or twice;
    with more than one round the sums are in float64. Four roundings of 2^-24 and one of the type's, both relative
    to the value; half the type's smallest step (2^-25 for float16) below its normal numbers."""
    import torch
    got = got.double().cpu().numpy()
    eps = 2.0 ** -22 + (0 if type == "float32" else torch.finfo(getattr(torch, type)).eps / 2)
    tiny = 2.0 ** -25 if type == "float16" else 1e-40
    # (the oracle's float64 product cancels to 2^-50 of the row's largest value)
    np.testing.assert_array_less(np.abs(got - want), eps * np.abs(want) * 1.01 + tiny + 2.0 ** -46 * np.abs(want).max(initial=0))


def _filled(ctx, fmt, lens, capacity, seed=4):
    rng = np.random.default_rng(seed)
    c = _cache(ctx, fmt, capacity, batch=len(lens))
    for b, n in enumerate(lens):
        if n:
            c.append_rotated(*(np.rint(rng.standard_normal((n, N_KV, fmt[0])) * 65536 * np.exp(rng.standard_normal((n, 1, 1))))
                               .astype(np.int32) for _ in "kv"), seq=b)
    return c


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rotated", [False, True])
def test_read_rows_are_the_decoded_ones(ctx, fmt, type, rotated):
    import torch
    lens = [133, 0, 40]
    c = _filled(ctx, fmt, lens, 150)
    want = _decoded(c, fmt, lens, rotated)
    dtype = getattr(torch, type)
    for t0, n in ((0, None), (0, 1), (17, 50), (39, 1), (130, 3)):
        got = c.read_float(t0, n, dtype=dtype, rotated=rotated)
        m = 133 - t0 if n is None else n
        for x, w in zip(got, range(2)):
            assert x.shape == (3, m, N_KV, fmt[0]) and x.dtype == dtype and x.transpose(1, 2).is_contiguous()
            for b, T in enumerate(lens):
                there = max(0, min(T - t0, m))
                _near(x[b, :there], want[b][w][t0:t0 + there], type, fmt[0], fmt[3])
                assert not x[b, there:].any()
    for b in (0, 2):
        k, v = c.read_float(3, 20, seq=b, dtype=dtype, rotated=rotated)
        assert k.shape == (20, N_KV, fmt[0])
        _near(k, want[b][0][3:23], type, fmt[0], fmt[3])
        _near(v, want[b][1][3:23], type, fmt[0], fmt[3])


@pytest.mark.parametrize("fmt", [FORMATS[0], FORMATS[5], FORMATS[11]])
@pytest.mark.parametrize("type", TYPES)
def test_read_into_tensors_of_any_strides(ctx, fmt, type):
    """Outputs with gaps, off 16 bytes, heads or tokens first; what lies between and behind stays."""
    import torch
    d, lens, n = fmt[0], [60, 31], 50
    c = _filled(ctx, fmt, lens, 70)
    dtype = getattr(torch, type)
    plain = c.read_float(2, n, dtype=dtype)
    for make in (lambda: torch.full((2, n, N_KV, d), 7.0), lambda: torch.full((2, n, N_KV, d + 3), 7.0)[..., 2:d + 2],
                 lambda: torch.full((2, N_KV, n + 5, d), 7.0).transpose(1, 2)[:, :n],
                 lambda: torch.full((n, 2, 2, N_KV, d), 7.0)[:, :, 1].transpose(0, 1),
                 lambda: torch.full((2 * n * N_KV * d + 1,), 7.0)[1:].view(2, n, N_KV, d)):
        # (the storage around the view goes along)
        out = []
        for _ in "kv":
            x = make()
            base = torch.full((x.untyped_storage().nbytes() // 4,), 7.0, dtype=dtype, device=ctx.torch_device)
            out.append((base, base.as_strided(x.shape, x.stride(), x.storage_offset())))
        views = [v for _, v in out]
        assert c.read_float(2, n, out=views)[0] is views[0]
        for (base, view), want in zip(out, plain):
            for b, T in enumerate(lens):
                there = min(T - 2, n)
                assert torch.equal(view[b, :there], want[b, :there])
                assert bool((view[b, there:] == 7).all())
                view[b, :there] = 7.0
            assert bool((base == 7).all())


def test_there_and_back(ctx):
    """What is read is what the codes of a written row stand for: written again it gives norms within a step of
    the cast, and the model's own values within the codebooks' error."""
    import torch
    rng = np.random.default_rng(6)
    c = _cache(ctx, FORMATS[0], 300)
    k, v = (torch.from_numpy(rng.standard_normal((300, N_KV, 64))).float().to(ctx.torch_device) for _ in "kv")
    c.append_float(k, v)
    a, b = c.read_float(seq=0)
    # mean squared error of a Lloyd-Max quantiser of a unit Gaussian: 0.0095 at 4 bits, 0.1175 at 2
    assert float(((a - k) ** 2).mean()) < 0.012 and float(((b - v) ** 2).mean()) < 0.13
    r, s = c.read_float(seq=0, rotated=True)
    m = torch.from_numpy(c.rotation.matrix()).float().to(ctx.torch_device)
    torch.testing.assert_close(r @ m, a, rtol=0, atol=64 * 8 * 2.0 ** -24)


def test_rows_far_into_a_long_cache(ctx):
    """A plane's bytes past 2^31 and rows past 2^27: written, read and attended there."""
    import torch
    from insitu_amd import QuantConfig
    from insitu_amd.attention import CompressedAttention
    from insitu_amd.cache import CompressedCache
    far = (1 << 27) + 1000
    c = CompressedCache(1, 64, far + 600, QuantConfig(key_bits=4, value_bits=2), n_q_heads=4, ctx=ctx)
    near = CompressedCache(1, 64, 600, QuantConfig(key_bits=4, value_bits=2), n_q_heads=4, ctx=ctx)
    rng = np.random.default_rng(7)
    k, v = (torch.from_numpy(rng.standard_normal((600, 1, 64))).to(torch.bfloat16).to(ctx.torch_device) for _ in "kv")
    c.set_length(far)
    c.append_float(k, v)
    near.append_float(k, v)
    np.testing.assert_array_equal(c.read_rows(0, far, 600), near.read_rows(0, 0, 600))
    for x, y in zip(c.read_float(far, 600, seq=0), near.read_float(0, 600, seq=0)):
        assert torch.equal(x, y)
    q = torch.from_numpy(np.rint(rng.standard_normal((300, 4, 64)) * 16384).astype(np.int32)).to(ctx.torch_device)
    for mode in ("online", "two_pass"):
        for n in (1, 300):
            got = CompressedAttention(c).attend_window(q[:n], 250, mode=mode, stats=False)[0]
            want = CompressedAttention(near).attend_window(q[:n], 250, mode=mode, stats=False)[0]
            assert torch.equal(got, want)
    c.close()


def test_other_streams(ctx):
    import torch
    rng = np.random.default_rng(8)
    c, d = _cache(ctx, FORMATS[0], 400), _cache(ctx, FORMATS[0], 400)
    k, v = (_floats(rng, "float16", 300, N_KV, 64)[0].to(ctx.torch_device) for _ in "kv")
    c.append_float(k, v)
    want = [x.clone() for x in c.read_float(seq=0)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream(ctx.torch_device)
    with torch.cuda.stream(side):
        big = torch.randn(2048, 2048, device=ctx.torch_device)
        for _ in range(20):
            big = big @ big * 1e-3                      # the rows come late
        d.append_float(k + (big[0, 0] * 0).to(k.dtype), v + (big[0, 0] * 0).to(k.dtype))
        got = [x + 0 for x in d.read_float(seq=0)]
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_a_captured_read(ctx):
    """Replayed after rows were appended and dropped: the lengths of the replay."""
    import torch
    from insitu_amd.runtime import Context
    rng = np.random.default_rng(9)
    side = torch.cuda.Stream(ctx.torch_device)
    own = Context(ctx.device, stream=side)
    with torch.cuda.stream(side):
        c = _cache(own, FORMATS[5], 120, batch=2)
        k, v = (_floats(rng, "bfloat16", 2, 30, N_KV, 128)[0].to(own.torch_device) for _ in "kv")
        c.append_float(k, v)
        out = [torch.zeros(2, 100, N_KV, 128, device=own.torch_device) for _ in "kv"]
        c.read_float(0, 100, out=out)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            c.read_float(0, 100, out=out)
        for step in range(4):
            if step == 2:
                c.keep(45)
            else:
                c.append_float(k, v)
            for x in out:
                x.fill_(5.0)
            g.replay()
            side.synchronize()
            n = c.length
            for x, want in zip(out, c.read_float(0, n)):
                assert torch.equal(x[:, :n], want) and bool((x[:, n:] == 5).all())


def test_refusals(ctx):
    import torch
    from insitu_amd import _lib
    dev = ctx.torch_device
    c = _cache(ctx, FORMATS[0], 20, batch=2)
    k = torch.zeros(2, 5, N_KV, 64, device=dev)
    for bad in (lambda: c.append_float(k, k.half()), lambda: c.append_float(k, k[:, :4]), lambda: c.append_float(k[..., :32], k[..., :32]),
                lambda: c.append_float(k[0], k[0]), lambda: c.append_float(k[0], k[0], seq=2), lambda: c.append_float(k[0], k[0], seq=-1),
                lambda: c.append_float(k[:1], k[:1]), lambda: c.append_float(k, k, seq=0)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: c.append_float(k.double(), k.double()), lambda: c.append_float(k.int(), k.int()),
                lambda: c.read_float(dtype=torch.float64)):
        with pytest.raises(TypeError):
            bad()
    assert c.lengths() == [0, 0]
    c.append_float(k, k)
    with pytest.raises(_lib.CapacityError):
        c.append_float(torch.zeros(2, 16, N_KV, 64, device=dev), torch.zeros(2, 16, N_KV, 64, device=dev))
    assert c.append_float(k[:, :0], k[:, :0]) is None and c.append_float(k[:, :0], k[:, :0], counts=True) == 0
    assert c.lengths() == [5, 5]
    for bad in (lambda: c.read_float(-1, 2), lambda: c.read_float(0, 21), lambda: c.read_float(4, 2, seq=0), lambda: c.read_float(0, -1),
                lambda: c.read_float(0, 2, seq=2), lambda: c.read_float(0, 2, seq=-1)):
        with pytest.raises(ValueError):
            bad()
    good = [torch.zeros(2, 5, N_KV, 64, device=dev) for _ in "kv"]
    for out in (good[:1], [good[0], good[1].half()], [x[:, :4] for x in good], [x.cpu() for x in good],
                [torch.zeros(2, 1, N_KV, 64, device=dev).expand(2, 5, N_KV, 64)] * 2,
                [torch.zeros(2, 5, N_KV, 128, device=dev)[..., ::2]] * 2):
        with pytest.raises(ValueError):
            c.read_float(0, 5, out=out)
    with pytest.raises(ValueError):
        c.read_float(0, 5, out=good, dtype=torch.float16)
    x, y = c.read_float(0, 0)
    assert x.shape == (2, 0, N_KV, 64)
    c.reset()
    assert c.read_float()[0].shape == (2, 0, N_KV, 64)
