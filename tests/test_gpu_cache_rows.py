"""GPU: sequences that continue others (CompressedCache.fork) and the rows of a draft that stay
(CompressedCache.keep), byte for byte against numpy on the planes, the bytes around them included."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

FORMATS = [(64, 4, 2, 8), (128, 3, 3, 2), (64, 3, 2, 3), (64, 1, 8, 1), (128, 5, 1, 2)]


def _cache(ctx, fmt, batch, capacity, lens, seed=0):
    """Random images (the rows behind a sequence's end as well) and lengths."""
    from insitu_amd import QuantConfig
    from insitu_amd.cache import CompressedCache
    d, kb, vb, n_kv = fmt
    c = CompressedCache(n_kv, d, capacity, QuantConfig(key_bits=kb, value_bits=vb), batch=batch, n_q_heads=n_kv, ctx=ctx)
    rng = np.random.default_rng(seed)
    imgs = rng.integers(0, 256, (batch, c.layout()["seq_stride"]), dtype=np.uint8)
    for b in range(batch):
        c.load_image(imgs[b], b)
        c.set_length(lens[b], b)
    return c, imgs


def _take(lay, dst, at, src, rows, n_kv):
    """Rows `rows` of image src become rows at, at + 1, .. of image dst, in every plane."""
    rows = np.asarray(rows, dtype=np.int64)
    old = src.copy()
    off = 0
    for h in range(n_kv):
        for w, span in zip(lay["plane_width"], lay["plane_span"]):
            for j, r in enumerate(rows):
                dst[off + (at + j) * w:off + (at + j + 1) * w] = old[off + r * w:off + (r + 1) * w]
            off += span


def _same(c, imgs, lens):
    assert c.lengths() == list(lens)
    for b in range(len(lens)):
        np.testing.assert_array_equal(c.image(b), imgs[b], err_msg=f"sequence {b}")


def _device_lengths(c):
    """An append on every sequence shows the lengths the device holds."""
    d, n = c.head_dim, c.n_kv_heads
    before = c.lengths()
    one = np.full((c.batch, 1, n, d), 65536, dtype=np.int32)
    c.append_rotated(one, one)
    rows = [c.read_rows(0, n0, 1, b)[0] for b, n0 in enumerate(before)]
    assert all(np.array_equal(r, rows[0]) for r in rows)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("length", [0, 1, 3, 16, 255, 1030])
def test_whole_forks(ctx, fmt, length):
    lens = [5, length, 9, 700, 2]
    c, imgs = _cache(ctx, fmt, 5, 1100, lens)
    c.fork(1, [0, 3, 4])
    for b in (0, 3, 4):
        _take(c.layout(), imgs[b], 0, imgs[1], np.arange(length), fmt[3])
        lens[b] = length
    _same(c, imgs, lens)
    _device_lengths(c)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("length,n,kept", [(7, 7, 3), (40, 5, 0), (300, 64, 9), (1030, 1029, 517), (33, 1, 1)])
def test_forks_with_a_selection(ctx, fmt, length, n, kept):
    rng = np.random.default_rng(length)
    lens = [4, length, 9]
    c, imgs = _cache(ctx, fmt, 3, 1100, lens)
    lists = [np.sort(rng.choice(n, kept, replace=False)), rng.integers(0, n, max(0, kept - 1))]
    c.fork(1, [0, 2], n=n, rows=[list(map(int, x)) for x in lists])
    for b, rows in zip((0, 2), lists):
        idx = np.concatenate([np.arange(length - n), length - n + rows]).astype(np.int64)
        _take(c.layout(), imgs[b], 0, imgs[1], idx, fmt[3])
        lens[b] = len(idx)
    _same(c, imgs, lens)
    _device_lengths(c)


def test_many_copies_of_several_sources(ctx):
    fmt = FORMATS[0]
    batch = 80
    rng = np.random.default_rng(0)
    lens = [int(x) for x in rng.integers(1, 60, batch)]
    c, imgs = _cache(ctx, fmt, batch, 64, lens)
    dst = [int(x) for x in rng.permutation(np.arange(3, batch))[:70]]
    src = [int(x) for x in rng.integers(0, 3, 70)]
    c.fork(src, dst)
    for s, t in zip(src, dst):
        _take(c.layout(), imgs[t], 0, imgs[s], np.arange(lens[s]), fmt[3])
        lens[t] = lens[s]
    _same(c, imgs, lens)


def test_one_list_for_all_on_the_device(ctx):
    import torch
    fmt = FORMATS[1]
    lens = [100, 0, 0]
    c, imgs = _cache(ctx, fmt, 3, 128, lens)
    rows = torch.tensor([1, 4, 90, -5, 1000], dtype=torch.int32, device=ctx.torch_device)   # the last two: 0 and 91
    c.fork(0, [1, 2], n=92, rows=rows, counts=[5, 3])
    for b, m in ((1, 5), (2, 3)):
        _take(c.layout(), imgs[b], 0, imgs[0], np.concatenate([np.arange(8), 8 + np.array([1, 4, 90, 0, 91])[:m]]), fmt[3])
        lens[b] = 8 + m
    _same(c, imgs, lens)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n,kept", [(1, 0), (1, 1), (64, 5), (13, 13), (300, 120), (1500, 1024), (1500, 1025), (2000, 1777)])
def test_keep(ctx, fmt, n, kept):
    rng = np.random.default_rng(n + kept)
    lens = [n, n + 3, n + 70]
    c, imgs = _cache(ctx, fmt, 3, n + 90, lens)
    lists = [np.sort(rng.choice(n, kept, replace=False)) for _ in lens]
    lists[1] = lists[1][:kept // 2]
    lists[2] = rng.permutation(lists[2])
    c.keep(n, [list(map(int, x)) for x in lists])
    for b, rows in enumerate(lists):
        base = lens[b] - n
        _take(c.layout(), imgs[b], base, imgs[b], base + rows, fmt[3])
        lens[b] = base + len(rows)
    _same(c, imgs, lens)
    _device_lengths(c)


def test_keep_none_and_of_many_sequences(ctx):
    fmt = FORMATS[0]
    lens = [int(x) for x in np.random.default_rng(0).integers(8, 40, 70)]
    c, imgs = _cache(ctx, fmt, 70, 48, lens)
    c.keep(3)
    lens = [x - 3 for x in lens]
    _same(c, imgs, lens)
    c.keep(5, [4, 1])
    for b in range(70):
        _take(c.layout(), imgs[b], lens[b] - 5, imgs[b], [lens[b] - 1, lens[b] - 4], fmt[3])
    _same(c, imgs, [x - 3 for x in lens])
    c.keep(0)
    c.fork(0, [])
    _same(c, imgs, [x - 3 for x in lens])


def test_on_another_stream(ctx):
    """Lists made late on a stream that is not the context's; the rows read there without a synchronisation."""
    import torch
    fmt = FORMATS[0]
    lens = [1500, 10, 1400]
    c, imgs = _cache(ctx, fmt, 3, 1600, lens)
    kept = np.sort(np.random.default_rng(1).choice(1300, 1200, replace=False))
    img = c.device_image()
    side = torch.cuda.Stream(ctx.torch_device)
    rows = torch.from_numpy(kept.astype(np.int32)).to(ctx.torch_device)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big = torch.randn(2048, 2048, device=ctx.torch_device)
        for _ in range(20):
            big = big @ big * 1e-3
        late = rows + (big[0, 0] * 0).to(torch.int32)
        c.fork(0, [1], n=1300, rows=late)
        first = img[1].clone()
        c.set_length(1400, 0)
        c.set_length(1400, 1)
        late = rows.clone() + (big[0, 0] * 0).to(torch.int32)
        c.keep(1300, late)
        second = img.clone()
        c.keep(3, torch.tensor([2, 0], dtype=torch.int32, device=ctx.torch_device))
        third = img.clone()
    side.synchronize()
    lay = c.layout()
    _take(lay, imgs[1], 0, imgs[0], np.concatenate([np.arange(200), 200 + kept]), fmt[3])
    np.testing.assert_array_equal(first.cpu().numpy(), imgs[1])
    for b in range(3):
        _take(lay, imgs[b], 100, imgs[b], 100 + kept, fmt[3])
    np.testing.assert_array_equal(second.cpu().numpy(), imgs)
    for b in range(3):
        _take(lay, imgs[b], 1297, imgs[b], [1299, 1297], fmt[3])
    np.testing.assert_array_equal(third.cpu().numpy(), imgs)
    assert c.lengths() == [1299] * 3


@pytest.mark.parametrize("n,kept", [(40, 9), (1500, 1200)])
def test_captured_and_replayed(ctx, n, kept):
    """A fork and a compaction in one graph: replays read the lists anew and begin at the captured lengths."""
    import torch
    from insitu_amd.runtime import Context
    fmt, T = FORMATS[1], 1600
    side = torch.cuda.Stream(ctx.torch_device)
    own = Context(ctx.device, stream=side)
    rng = np.random.default_rng(2)
    with torch.cuda.stream(side):
        c, imgs = _cache(own, fmt, 2, 1700, [T, T])
        start = imgs.copy()
        rows = torch.zeros((2, kept), dtype=torch.int32, device=own.torch_device)
        c.keep(n, rows)                                 # (the buffer is allocated before the capture)
        for b in range(2):
            c.set_length(T, b)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            c.fork(0, [1], n=n, rows=rows[0], counts=[kept - 1])
            c.keep(kept - 1, rows[:, :3].contiguous() % (kept - 1), counts=[3, 2])
        for _ in range(3):
            imgs = start.copy()
            for b in range(2):
                c.load_image(imgs[b], b)
            new = rng.integers(0, n, (2, kept))
            rows.copy_(torch.from_numpy(new.astype(np.int32)))
            g.replay()
            side.synchronize()
            lay, cut = c.layout(), new[:, :3] % (kept - 1)
            _take(lay, imgs[1], 0, imgs[0], np.concatenate([np.arange(T - n), T - n + new[0, :kept - 1]]), fmt[3])
            for b, m, end in ((0, 3, T), (1, 2, T - n + kept - 1)):
                base = end - (kept - 1)
                _take(lay, imgs[b], base, imgs[b], base + cut[b, :m], fmt[3])
            _same(c, imgs, [T - (kept - 1) + 3, T - n + 2])
            for b in range(2):                          # (and eager work between the replays)
                c.read_rows(0, 0, 5, b)


def test_device_image_is_the_caches_memory(ctx):
    import torch
    fmt = FORMATS[0]
    c, imgs = _cache(ctx, fmt, 2, 40, [20, 7])
    img = c.device_image()
    assert img.shape == imgs.shape and img.is_cuda and img.dtype == torch.uint8
    np.testing.assert_array_equal(img.cpu().numpy(), imgs)
    c.fork(0, [1])
    torch.cuda.synchronize()
    np.testing.assert_array_equal(img[1].cpu().numpy(), c.image(1))


def test_refusals(ctx):
    from insitu_amd import _lib
    c, imgs = _cache(ctx, FORMATS[0], 4, 64, [10, 20, 30, 40])
    bad = [dict(src=0, dst=[0]), dict(src=0, dst=[4]), dict(src=-1, dst=[1]), dict(src=0, dst=[1, 1]),
           dict(src=[0, 1], dst=[2, 0]), dict(src=[0], dst=[1, 2]), dict(src=0, dst=[1], rows=[0]),
           dict(src=0, dst=[1], n=11, rows=[0]), dict(src=0, dst=[1], n=5, rows=[5]), dict(src=0, dst=[1], n=5, rows=[-1]),
           dict(src=0, dst=[1], n=5, rows=[0, 1], counts=[3]), dict(src=0, dst=[1, 2], n=5, rows=[[0], [1], [2]]),
           dict(src=0, dst=[1], n=5, counts=[1])]
    for kw in bad:
        with pytest.raises((_lib.InsituError, ValueError)):
            c.fork(kw.pop("src"), kw.pop("dst"), **kw)
    for kw in (dict(n=11), dict(n=-1), dict(n=5, rows=[5]), dict(n=5, rows=[0], counts=[2, 0, 0, 0]),
               dict(n=5, rows=[[0], [1]]), dict(n=5, counts=[1, 1, 1, 1])):
        with pytest.raises((_lib.InsituError, ValueError)):
            c.keep(kw.pop("n"), **kw)
    _same(c, imgs, [10, 20, 30, 40])


def test_lists_shorter_than_their_counts(ctx):
    from insitu_amd import _lib
    lens = [10, 20, 30, 40]
    c, imgs = _cache(ctx, FORMATS[0], 4, 64, lens)
    for counts in ([2, 2], [1], [2, 1, 1]):
        with pytest.raises(ValueError, match="counts"):
            c.fork(3, [0, 1], n=5, rows=[[1, 2], [3]], counts=counts)
    with pytest.raises(ValueError, match="counts"):
        c.keep(5, [[0], [1, 2], [3], []], counts=[1, 1, 1, 1])
    _same(c, imgs, lens)
    c.fork(3, [0, 1], n=5, rows=[[1, 2], [3]], counts=[1, 1])
    for b, r in ((0, 1), (1, 3)):
        _take(c.layout(), imgs[b], 0, imgs[3], list(range(35)) + [35 + r], 8)
        lens[b] = 36
    _same(c, imgs, lens)


def test_rows_past_32_bits(ctx):
    import torch
    lens = [30, 5]
    c, imgs = _cache(ctx, FORMATS[0], 2, 64, lens)
    c.fork(0, [1], n=20, rows=torch.tensor([(1 << 32) + 3, -(1 << 33), 7], device=ctx.torch_device))
    _take(c.layout(), imgs[1], 0, imgs[0], list(range(10)) + [29, 10, 17], 8)
    _same(c, imgs, [30, 13])
