"""GPU: captured trees, compactions and forks between appends and steps. Every append and step moves the lengths
to the other half of a double buffer; a graph holds one address. Its replays have to find the lengths that the
cache has by then, and what they set has to be what every later call finds, after one turn, two and three."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

N, T = 3, 150                                          # nodes of the trees; rows of a sequence at the capture
# who writes a turn's rows: (query heads a KV head, key bits, value bits, softmax, pinned kernel)
WRITERS = {
    "append_rotated": (4, 4, 2, "online", None),
    "append_seq": (4, 4, 2, "online", None),
    "append_wire": (4, 3, 3, "online", None),
    "append of many rows": (4, 4, 2, "online", 2),
    "step kernel": (4, 4, 2, "online", "step"),
    "chunked step": (4, 4, 2, "online", "chunked"),
    "two-launch step": (8, 3, 2, "online", "chunked"),
    "scan step": (8, 4, 2, "online", "scan"),
    "split step": (4, 4, 2, "two_pass", None),
    "serial step": (4, 4, 2, "serial", None),
}


def _draw(rng, *shape):
    return np.rint(rng.standard_normal(shape) * 40000).astype(np.int32)


class Serving:
    """A block on a stream of its own, two sequences, T rows each."""

    def __init__(self, ctx, writer):
        import torch
        from insitu_amd import AttentionBlock, ModelConfig, QuantConfig, _lib
        from insitu_amd.runtime import Context
        self.side = torch.cuda.Stream(ctx.torch_device)
        self.own = Context(ctx.device, stream=self.side)
        G, kb, vb, softmax, pin = WRITERS[writer]
        self.name, self.heads, self.mode = writer, 2 * G, softmax
        self.rng = np.random.default_rng(len(writer))
        model = ModelConfig(hidden_size=256, num_heads=self.heads, num_kv_heads=2, head_dim=64)
        mk = lambda: AttentionBlock(model, QuantConfig(key_bits=kb, value_bits=vb), capacity=3000, batch=2, softmax=softmax, ctx=self.own)
        self.blk, self.ref = mk(), mk()
        if isinstance(pin, str):
            self.blk.cache.pin_kernel(pin)
        elif pin:
            _lib.check(self.own.lib.insitu_cache_debug(self.blk.cache.handle, _lib.DEBUG_APPEND, pin))
        self.c = self.blk.cache
        self.rows(T, plain=True)

    def rows(self, n, plain=False):
        """n new rows of both sequences."""
        import torch
        if plain or self.name in ("append_rotated", "append of many rows"):
            self.c.append_rotated(*(_draw(self.rng, 2, n, 2, 64) for _ in "kv"))
        elif self.name == "append_seq":
            for b in (0, 1):
                self.c.append_rotated(*(_draw(self.rng, n, 2, 64) for _ in "kv"), seq=b)
        elif self.name == "append_wire":
            self.c.append_wire(*(_draw(self.rng, 2, n, 2, 64) for _ in "kv"))
        else:
            for _ in range(n):
                self.blk.step(*(torch.from_numpy(_draw(self.rng, 2, h, 64)).to(self.own.torch_device)
                                for h in (self.heads, 2, 2)), stats=False)
        self.side.synchronize()

    def like(self, lens):
        """A cache of the same rows with lengths given by the host alone."""
        r = self.ref.cache
        for b, n in enumerate(lens):
            r.load_image(self.c.image(b), b)
            r.set_length(n, b)
        return self.ref.attn

    def lengths_are(self, lens):
        """What the device has for lengths, as a decode attend and a tree see them and as an append takes them on
        (whatever the host's copy says, which only needs to be no shorter)."""
        import torch
        q = torch.from_numpy(_draw(self.rng, 2, self.heads, 64)).to(self.own.torch_device)
        qt = torch.from_numpy(_draw(self.rng, 2, 2, self.heads, 64)).to(self.own.torch_device)
        ref = self.like(lens)
        got = [self.blk.attn.attend(q, mode=self.mode, stats=False)[0].clone(),
               self.blk.attn.attend_tree(qt, [-1, 0], self.mode, stats=False)[0].clone()]
        want = [ref.attend(q, mode=self.mode, stats=False)[0], ref.attend_tree(qt, [-1, 0], self.mode, stats=False)[0]]
        self.side.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("writer", WRITERS)
def test_tree(ctx, writer):
    import torch
    s = Serving(ctx, writer)
    dev = s.own.torch_device
    with torch.cuda.stream(s.side):
        q = torch.from_numpy(_draw(s.rng, 2, N, s.heads, 64)).to(dev)
        p = torch.tensor([-1, 0, 0], dtype=torch.int32, device=dev)
        out = torch.zeros_like(q)
        s.blk.attn.attend_tree(q, p, s.mode, out=out, stats=False)
        s.side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s.side):
            s.blk.attn.attend_tree(q, p, s.mode, out=out, stats=False)
        for turn in range(4):
            if turn:                                    # drop the draft, write another
                s.c.keep(N)
                s.rows(N)
            q.copy_(torch.from_numpy(_draw(s.rng, 2, N, s.heads, 64)))
            out.zero_()
            g.replay()
            got = out.clone()
            want = s.like([T, T]).attend_tree(q, p, s.mode, stats=False)[0]
            s.side.synchronize()
            assert torch.equal(got, want), f"turn {turn}"
        s.rows(1)                                       # a longer sequence: the rows up to the capture's longest
        out.zero_()
        g.replay()
        got = out.clone()
        want = s.like([T, T]).attend_tree(q, p, s.mode, stats=False)[0]
        s.side.synchronize()
        assert torch.equal(got, want)
        s.c.keep(11)                                    # and shorter ones as they are
        g.replay()
        got = out.clone()
        want = s.like([T - 10] * 2).attend_tree(q, p, s.mode, stats=False)[0]
        s.side.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("writer,kept", [(w, 1) for w in WRITERS] + [("append_rotated", 1100), ("step kernel", 1100)])
def test_keep(ctx, writer, kept):
    """Both ways of keeping: in place, and through a buffer."""
    import torch
    s = Serving(ctx, writer)
    n = kept + N - 1
    with torch.cuda.stream(s.side):
        s.rows(n, plain=True)
        full = s.c.length
        rows = torch.arange(N - 1, n, dtype=torch.int32, device=s.own.torch_device)
        if kept > 1024:                                 # (the buffer is allocated before the capture)
            s.c.keep(n, rows)
            s.rows(n - kept, plain=True)
        assert s.c.lengths() == [full] * 2
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s.side):
            s.c.keep(n, rows)
        for turn in range(4):
            if turn:
                s.rows(n - kept)
                assert s.c.lengths() == [full] * 2
            before = [s.c.image(b) for b in (0, 1)]
            g.replay()
            s.side.synchronize()
            for b in (0, 1):
                lay, img, off = s.c.layout(), before[b], 0
                for _ in range(2):
                    for w, span in zip(lay["plane_width"], lay["plane_span"]):
                        part = img[off:off + span]
                        part[(full - n) * w:(full - n + kept) * w] = part[(full - kept) * w:full * w].copy()
                        off += span
                np.testing.assert_array_equal(s.c.image(b), img)
            s.lengths_are([full - n + kept] * 2)
            for b in (0, 1):                            # the host's copy follows
                s.c.set_length(full - n + kept, b)


@pytest.mark.parametrize("writer", WRITERS)
def test_fork(ctx, writer):
    import torch
    s = Serving(ctx, writer)
    with torch.cuda.stream(s.side):
        rows = torch.tensor([4, 0, 2], dtype=torch.int32, device=s.own.torch_device)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s.side):
            s.c.fork(0, [1], n=9, rows=rows)
        for turn in range(4):
            if turn:                                    # both go on, the source comes back to where it was
                s.rows(1)
                s.c.set_length(T, 0)
            g.replay()
            s.side.synchronize()
            s.lengths_are([T, T - 6])
            for b, x in ((0, T), (1, T - 6)):
                s.c.set_length(x, b)
        for h in range(2):
            a = [s.c.read_rows(h, 0, T, 0), s.c.read_rows(h, 0, T - 6, 1)]
            np.testing.assert_array_equal(a[1], a[0][np.r_[0:T - 9, T - 5, T - 9, T - 7]])


def test_a_step_after_a_replayed_keep(ctx):
    """A step takes its place from the lengths that the replay set."""
    import torch
    s = Serving(ctx, "step kernel")
    with torch.cuda.stream(s.side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s.side):
            s.c.keep(5)
        for turn in range(3):
            g.replay()                                  # (the host's copy says T after the first time)
            s.side.synchronize()
            qkv = [torch.from_numpy(_draw(s.rng, 2, h, 64)).to(s.own.torch_device) for h in (s.heads, 2, 2)]
            s.like([T - 5] * 2)
            assert torch.equal(s.blk.step(*qkv), s.ref.step(*qkv))
            for b in (0, 1):
                s.c.set_length(T - 4, b)
            s.rows(4)
            assert s.c.lengths() == [T] * 2


def test_captured_on_the_callers_stream(ctx):
    """A tree and a compaction of a block whose stream is not the capturing one: both are in the graph."""
    import torch
    s = Serving(ctx, "append_rotated")
    dev = s.own.torch_device
    mine = torch.cuda.Stream(dev)
    q = torch.from_numpy(_draw(s.rng, 2, N, s.heads, 64)).to(dev)
    p = torch.tensor([-1, 0, 1], dtype=torch.int32, device=dev)
    rows = torch.tensor([0, 2], dtype=torch.int32, device=dev)
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(mine):
        s.blk.attn.attend_tree(q, p, out=out, stats=False)
        mine.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=mine):
            s.blk.attn.attend_tree(q, p, out=out, stats=False)
            s.c.keep(N, rows)
            out += 1
    for turn in range(3):
        if turn:
            s.rows(1)
            assert s.c.lengths() == [T] * 2
        with torch.cuda.stream(s.side):
            want = s.like([T, T]).attend_tree(q, p, stats=False)[0]
        s.side.synchronize()
        with torch.cuda.stream(mine):
            g.replay()
            mine.synchronize()
        assert torch.equal(out, want + 1)
        with torch.cuda.stream(s.side):
            s.lengths_are([T - 1] * 2)
        for b in (0, 1):
            s.c.set_length(T - 1, b)
