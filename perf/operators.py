"""The operators around speculative decoding on the compressed cache, as cases that can be
timed and compared.

    tree   CompressedAttention.attend_tree: the queries of a tree of drafted tokens, whose rows
           are the last of each sequence; a node attends the context and its own ancestors
    turn   one verification turn over a batch, as a serving loop runs it: CompressedCache.keep
           drops the tail of the turn before, append_rotated writes the drafted rows, attend_tree
           attends them, keep moves the accepted path's rows together behind the context
    fork   CompressedCache.fork: sequences that continue another one's rows, whole (n-best
           answers) or with a selection of its last rows (a branch of a draft, a conversation
           with turns taken out)
    seam   Seam.wire: the q|k|v projections to wire rows: bias, the norm of each query and key
           head, the attention scale, the rotation of positions (half or interleaved pairs, the
           whole head or part of it) and the cast to Q8.16

The cache holds bit-packed rows: codes of Lloyd-Max centroids (Q1.15) and an int16 norm (Q9) for
keys and values, in planes of at most 16 bytes a row. Scores are floor(sum(q c) norm / 2^24) in
Q16; the weights come from a table, p = floor(2^15 2^-(i / 256)), i = floor(delta log2(e) 2^8);
a value adds floor(norm p c / 2^23) a channel. Online mode takes the rows in order and, when a
score passes the maximum so far, scales what it has by the table's value for the difference, with
a floor; two-pass mode takes the maximum of all first. All of that is integers: the outputs are
the same whatever the order of the sums. Shapes are the repository's: 32 query heads of 64 over 8
KV heads (4-bit keys, 2-bit values), over 4 KV heads with 3-bit keys, and 32 heads of 128 over 8
KV heads with 3-bit keys and values.
"""

import math

import numpy as np
import torch

own = False

N_Q = 32                       # query heads of every shape
# (head_dim, KV heads, key bits, value bits)
SHAPES = [(64, 8, 4, 2), (64, 4, 3, 2), (128, 8, 3, 3), (64, 8, 3, 2), (128, 8, 4, 2)]
CENTROIDS = {
    2: [-49490, -14835, 14835, 49490],
    3: [-70498, -44018, -24759, -8027, 8027, 24759, 44018, 70498],
    4: [-89465, -67707, -52923, -41069, -30794, -21451, -12667, -4189,
        4189, 12667, 21451, 30794, 41069, 52923, 67707, 89465],
}
BOUNDS = {
    2: [-32163, 0, 32162],
    3: [-57258, -34389, -16393, 0, 16393, 34388, 57258],
    4: [-78586, -60315, -46996, -35932, -26123, -17059, -8428, 0, 8428, 17059, 26122, 35931, 46996, 60315, 78586],
}
LOG2E = 94548                  # round(log2(e) 2^16)
LUT_SPAN = 17 << 8             # table indices from here on give 0
DELTA_MAX = -(-(LUT_SPAN << 24) // LOG2E)
SCORE_LO = -(1 << 47)
ACC_LO, ACC_HI = -(1 << 31), (1 << 31) - 1


def _kv(shape):
    d, n_kv, kb, vb = shape
    return {"d": d, "n_kv": n_kv, "key_bits": kb, "value_bits": vb}


def _tree(shape, *, ctx, n, tree, batch=1, mode="online", scaled=True, keep=0, name=None):
    c = {"kind": "turn" if keep else "tree", **_kv(shape), "ctx": ctx, "n": n, "tree": tree, "batch": batch,
         "mode": mode, "scaled": scaled, "keep": keep}
    return {"name": name, **c} if name else c


def _fork(shape, *, ctx, copies, n=0, kept=0, name=None):
    c = {"kind": "fork", **_kv(shape), "ctx": ctx, "copies": copies, "n": n, "kept": kept}
    return {"name": name, **c} if name else c


def _seam(d, n_kv, *, n, rotary=None, interleaved=False, norm=True, bias=False, table=8192, name=None):
    c = {"kind": "seam", "d": d, "n_kv": n_kv, "n": n, "rotary": rotary or d, "interleaved": interleaved,
         "norm": norm, "bias": bias, "table": table}
    return {"name": name, **c} if name else c


def listed():
    return [
        # a short question's first drafts, one path of a small draft model: latency and launches
        _tree(SHAPES[0], ctx=100, n=5, tree="chain", name="tree_chain5_ctx100"),
        # an ordinary tree as the model adapter runs its softmax by default
        _tree(SHAPES[0], ctx=4097, n=64, tree="random", mode="two_pass", name="tree_64_two_pass_ctx4097"),
        # a tree at the benchmark's long context, peaked softmax
        _tree(SHAPES[0], ctx=32768, n=26, tree="random", scaled=False, name="tree_26_ctx32768"),
        # a serving batch of ragged sequences with small trees
        _tree(SHAPES[0], ctx=8192, n=9, tree="binary", batch=16, scaled=False, name="tree_9_batch16_ragged"),
        # the larger heads at long contexts, one layer of a batch
        _tree(SHAPES[2], ctx=32768, n=32, tree="random", batch=8, name="tree_d128_32_batch8_ctx32768"),
        # a whole verification turn, 8 query heads a KV head
        _tree(SHAPES[1], ctx=2047, n=13, tree="binary", batch=4, keep=4, name="turn_13_batch4_ctx2047"),
        # three answers to a short question: latency
        _fork(SHAPES[0], ctx=100, copies=3, name="fork_3_ctx100"),
        # eight answers to one long conversation
        _fork(SHAPES[0], ctx=32768, copies=8, name="fork_8_ctx32768"),
        # a long conversation with turns taken out, the larger heads
        _fork(SHAPES[2], ctx=32767, copies=1, n=30001, kept=14003, name="fork_kept_d128_ctx32767"),
        # one decode token of a model with norms of queries and keys
        _seam(64, 8, n=1, name="seam_norm_1"),
        # a prompt of such a model, the larger heads
        _seam(128, 8, n=4096, name="seam_norm_d128_4096"),
        # a part of each head rotated in interleaved pairs, biases, far positions
        _seam(64, 8, n=777, rotary=32, interleaved=True, norm=False, bias=True, table=131072,
              name="seam_interleaved_777"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "tree", "turn", "fork", "seam", "seam"])
    shape = rng.choice(SHAPES)
    if kind in ("tree", "turn"):
        # the work of a tree is its nodes times its context: no more than half the largest listed one's
        ctx = _log(rng, 1, 65536)
        room = 4 * 32768 * 32 * 128 // (shape[0] * ctx)
        n = _log(rng, 1, max(1, min(256, room)))
        batch = _log(rng, 1, max(1, min(32, room // n, (1 << 18) // ctx)))
        keep = rng.randint(1, min(n, 8)) if kind == "turn" else 0
        return _tree(shape, ctx=ctx, n=n, tree=rng.choice(["chain", "binary", "star", "random"]), batch=batch,
                     mode=rng.choice(["online", "online", "two_pass"]), scaled=rng.random() < 0.6, keep=keep)
    if kind == "fork":
        ctx = _log(rng, 1, 65536)
        n = rng.choice([0, _log(rng, 1, ctx)])
        return _fork(shape, ctx=ctx, copies=_log(rng, 1, min(8, max(1, (1 << 18) // ctx))), n=n,
                     kept=rng.randint(0, n))
    d = shape[0]
    return _seam(d, shape[1], n=_log(rng, 1, 4096), rotary=rng.choice([d, d, d // 2, d // 4]),
                 interleaved=rng.random() < 0.4, norm=rng.random() < 0.7, bias=rng.random() < 0.4,
                 table=rng.choice([8192, 8192, 131072]))


# -- the rows of a cache -------------------------------------------------------------------


def _planes(c):
    """(first byte of the row, width) of each plane: the key, value and norm fields in 16-byte pieces."""
    kbytes, vbytes = c["d"] * c["key_bits"] // 8, c["d"] * c["value_bits"] // 8
    out = []
    for lo, hi in ((0, kbytes), (kbytes, kbytes + vbytes), (kbytes + vbytes, kbytes + vbytes + 4)):
        out += [(a, min(16, hi - a)) for a in range(lo, hi, 16)]
    return out


def _span(capacity):
    return -(-capacity * 16 // 4096) * 4096


def _pack(codes, bits):
    """LSB-first codes: 8 of them are `bits` bytes."""
    x = codes.reshape(*codes.shape[:-1], -1, 8).long()
    word = (x << (torch.arange(8, device=x.device) * bits)).sum(-1)
    return ((word[..., None] >> (8 * torch.arange(bits, device=x.device))) & 255).to(torch.uint8).flatten(-2)


def _random_rows(c, gen, n):
    """n packed rows: Gaussian codes, norms around 2.2 (rows with outlier channels)."""
    dev = gen.device
    fields = []
    for bits in (c["key_bits"], c["value_bits"]):
        x = torch.randn((n, c["d"]), device=dev, generator=gen)
        codes = torch.bucketize(x, torch.tensor(BOUNDS[bits], device=dev, dtype=torch.float32) / 32768.0)
        fields.append(_pack(codes, bits))
    norms = (2.2 * 512 * torch.exp(0.1 * torch.randn((n, 2), device=dev, generator=gen))).round().long()
    return torch.cat(fields + [((norms[..., None] >> torch.tensor([0, 8], device=dev)) & 255).to(torch.uint8).flatten(-2)], -1)


def _image(c, gen, lens, capacity):
    """The plane image of a batch, (batch, n_kv, planes, span) bytes: rows for each sequence's
    length, zeros behind them."""
    planes = _planes(c)
    img = torch.zeros((len(lens), c["n_kv"], len(planes), _span(capacity)), dtype=torch.uint8, device="cuda")
    for b, n in enumerate(lens):
        if not n:
            continue
        rows = _random_rows(c, gen, n * c["n_kv"]).reshape(c["n_kv"], n, -1)
        for p, (lo, w) in enumerate(planes):
            img[b, :, p, :n * w] = rows[:, :, lo:lo + w].reshape(c["n_kv"], n * w)
    return img


def _cache(c, img, lens, capacity):
    from insitu_amd import CompressedCache, QuantConfig
    cache = CompressedCache(c["n_kv"], c["d"], capacity, QuantConfig(key_bits=c["key_bits"], value_bits=c["value_bits"]),
                            batch=len(lens), n_q_heads=N_Q)
    for b, n in enumerate(lens):
        cache.load_image(img[b].reshape(-1).cpu().numpy(), b)
        cache.set_length(n, b)
    return cache


def _lengths(c):
    """Ragged lengths of a batch, ctx / 8 to ctx, the longest in full."""
    b, ctx = c["batch"], c["ctx"]
    if b == 1 or (c["d"] == 128 and ctx >= 32768):
        return [ctx] * b
    lens = np.random.default_rng(3).integers(max(1, ctx // 8), ctx + 1, size=b)
    lens[b // 2] = ctx
    return [int(x) for x in lens]


def _parents(c, seed):
    n, b = c["n"], c["batch"]
    if c["tree"] == "chain":
        p = np.tile(np.arange(n) - 1, (b, 1))
    elif c["tree"] == "binary":
        p = np.tile((np.arange(n) - 1) // 2, (b, 1))
        p[:, 0] = -1
    elif c["tree"] == "star":
        p = np.full((b, n), -1)
    else:
        p = np.random.default_rng(seed).integers(-1, np.maximum(np.arange(n), 0), size=(b, n), endpoint=False) \
            if n > 1 else np.full((b, n), -1)
    return p.astype(np.int32)


def _accepted(parents, keep, rng):
    """A path of `keep` nodes for each sequence where there is one so deep, else nodes in order."""
    b, n = parents.shape
    rows = np.empty((b, keep), np.int32)
    for i in range(b):
        depth, path = 0, None
        for node in rng.permutation(n):
            p, j = [], int(node)
            while j >= 0:
                p.append(j)
                j = int(parents[i, j])
            if len(p) >= keep:
                path = p[::-1][:keep]
                break
        rows[i] = path if path else np.sort(rng.choice(n, keep, replace=False))
    return rows


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if c["kind"] == "seam":
        return _prepare_seam(c, gen)
    dev = "cuda"
    s = {"c": c}
    if c["kind"] == "fork":
        lens = [c["ctx"]] + [0] * c["copies"]
        capacity = c["ctx"] + 64
        img = _image(c, gen, lens, capacity)
        if c["n"]:
            order = torch.rand(c["n"], device=dev, generator=gen).argsort()[:c["kept"]]
            s["rows"] = order.sort().values.to(torch.int32)
    else:
        ctx = _lengths(c)
        tail = c["keep"] or c["n"]                       # a turn's cache holds the rows kept a turn before
        lens = [x + tail for x in ctx]
        capacity = max(ctx) + c["n"] + 64
        img = _image(c, gen, lens, capacity)
        scale = 2.2 * 65536 / (math.sqrt(c["d"]) if c["scaled"] else 1.0)
        rows = (c["batch"], c["n"])
        s["q"] = (torch.randn(rows + (N_Q, c["d"]), device=dev, generator=gen) * scale).round().to(torch.int32)
        parents = _parents(c, seed)
        s["parents"] = torch.from_numpy(parents).to(dev)
        if c["keep"]:
            for k in "kv":
                s[k] = (torch.randn(rows + (c["n_kv"], c["d"]), device=dev, generator=gen) * 2.2 * 65536).round().to(torch.int32)
            s["rows"] = torch.from_numpy(_accepted(parents, c["keep"], np.random.default_rng(seed))).to(dev)
        s["ctx"] = ctx
    s["lens"] = lens
    if own:
        from insitu_amd import CompressedAttention
        s["cache"] = _cache(c, img, lens, capacity)
        s["attn"] = CompressedAttention(s["cache"])
    else:
        s["img"] = img
    return s


def run(s):
    c = s["c"]
    if c["kind"] == "seam":
        return _run_seam(s)
    if own:
        cache = s["cache"]
        if c["kind"] == "fork":
            dst = list(range(1, c["copies"] + 1))
            if c["n"]:
                cache.fork(0, dst, n=c["n"], rows=s["rows"])
            else:
                cache.fork(0, dst)
            return cache.device_image()[1:]
        if c["kind"] == "tree":
            return s["attn"].attend_tree(s["q"], s["parents"], c["mode"], stats=False)[0]
        cache.keep(c["keep"])                            # none of them: the tail is dropped
        cache.append_rotated(s["k"], s["v"]) if c["batch"] > 1 else cache.append_rotated(s["k"][0], s["v"][0], seq=0)
        out, _ = s["attn"].attend_tree(s["q"], s["parents"], c["mode"], stats=False)
        cache.keep(c["n"], s["rows"])
        return {"out": out, "image": cache.device_image()}
    if c["kind"] == "fork":
        return _plain_fork(c, s)
    if c["kind"] == "tree":
        return _plain_tree(c, s["img"], s["ctx"], s["q"], s["parents"])
    _plain_append(c, s["img"], s["ctx"], s["k"], s["v"])
    out = _plain_tree(c, s["img"], s["ctx"], s["q"], s["parents"])
    _plain_keep(c, s["img"], s["ctx"], s["rows"])
    return {"out": out, "image": s["img"].flatten(1)}


# -- the plain forms -------------------------------------------------------------------------


def _plain_fork(c, s):
    img, ctx = s["img"], c["ctx"]
    head = ctx - c["n"]
    for p, (_, w) in enumerate(_planes(c)):
        src = img[0, :, p]
        img[1:, :, p, :head * w] = src[:, :head * w]
        if c["n"]:
            tail = src[:, head * w:ctx * w].reshape(c["n_kv"], c["n"], w)[:, s["rows"].long()]
            img[1:, :, p, head * w:(head + c["kept"]) * w] = tail.reshape(c["n_kv"], -1)
    return img[1:].flatten(1)


def _plain_keep(c, img, ctx, rows):
    for b, base in enumerate(ctx):
        for p, (_, w) in enumerate(_planes(c)):
            tail = img[b, :, p, base * w:(base + c["n"]) * w].reshape(c["n_kv"], c["n"], w)
            img[b, :, p, base * w:(base + c["keep"]) * w] = tail[:, rows[b].long()].reshape(c["n_kv"], -1)


def _plain_append(c, img, ctx, k, v):
    """Norm (the root mean square, floored, rounded half to even into Q9), codes by thresholds, packed."""
    d = c["d"]
    fields, norms = [], []
    for x, bits in ((k, c["key_bits"]), (v, c["value_bits"])):
        x = x.long()
        ms = torch.div((x * x).sum(-1), d, rounding_mode="floor")
        r = ms.double().sqrt().long()
        r = torch.where(r * r > ms, r - 1, r)
        r = torch.where((r + 1) * (r + 1) <= ms, r + 1, r)
        half = r & 127
        n = (r >> 7) + ((half > 64) | ((half == 64) & ((r >> 7) & 1 == 1))).long()
        n = n.clamp(max=32767)
        codes = torch.zeros_like(x)
        for b in BOUNDS[bits]:
            codes += (x << 8) > n[..., None] * b
        fields.append(_pack(codes, bits))
        norms.append(n)
    nn = torch.stack(norms, -1)
    rows = torch.cat(fields + [((nn[..., None] >> torch.tensor([0, 8], device=nn.device)) & 255).to(torch.uint8).flatten(-2)], -1)
    rows = rows.transpose(1, 2)                              # (batch, n_kv, n, row bytes)
    for b, base in enumerate(ctx):
        for p, (lo, w) in enumerate(_planes(c)):
            img[b, :, p, base * w:(base + c["n"]) * w] = rows[b, :, :, lo:lo + w].reshape(c["n_kv"], -1)


def _rows(c, img, t0, t1):
    """Row bytes (batch, n_kv, t1 - t0, row bytes) of the plane image."""
    return torch.cat([img[:, :, p, t0 * w:t1 * w].reshape(img.shape[0], img.shape[1], t1 - t0, w)
                      for p, (_, w) in enumerate(_planes(c))], -1)


def _codes(field, bits, d):
    """The codes of LSB-first fields: code i is in bits [i b, (i + 1) b)."""
    pos = torch.arange(d, device=field.device) * bits
    lo = field[..., pos >> 3].int()
    hi = field[..., ((pos >> 3) + 1).clamp(max=field.shape[-1] - 1)].int()
    return (((hi << 8) | lo) >> (pos & 7).int()) & ((1 << bits) - 1)


def _lut(delta):
    """2^15 exp(-delta / 2^16) from 256 values an octave."""
    table = torch.exp2(-torch.arange(256, dtype=torch.float64, device=delta.device) / 256).mul(32768).round().long()
    u = (delta.clamp(max=DELTA_MAX) * LOG2E) >> 24
    return torch.where(u < LUT_SPAN, table[u & 255] >> (u >> 8).clamp(max=16), 0)


def _finish(acc, l):
    """acc / l by a 32-bit reciprocal of l's leading bits."""
    k = torch.frexp(l.clamp(min=1).double())[1].long() - 1 - 31
    ln = torch.where(k >= 0, l >> k.clamp(min=0), l << (-k).clamp(min=0))
    r = torch.where(l > 0, torch.div(torch.full_like(l, 1 << 62), ln.clamp(min=1), rounding_mode="floor"), 0)
    return ((acc * r[..., None]) >> (47 + k)[..., None]).to(torch.int32)


def _plain_tree(c, img, ctx, q, parents, step=2048):
    dev = q.device
    b, n, d, h = c["batch"], c["n"], c["d"], c["n_kv"]
    g = N_Q // h
    two = c["mode"] == "two_pass"
    kbytes, vbytes = d * c["key_bits"] // 8, d * c["value_bits"] // 8
    kc = torch.tensor(CENTROIDS[c["key_bits"]], dtype=torch.float64, device=dev)
    vc = CENTROIDS[c["value_bits"]]
    base = torch.tensor(ctx, device=dev)
    # up[b, i, j]: node j is node i or an ancestor of it
    up = torch.zeros((b, n, n), dtype=torch.bool, device=dev)
    at = torch.arange(n, device=dev).expand(b, n)
    depth = torch.ones((b, n), dtype=torch.long, device=dev)
    for _ in range(n):
        live = at >= 0
        up |= torch.nn.functional.one_hot(at.clamp(min=0), n).bool() & live[..., None]
        at = torch.where(live, parents.long().gather(1, at.clamp(min=0)), at)
        if not bool((at >= 0).any()):
            break
    # query rows in the order (node, head of the group) of each KV head
    qr = q.reshape(b, n, h, g, d).permute(0, 2, 1, 3, 4).reshape(b * h, n * g, d).double()
    total = max(ctx) + n

    def scores(t0, t1):
        rows = _rows(c, img, t0, t1)
        keys = kc[_codes(rows[..., :kbytes], c["key_bits"], d)].reshape(b * h, t1 - t0, d)
        norm = rows[..., kbytes + vbytes:].int()
        kn = (norm[..., 0] | norm[..., 1] << 8).short().long()
        vn = (norm[..., 2] | norm[..., 3] << 8).short().long()
        dot = torch.bmm(qr, keys.transpose(1, 2).contiguous()).long()
        sc = ((dot * kn.reshape(b * h, 1, -1)) >> 24).clamp(SCORE_LO, -SCORE_LO - 1)
        t = torch.arange(t0, t1, device=dev)
        rel = t[None] - base[:, None]                        # (batch, rows): the node a row holds
        node = rel.clamp(0, n - 1)[:, None].expand(b, n, t1 - t0)
        seen = (rel < 0)[:, None] | (up.gather(2, node) & ((rel >= 0) & (rel < n))[:, None])
        seen = seen[:, None, :, None].expand(b, h, n, g, t1 - t0).reshape(b * h, n * g, t1 - t0)
        return sc, seen, vn.reshape(b * h, 1, -1), rows

    m = torch.full((b * h, n * g), SCORE_LO, dtype=torch.long, device=dev)
    acc = torch.zeros((b * h, n * g, d), dtype=torch.long, device=dev)
    l = torch.zeros((b * h, n * g), dtype=torch.long, device=dev)
    if two:
        for t0 in range(0, total, step):
            sc, seen, _, _ = scores(t0, min(total, t0 + step))
            m = torch.maximum(m, torch.where(seen, sc, SCORE_LO).amax(-1))
    for t0 in range(0, total, step):
        t1 = min(total, t0 + step)
        sc, seen, vn, rows = scores(t0, t1)
        hot = torch.nn.functional.one_hot(_codes(rows[..., kbytes:kbytes + vbytes], c["value_bits"], d).long(),
                                          len(vc)).reshape(b * h, t1 - t0, d, len(vc))
        hot = [hot[..., i].double().contiguous() for i in range(len(vc))]
        if two:
            p, seg, last = torch.where(seen, _lut(m[..., None] - sc), 0), None, 0
        else:
            sm = torch.where(seen, sc, SCORE_LO)
            top = torch.cummax(torch.cat([m[..., None], sm], -1), -1).values
            before, after = top[..., :-1], top[..., 1:]
            grew = sm > before
            seg = grew.long().cumsum(-1)
            f = torch.where(grew, _lut(torch.where(grew, sm - before, 0)), 0)
            p = torch.where(seen, _lut(torch.where(seen, after - sm, 0)), 0)
            last, m = int(seg[..., -1].max()), after[..., -1]
        for e in range(last + 1):
            if e:
                fe = torch.where(seg == e, f, 0).sum(-1)
                has = seg[..., -1] >= e
                acc = torch.where(has[..., None], (acc * fe[..., None]) >> 15, acc)
                l = torch.where(has, (l * fe) >> 15, l)
            pe = p if seg is None else torch.where(seg == e, p, 0)
            l = l + pe.sum(-1)
            w = vn * pe
            for i, cv in enumerate(vc):
                acc = acc + torch.bmm(((w * cv) >> 23).double(), hot[i]).long()
    out = _finish(acc.clamp(ACC_LO, ACC_HI), l)
    return out.reshape(b, h, n, g, d).permute(0, 2, 1, 3, 4).reshape(b, n, N_Q, d).contiguous()


# -- the seam ----------------------------------------------------------------------------------


def _angles(c):
    half = c["rotary"] // 2
    inv = 1.0 / (500000.0 ** (np.arange(half) * 2.0 / c["rotary"]))
    return np.arange(c["table"])[:, None] * inv[None]


def _prepare_seam(c, gen):
    dev = "cuda"
    d, h = c["d"], c["n_kv"]
    heads = N_Q + 2 * h
    s = {"c": c}
    # a projection's outputs: of unit scale with a few channels that stand out
    big = 1.0 + 7.0 * (torch.rand((heads, d), device=dev, generator=gen) < 0.05)
    s["p"] = (torch.randn((c["n"], heads, d), device=dev, generator=gen) * big * 0.7).reshape(c["n"], heads * d)
    first = int(torch.randint(0, c["table"] - c["n"] + 1, (1,), device=dev, generator=gen))
    depth = torch.arange(c["n"], device=dev) if c["n"] > 64 else torch.randint(0, c["n"], (c["n"],), device=dev, generator=gen)
    s["pos"] = first + depth
    w = [1.0 + 0.3 * torch.randn(d, device=dev, generator=gen) for _ in range(2)] if c["norm"] else [None, None]
    bias = 0.2 * torch.randn(heads * d, device=dev, generator=gen) if c["bias"] else None
    if own:
        from insitu_amd import ModelConfig, Seam
        model = ModelConfig(hidden_size=N_Q * d, num_heads=N_Q, num_kv_heads=h, head_dim=d, rope_theta=500000.0,
                            max_position=c["table"], rotary_dim=c["rotary"], rope_interleaved=c["interleaved"],
                            qk_norm_eps=1e-6)
        s["seam"] = Seam(model, q_norm=w[0], k_norm=w[1], bias=bias)
    else:
        ang = torch.from_numpy(_angles(c))
        s["cos"], s["sin"] = ((f(ang) * 32768).round().to(dev) for f in (torch.cos, torch.sin))
        s["w"], s["bias"] = w, bias
    return s


def _run_seam(s):
    if own:
        return s["seam"].wire(s["p"], s["pos"], counts=False)
    c = s["c"]
    d, r, n = c["d"], c["rotary"], c["n"]
    p = s["p"] if s["bias"] is None else s["p"] + s["bias"]
    x = p.double().reshape(n, -1, d)
    cos, sin = (s[k][s["pos"]][:, None] / 32768 for k in ("cos", "sin"))
    out = []
    for i, y in enumerate((x[:, :N_Q], x[:, N_Q:N_Q + c["n_kv"]], x[:, N_Q + c["n_kv"]:])):
        if i < 2:
            if c["norm"]:
                y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * s["w"][i].double()
            if i == 0:
                y = y * (1.0 / math.sqrt(d))
            rot, rest = y[..., :r], y[..., r:]
            a, b = (rot[..., 0::2], rot[..., 1::2]) if c["interleaved"] else (rot[..., :r // 2], rot[..., r // 2:])
            a, b = a * cos - b * sin, a * sin + b * cos
            rot = torch.stack([a, b], -1).flatten(-2) if c["interleaved"] else torch.cat([a, b], -1)
            y = torch.cat([rot, rest], -1)
        out.append((y * 65536).round().clamp(-(1 << 23), (1 << 23) - 1).to(torch.int32))
    return tuple(out)


# -- what the operators are, in 64 bits, written apart ------------------------------------------


def exact(case, seed):
    global own
    c = dict(case)
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    if c["kind"] == "seam":
        return _exact_seam(c, s)
    if c["kind"] == "fork":
        img = s["img"].cpu().numpy()
        keep = np.arange(c["ctx"])
        if c["n"]:
            keep = np.concatenate([keep[:c["ctx"] - c["n"]], c["ctx"] - c["n"] + s["rows"].cpu().numpy()])
        out = np.zeros_like(img[1:])
        for p, (_, w) in enumerate(_planes(c)):
            for b in range(c["copies"]):
                out[b, :, p, :len(keep) * w] = img[0, :, p].reshape(c["n_kv"], -1)[:, (keep[:, None] * w + np.arange(w)).reshape(-1)]
        return torch.from_numpy(out.reshape(c["copies"], -1))
    rows = c["batch"] * c["n"] * N_Q
    if (max(s["ctx"]) + c["n"]) * (1.5 if c["mode"] == "two_pass" else 1.0) * (200e-6 + rows * c["d"] * 1.2e-10) > 8:
        return None
    img = s["img"]
    if c["kind"] == "turn":
        img = img.clone()
        _exact_append(c, img, s)
    out = _exact_tree(c, img, s["ctx"], s["q"].long(), s["parents"].cpu().numpy())
    if c["kind"] == "tree":
        return out
    for b, base in enumerate(s["ctx"]):
        for p, (_, w) in enumerate(_planes(c)):
            old = img[b, :, p].clone()
            for j, r in enumerate(s["rows"][b].tolist()):
                img[b, :, p, (base + j) * w:(base + j + 1) * w] = old[:, (base + r) * w:(base + r + 1) * w]
    return {"out": out, "image": img.flatten(1)}


def _exact_append(c, img, s):
    """Rows on the host, in integers: a row's square root by math.isqrt."""
    bits, norms = [], []
    for x, w in ((s["k"], c["key_bits"]), (s["v"], c["value_bits"])):
        x = x.cpu().numpy().astype(np.int64)
        ms = np.einsum("...d,...d->...", x, x) // c["d"]
        r = np.array([math.isqrt(int(y)) for y in ms.reshape(-1)]).reshape(ms.shape)
        q = np.minimum(np.rint(r / 128.0).astype(np.int64), 32767)
        code = np.zeros(x.shape, np.uint8)
        for t in BOUNDS[w]:
            code += x * 256 > q[..., None] * t
        bits.append(np.unpackbits(code[..., None], axis=-1, bitorder="little")[..., :w].reshape(x.shape[:-1] + (-1,)))
        norms.append(q.astype("<i2"))
    rows = np.concatenate([np.packbits(np.concatenate(bits, -1), axis=-1, bitorder="little"),
                           np.stack(norms, -1).view(np.uint8)], -1)
    rows = torch.from_numpy(rows).to(img.device)
    for b, base in enumerate(s["ctx"]):
        for i in range(c["n"]):
            for p, (lo, w) in enumerate(_planes(c)):
                img[b, :, p, (base + i) * w:(base + i + 1) * w] = rows[b, i, :, lo:lo + w]


def _exact_tree(c, img, ctx, q, parents):
    """Row after row of the cache for every (sequence, KV head, node, head of the group) at once."""
    dev = q.device
    b, n, d, h = c["batch"], c["n"], c["d"], c["n_kv"]
    g = N_Q // h
    q = q.reshape(b, n, h, g, d).permute(0, 2, 1, 3, 4)
    chains = np.zeros((b, n, n), bool)
    for x in range(b):
        for i in range(n):
            chains[x, i, i] = True
            if parents[x, i] >= 0:
                chains[x, i] |= chains[x, parents[x, i]]
    total = max(ctx) + n
    seen = np.zeros((total, b, n), bool)
    for x in range(b):
        seen[:ctx[x], x] = True
        seen[ctx[x]:ctx[x] + n, x] = chains[x].T
    seen = torch.from_numpy(seen).to(dev)
    kc = torch.tensor(CENTROIDS[c["key_bits"]], device=dev)
    vc = torch.tensor(CENTROIDS[c["value_bits"]], device=dev)
    kbits, vbits = d * c["key_bits"], d * c["value_bits"]
    table = torch.tensor([round(2.0 ** (-i / 256) * 32768) for i in range(256)], device=dev)
    flat = torch.cat([table >> i for i in range(17)] + [torch.zeros(1, dtype=torch.long, device=dev)])
    eight = torch.arange(8, device=dev)

    def weight(delta):
        return flat[(delta.clamp(max=DELTA_MAX) * LOG2E >> 24).clamp(max=LUT_SPAN)]

    def block(t0, t1):                                   # decoded rows [t0, t1), by single bits
        by = torch.cat([img[:, :, p, t0 * w:t1 * w].unflatten(-1, (t1 - t0, w)) for p, (_, w) in enumerate(_planes(c))], -1)
        bit = ((by[..., None] >> eight) & 1).flatten(-2)
        key = (bit[..., :kbits].unflatten(-1, (d, -1)).long() << torch.arange(c["key_bits"], device=dev)).sum(-1)
        val = (bit[..., kbits:kbits + vbits].unflatten(-1, (d, -1)).long() << torch.arange(c["value_bits"], device=dev)).sum(-1)
        norm = (bit[..., kbits + vbits:].unflatten(-1, (2, 16)).long() << torch.arange(16, device=dev)).sum(-1)
        norm = torch.where(norm >= 1 << 15, norm - (1 << 16), norm)
        return kc[key], norm[..., 0], vc[val], norm[..., 1]

    m = torch.full((b, h, n, g), SCORE_LO, dtype=torch.long, device=dev)
    acc = torch.zeros((b, h, n, g, d), dtype=torch.long, device=dev)
    l = torch.zeros_like(m)
    for first in ([True, False] if c["mode"] == "two_pass" else [False]):
        for t0 in range(0, total, 256):
            t1 = min(total, t0 + 256)
            key, kn, val, vn = block(t0, t1)
            for t in range(t0, t1):
                i = t - t0
                s = (q * key[:, :, i, None, None]).sum(-1) * kn[:, :, i, None, None] >> 24
                s = s.clamp(SCORE_LO, -SCORE_LO - 1)
                on = seen[t][:, None, :, None]
                if c["mode"] != "two_pass":
                    f = torch.where(on & (s > m), weight((s - m).clamp(min=0)), 1 << 15)
                    acc = acc * f[..., None] >> 15
                    l = l * f >> 15
                if first or c["mode"] != "two_pass":
                    m = torch.where(on & (s > m), s, m)
                if first:
                    continue
                p = torch.where(on, weight((m - s).clamp(min=0)), 0)
                l = l + p
                acc = acc + ((vn[:, :, i, None, None] * p)[..., None] * val[:, :, i, None, None] >> 23)
                if c["mode"] != "two_pass":
                    acc = acc.clamp(ACC_LO, ACC_HI)
    acc = acc.clamp(ACC_LO, ACC_HI).cpu().numpy()
    l = l.cpu().numpy()
    k = np.frexp(l.astype(np.float64))[1].astype(np.int64) - 32
    ln = np.where(k >= 0, l >> np.maximum(k, 0), l << np.maximum(-k, 0))
    r = (1 << 62) // np.maximum(ln, 1)
    out = acc * r[..., None] >> (47 + k)[..., None]
    return torch.from_numpy(np.ascontiguousarray(out.transpose(0, 2, 1, 3, 4)).reshape(b, n, N_Q, d).astype(np.int32))


def _exact_seam(c, s):
    d, r, n = c["d"], c["rotary"], c["n"]
    p = s["p"].cpu().numpy()
    if s["bias"] is not None:
        p = p + s["bias"].cpu().numpy()
    x = p.astype(np.float64).reshape(n, -1, d)
    ang = _angles(c)
    pos = s["pos"].cpu().numpy()
    half = r // 2
    lo = np.arange(half) * 2 if c["interleaved"] else np.arange(half)
    hi = lo + 1 if c["interleaved"] else lo + half
    cos = np.rint(np.cos(ang[pos]) * 32768)[:, None] / 32768
    sin = np.rint(np.sin(ang[pos]) * 32768)[:, None] / 32768
    got, at = [], 0
    for i, heads in enumerate((N_Q, c["n_kv"], c["n_kv"])):
        y = x[:, at:at + heads].copy()
        at += heads
        if i < 2 and c["norm"]:
            ms = np.einsum("nhd,nhd->nh", y, y) / d
            y = y / np.sqrt(ms + 1e-6)[..., None] * s["w"][i].cpu().numpy().astype(np.float64)
        if i == 0:
            y *= 1.0 / math.sqrt(d)
        if i < 2:
            a, b = y[..., lo].copy(), y[..., hi].copy()
            y[..., lo] = a * cos - b * sin
            y[..., hi] = a * sin + b * cos
        got.append(torch.from_numpy(np.clip(np.rint(y * 65536), -(1 << 23), (1 << 23) - 1).astype(np.int32)))
    return tuple(got)


def work(case):
    c = case
    d = c["d"]
    if c["kind"] == "seam":
        heads = N_Q + 2 * c["n_kv"]
        # the projections in, the wire rows out, a row of each table a token, the norms' weights
        by = c["n"] * (heads * d * 8 + c["rotary"] * 8) + (8 * d if c["norm"] else 0) + (4 * heads * d if c["bias"] else 0)
        return {"bytes": by, "flops": c["n"] * (N_Q + c["n_kv"]) * (3 * c["rotary"] + (4 * d if c["norm"] else 0))}
    row = d * (c["key_bits"] + c["value_bits"]) // 8 + 4
    if c["kind"] == "fork":
        n = c["ctx"] - c["n"] + (c["kept"] if c["n"] else 0)
        return {"bytes": n * c["n_kv"] * row * (1 + c["copies"]), "flops": 0}
    rows, seen = 0, 0
    for ctx in _lengths(c):
        rows += ctx + c["n"]
        seen += (ctx + 1) * c["n"]
    by = rows * c["n_kv"] * row + 2 * 4 * c["batch"] * c["n"] * N_Q * d
    if c["kind"] == "turn":
        # the drafted rows in, and the accepted ones moved
        by += c["batch"] * c["n_kv"] * (c["n"] * (8 * d + row) + 2 * c["keep"] * row)
    return {"bytes": by, "flops": 4 * seen * N_Q * d}
