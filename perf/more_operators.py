"""The operators of layers with a sliding window, and of a cache taken over from floating rows and
handed back, as cases that can be timed and compared.

    window CompressedAttention.attend_window: the last n rows of each sequence are the queries'
           own; a query at row p attends the rows t <= p with t < sinks or t > p - window
    write  CompressedCache.append_float: floating keys and values of a dense cache (float32,
           float16 or bfloat16, tokens first or heads first) cast to Q8.16, rotated, quantised
           and packed behind each sequence (CompressedCache.keep drops the ones of the pass before)
    read   CompressedCache.read_float: the rows of a cache as floating keys and values in the
           model's own basis

The cache holds bit-packed rows: codes of Lloyd-Max centroids (Q1.15) and an int16 norm (Q9) for
keys and values, in planes of at most 16 bytes a row. Scores are floor(sum(q c) norm / 2^24) in
Q16; the weights come from a table, p = floor(2^15 2^-(i / 256)), i = floor(delta log2(e) 2^8);
a value adds floor(norm p c / 2^23) a channel. Online mode takes the rows in order and, when a
score passes the maximum so far, scales what it has by the table's value for the difference, with
a floor; two-pass mode takes the maximum of all first. A written row is the value times a diagonal
of signs times a Hadamard matrix over the square root of the width, floored; its norm is its root
mean square, floored, rounded half to even into Q9; its codes count the boundaries that are below.
All of that is integers. A row that is read back is the centroids times the norm, turned back by
the transposed matrix. Shapes are the repository's: 32 query heads of 64 over 8 KV heads (4-bit
keys, 2-bit values), over 4 KV heads with 3-bit keys, and 32 heads of 128 over 8 KV heads with
3-bit keys and values.
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
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _kv(shape):
    d, n_kv, kb, vb = shape
    return {"d": d, "n_kv": n_kv, "key_bits": kb, "value_bits": vb}


def _window(shape, *, ctx, n, window, sinks=0, batch=1, mode="online", scaled=True, name=None):
    """ctx: rows before the queries' own, of the longest sequence."""
    c = {"kind": "window", **_kv(shape), "ctx": ctx, "n": n, "window": window, "sinks": sinks, "batch": batch,
         "mode": mode, "scaled": scaled}
    return {"name": name, **c} if name else c


def _write(shape, *, ctx, n, type, batch=1, heads_first=True, name=None):
    """ctx: rows before the n that are written."""
    c = {"kind": "write", **_kv(shape), "ctx": ctx, "n": n, "type": type, "batch": batch, "heads_first": heads_first}
    return {"name": name, **c} if name else c


def _read(shape, *, ctx, n, type, batch=1, name=None):
    """ctx: rows before the n that are read, of the longest sequence."""
    c = {"kind": "read", **_kv(shape), "ctx": ctx, "n": n, "type": type, "batch": batch}
    return {"name": name, **c} if name else c


def listed():
    return [
        # a token of a short conversation, a narrow window: latency
        _window(SHAPES[0], ctx=300, n=1, window=128, sinks=4, name="window_step_ctx300"),
        # a token of each of a serving batch's ragged long conversations
        _window(SHAPES[0], ctx=32767, n=1, window=4096, sinks=4, batch=32, name="window_step_batch32"),
        # the same for 8 query heads a KV head in the adapter's softmax, peaked
        _window(SHAPES[1], ctx=2047, n=1, window=1024, batch=4, mode="two_pass", scaled=False,
                name="window_step_group8_two_pass"),
        # a prompt through a local layer
        _window(SHAPES[0], ctx=0, n=4096, window=1024, sinks=4, name="window_prompt_4096"),
        # a later turn of a few conversations, odd sizes, the adapter's softmax
        _window(SHAPES[3], ctx=2000, n=333, window=777, sinks=5, batch=3, mode="two_pass",
                name="window_turn_333_two_pass"),
        # a chunk of a long prompt, the larger heads
        _window(SHAPES[2], ctx=4096, n=4096, window=2048, sinks=16, name="window_chunk_d128_4096"),
        # a short prompt's keys and values taken over
        _write(SHAPES[0], ctx=100, n=65, type="bf16", name="write_65_bf16"),
        # a long conversation taken over from a dense cache, heads first as such a cache lies
        _write(SHAPES[0], ctx=0, n=32767, type="bf16", name="write_32767_bf16"),
        # the larger heads of a batch, tokens first, in single precision
        _write(SHAPES[2], ctx=33, n=1000, type="fp32", batch=4, heads_first=False,
               name="write_d128_1000_batch4_fp32"),
        # the last tokens' rows, looked at
        _read(SHAPES[0], ctx=200, n=100, type="fp32", name="read_100_fp32"),
        # a long conversation handed back to a dense cache
        _read(SHAPES[0], ctx=0, n=32767, type="bf16", name="read_32767_bf16"),
        # the larger heads of a batch, 4-bit keys
        _read(SHAPES[4], ctx=0, n=2047, type="fp16", batch=4, name="read_d128_2047_batch4_fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["window", "window", "window", "write", "read"])
    shape = rng.choice(SHAPES)
    if kind == "window":
        # a window's work is its queries times the rows each sees: no more than half the largest listed one's
        window, sinks = _log(rng, 1, 8192), rng.choice([0, rng.randint(1, 64)])
        ctx = _log(rng, 1, 65536) - 1
        room = 4096 * 2048 * 64 // (shape[0] * max(min(window, ctx + 1), 64))
        n = rng.choice([1, 1, _log(rng, 1, max(1, min(4096, room)))])
        batch = _log(rng, 1, max(1, min(64, room // n, (1 << 20) // (ctx + n))))
        return _window(shape, ctx=ctx, n=n, window=window, sinks=sinks, batch=batch,
                       mode=rng.choice(["online", "online", "two_pass"]), scaled=rng.random() < 0.6)
    # (an element is at most 4 bytes: half the largest listed rows)
    n = _log(rng, 1, 16384 * 64 // shape[0])
    batch = _log(rng, 1, max(1, min(16, 16384 * 64 // (shape[0] * n))))
    c = {"ctx": rng.choice([0, _log(rng, 1, 4096)]), "n": n, "type": rng.choice(list(TYPES)), "batch": batch}
    return _read(shape, **c) if kind == "read" else _write(shape, **c, heads_first=rng.random() < 0.7)


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
    x = codes.reshape(*codes.shape[:-1], -1, 8).int()
    word = (x << (torch.arange(8, device=x.device, dtype=torch.int32) * bits)).sum(-1)
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
    cache.device_image().copy_(img.flatten(1))
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        cache.set_length(n, b)
    return cache


def _lengths(c):
    """Rows before the last n of each sequence: ragged, ctx / 8 to ctx, the longest in full."""
    b, ctx = c["batch"], c["ctx"]
    if b == 1:
        return [ctx]
    lens = np.random.default_rng(3).integers(ctx // 8, ctx + 1, size=b)
    lens[b // 2] = ctx
    return [int(x) for x in lens]


def _signs(d):
    """The diagonal of a cache's rotation, as the quantisation's default seed gives it."""
    return np.random.Generator(np.random.PCG64(0)).integers(0, 2, size=(1, d))[0].astype(np.int64) * 2 - 1


def _hadamard(d):
    h = np.array([[1.0]])
    while h.shape[0] < d:
        h = np.block([[h, h], [h, -h]])
    return h


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    ctx = _lengths(c)
    lens = [x + c["n"] for x in ctx]
    capacity = max(lens) + 64
    s = {"c": c, "ctx": ctx, "lens": lens}
    d = c["d"]
    img = _image(c, gen, lens, capacity)
    rows = (c["batch"], c["n"])
    if c["kind"] == "window":
        scale = 2.2 * 65536 / (math.sqrt(d) if c["scaled"] else 1.0)
        s["q"] = (torch.randn(rows + (N_Q, d), device="cuda", generator=gen) * scale).round().to(torch.int32)
    elif c["kind"] == "write":
        # keys and values of unit scale with a few channels that stand out
        shape = (c["batch"], c["n_kv"], c["n"], d) if c["heads_first"] else rows + (c["n_kv"], d)
        for k in "kv":
            big = 1.0 + 7.0 * (torch.rand((c["n_kv"], 1, d), device="cuda", generator=gen) < 0.06)
            big = big if c["heads_first"] else big.transpose(0, 1)
            x = (torch.randn(shape, device="cuda", generator=gen) * big).to(TYPES[c["type"]])
            s[k] = x.transpose(1, 2) if c["heads_first"] else x
    if own:
        from insitu_amd import CompressedAttention
        s["cache"] = _cache(c, img, lens, capacity)
        s["attn"] = CompressedAttention(s["cache"])
    else:
        s["img"] = img
        h = torch.from_numpy(_hadamard(d)).float().cuda()
        s["signs"] = torch.from_numpy(_signs(d)).cuda()
        s["back"] = h * (s["signs"].float() / math.sqrt(d))       # a rotated row times this is the row
    return s


def run(s):
    c = s["c"]
    if own:
        cache = s["cache"]
        if c["kind"] == "window":
            return s["attn"].attend_window(s["q"], c["window"], c["sinks"], c["mode"], stats=False)[0]
        if c["kind"] == "write":
            cache.keep(c["n"])                               # none of them: the pass before's are dropped
            cache.append_float(s["k"], s["v"])
            return cache.device_image()
        return cache.read_float(min(s["ctx"]), c["n"], dtype=TYPES[c["type"]])
    if c["kind"] == "window":
        return _plain_window(c, s["img"], s["ctx"], s["q"])
    if c["kind"] == "write":
        _plain_write(c, s)
        return s["img"].flatten(1)
    return _plain_read(c, s)


# -- the plain forms -------------------------------------------------------------------------


def _plain_write(c, s):
    """Q8.16, signs and butterflies, the floor; the norm's square root; codes by thresholds; packed."""
    d, img = c["d"], s["img"]
    fields, norms = [], []
    for x, bits in ((s["k"], c["key_bits"]), (s["v"], c["value_bits"])):
        y = (x.float() * 65536.0).round().clamp(-(1 << 23), (1 << 23) - 1).int() * s["signs"].int()
        w = 1
        while w < d:
            y = y.reshape(*y.shape[:3], d // (2 * w), 2, w)
            y = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], -2).flatten(-3)
            w *= 2
        y = (y >> 3).long() if d == 64 else (y.long() * 2896) >> 15
        ms = (y * y).sum(-1) // d
        r = ms.double().sqrt().long()
        r = torch.where(r * r > ms, r - 1, r)
        r = torch.where((r + 1) * (r + 1) <= ms, r + 1, r)
        half = r & 127
        n = (r >> 7) + ((half > 64) | ((half == 64) & ((r >> 7) & 1 == 1))).long()
        n = n.clamp(max=32767)
        y = y << 8
        codes = torch.zeros(y.shape, dtype=torch.uint8, device=y.device)
        for b in BOUNDS[bits]:
            codes += y > n[..., None] * b
        fields.append(_pack(codes, bits))
        norms.append(n)
    nn = torch.stack(norms, -1)
    rows = torch.cat(fields + [((nn[..., None] >> torch.tensor([0, 8], device=nn.device)) & 255).to(torch.uint8).flatten(-2)], -1)
    rows = rows.transpose(1, 2)                              # (batch, n_kv, n, row bytes)
    for b, base in enumerate(s["ctx"]):
        for p, (lo, w) in enumerate(_planes(c)):
            img[b, :, p, base * w:(base + c["n"]) * w] = rows[b, :, :, lo:lo + w].reshape(c["n_kv"], -1)


def _take(c, img, at):
    """Row bytes (batch, n_kv, rows, row bytes) of rows at (batch, rows)."""
    out = []
    for p, (_, w) in enumerate(_planes(c)):
        plane = img[:, :, p, :img.shape[-1] // w * w].unflatten(-1, (-1, w))
        out.append(torch.stack([plane[b, :, at[b]] for b in range(len(at))]))
    return torch.cat(out, -1)


def _codes(field, bits, d):
    """The codes of LSB-first fields: code i is in bits [i b, (i + 1) b)."""
    pos = torch.arange(d, device=field.device) * bits
    lo = field[..., pos >> 3].int()
    hi = field[..., ((pos >> 3) + 1).clamp(max=field.shape[-1] - 1)].int()
    return (((hi << 8) | lo) >> (pos & 7).int()) & ((1 << bits) - 1)


def _fields(c, rows):
    """Key codes, value codes and the two norms of row bytes."""
    d = c["d"]
    kbytes, vbytes = d * c["key_bits"] // 8, d * c["value_bits"] // 8
    norm = rows[..., kbytes + vbytes:].int()
    return (_codes(rows[..., :kbytes], c["key_bits"], d), _codes(rows[..., kbytes:kbytes + vbytes], c["value_bits"], d),
            (norm[..., 0] | norm[..., 1] << 8).short(), (norm[..., 2] | norm[..., 3] << 8).short())


def _behind(c, s):
    """Which of the rows [min(ctx), min(ctx) + n) are behind a sequence's end: none."""
    t0 = min(s["ctx"])
    return torch.arange(t0, t0 + c["n"], device="cuda").expand(c["batch"], c["n"])


def _plain_read(c, s):
    kc, vc, kn, vn = _fields(c, _take(c, s["img"], _behind(c, s)))
    out = []
    for codes, norm, bits in ((kc, kn, c["key_bits"]), (vc, vn, c["value_bits"])):
        x = torch.tensor(CENTROIDS[bits], dtype=torch.float32, device=codes.device)[codes] @ s["back"]
        x = x * (norm.float() / (1 << 24))[..., None]
        out.append(x.transpose(1, 2).to(TYPES[c["type"]]))
    return tuple(out)


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


def _plain_window(c, img, ctx, q):
    """Blocks of queries; each over the rows that any of them sees, in steps."""
    some = max(1, 16384 // (c["batch"] * N_Q))
    return torch.cat([_plain_block(c, img, ctx, q, i, min(c["n"], i + some)) for i in range(0, c["n"], some)], 1)


def _plain_block(c, img, ctx, q, i0, i1):
    dev = q.device
    b, n, d, h = c["batch"], i1 - i0, c["d"], c["n_kv"]
    g = N_Q // h
    two = c["mode"] == "two_pass"
    kcent = torch.tensor(CENTROIDS[c["key_bits"]], dtype=torch.float64, device=dev)
    vcent = CENTROIDS[c["value_bits"]]
    base = torch.tensor(ctx, device=dev) + i0                # the first query's own row
    sinks = min(c["sinks"], max(ctx) + c["n"])
    window = min(c["window"], max(ctx) + c["n"])
    total = sinks + window + n - 1
    qr = q[:, i0:i1].reshape(b, n, h, g, d).permute(0, 2, 1, 3, 4).reshape(b * h, n * g, d).double()
    own_row = base[:, None] + torch.arange(n, device=dev)

    def scores(u0, u1):
        u = torch.arange(u0, u1, device=dev).expand(b, u1 - u0)
        t = torch.where(u < sinks, u, u - sinks + base[:, None] - window + 1)
        there = (t >= 0) & ((u < sinks) | (t >= sinks)) & (t < base[:, None] + n)
        t = torch.where(there, t, 0)
        kc, vcodes, kn, vn = _fields(c, _take(c, img, t))
        keys = kcent[kc].reshape(b * h, u1 - u0, d)
        dot = torch.bmm(qr, keys.transpose(1, 2).contiguous()).long()
        sc = ((dot * kn.long().reshape(b * h, 1, -1)) >> 24).clamp(SCORE_LO, -SCORE_LO - 1)
        t, p = t[:, None], own_row[..., None]
        seen = there[:, None] & (t <= p) & ((t < sinks) | (t > p - window))
        seen = seen[:, None, :, None].expand(b, h, n, g, u1 - u0).reshape(b * h, n * g, u1 - u0)
        return sc, seen, vn.long().reshape(b * h, 1, -1), vcodes.reshape(b * h, u1 - u0, d)

    steps = [0, min(total, 64)]
    while steps[-1] < total:
        steps.append(min(total, steps[-1] + 1024))
    m = torch.full((b * h, n * g), SCORE_LO, dtype=torch.long, device=dev)
    acc = torch.zeros((b * h, n * g, d), dtype=torch.long, device=dev)
    l = torch.zeros((b * h, n * g), dtype=torch.long, device=dev)
    if two:
        for u0, u1 in zip(steps, steps[1:]):
            sc, seen, _, _ = scores(u0, u1)
            m = torch.maximum(m, torch.where(seen, sc, SCORE_LO).amax(-1))
    for u0, u1 in zip(steps, steps[1:]):
        sc, seen, vn, vcodes = scores(u0, u1)
        hot = [(vcodes == i).double() for i in range(len(vcent))]
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
            for i, cv in enumerate(vcent):
                acc = acc + torch.bmm(((w * cv) >> 23).double(), hot[i]).long()
    out = _finish(acc.clamp(ACC_LO, ACC_HI), l)
    return out.reshape(b, h, n, g, d).permute(0, 2, 1, 3, 4).reshape(b, n, N_Q, d).contiguous()


# -- what the operators are, in 64 bits, written apart ------------------------------------------


def exact(case, seed):
    global own
    c = dict(case)
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    if c["kind"] == "read":
        return _exact_read(c, s)
    if c["kind"] == "write":
        if c["batch"] * c["n"] * c["n_kv"] * c["d"] > 1 << 24:
            return None
        return _exact_write(c, s)
    rows = c["batch"] * c["n"] * N_Q
    steps = min(c["window"], max(s["lens"])) + min(c["sinks"], max(s["lens"]))
    if steps * (1.5 if c["mode"] == "two_pass" else 1.0) * (400e-6 + rows * c["d"] * 1.5e-10) > 8:
        return None
    return _exact_window(c, s)


def _bits(c, s, at):
    """Codes and norms on the host, by single bits, of rows at[b] of each sequence: (batch, n_kv, rows, ...)."""
    img = s["img"].cpu().numpy()
    rows = max(s["lens"])
    by = np.stack([np.concatenate([img[b, :, p, :rows * w].reshape(c["n_kv"], rows, w)[:, at[b]]
                                   for p, (_, w) in enumerate(_planes(c))], -1) for b in range(c["batch"])])
    d, kb, vb = c["d"], c["key_bits"], c["value_bits"]
    bit = np.unpackbits(by, axis=-1, bitorder="little")
    kc = (bit[..., :d * kb].reshape(bit.shape[:-1] + (d, kb)) << np.arange(kb, dtype=np.uint8)).sum(-1, dtype=np.uint8)
    vc = (bit[..., d * kb:d * (kb + vb)].reshape(bit.shape[:-1] + (d, vb)) << np.arange(vb, dtype=np.uint8)).sum(-1, dtype=np.uint8)
    norm = np.ascontiguousarray(by[..., -4:]).view("<i2").astype(np.int64)
    return kc, vc, norm[..., 0], norm[..., 1]


def _exact_read(c, s):
    kc, vc, kn, vn = _bits(c, s, [min(s["ctx"]) + np.arange(c["n"])] * c["batch"])
    out = []
    turn = _hadamard(c["d"]) * _signs(c["d"])
    for codes, norm, bits in ((kc, kn, c["key_bits"]), (vc, vn, c["value_bits"])):
        x = np.array(CENTROIDS[bits], np.float64)[codes]
        x = (x @ turn) * (norm[..., None] / (16777216.0 * math.sqrt(c["d"])))
        out.append(torch.from_numpy(np.ascontiguousarray(x.transpose(0, 2, 1, 3))))
    return tuple(out)


def _exact_write(c, s):
    """Rows on the host, in integers: a row's square root by math.isqrt."""
    d = c["d"]
    bits, norms = [], []
    turn = (_hadamard(d) * _signs(d)).T
    for x, w in ((s["k"], c["key_bits"]), (s["v"], c["value_bits"])):
        x = np.rint(x.float().cpu().numpy().astype(np.float64) * 65536.0)
        y = (np.clip(x, -(1 << 23), (1 << 23) - 1) @ turn).astype(np.int64)
        y = y >> 3 if d == 64 else y * 2896 >> 15
        ms = np.einsum("...d,...d->...", y, y) // d
        r = np.array([math.isqrt(int(a)) for a in ms.reshape(-1)]).reshape(ms.shape)
        q = np.minimum(np.rint(r / 128.0).astype(np.int64), 32767)
        code = np.zeros(y.shape, np.uint8)
        for t in BOUNDS[w]:
            code += y * 256 > q[..., None] * t
        bits.append(np.unpackbits(code[..., None], axis=-1, bitorder="little")[..., :w].reshape(y.shape[:-1] + (-1,)))
        norms.append(q.astype("<i2"))
    rows = np.concatenate([np.packbits(np.concatenate(bits, -1), axis=-1, bitorder="little"),
                           np.stack(norms, -1).view(np.uint8)], -1)
    img = s["img"].cpu().numpy()
    for b, base in enumerate(s["ctx"]):
        for p, (lo, w) in enumerate(_planes(c)):
            img[b, :, p, base * w:(base + c["n"]) * w] = rows[b, :, :, lo:lo + w].transpose(1, 0, 2).reshape(c["n_kv"], -1)
    return torch.from_numpy(img.reshape(c["batch"], -1))


def _exact_window(c, s):
    """For every query at once: a visible row after the other, its first ones and then its window's."""
    dev = s["q"].device
    b, n, d, h = c["batch"], c["n"], c["d"], c["n_kv"]
    g = N_Q // h
    longest = max(s["lens"])
    sinks, window = min(c["sinks"], longest), min(c["window"], longest)
    # the first rows, and those from the first query's window on
    at = [np.concatenate([np.arange(sinks), np.maximum(np.arange(x - window + 1, x + n), 0)]) for x in s["ctx"]]
    kc, vc, kn, vn = (torch.from_numpy(x).to(dev) for x in _bits(c, s, at))
    kcent = torch.tensor(CENTROIDS[c["key_bits"]], device=dev)
    vcent = torch.tensor(CENTROIDS[c["value_bits"]], device=dev)
    table = torch.tensor([round(2.0 ** (-i / 256) * 32768) for i in range(256)], device=dev)
    flat = torch.cat([table >> i for i in range(17)] + [torch.zeros(1, dtype=torch.long, device=dev)])

    def weight(delta):
        return flat[(delta.clamp(max=DELTA_MAX) * LOG2E >> 24).clamp(max=LUT_SPAN)]

    q = s["q"].long().reshape(b, n, h, g, d).permute(0, 2, 1, 3, 4)
    query = torch.arange(n, device=dev)
    place = torch.tensor(s["ctx"], device=dev)[:, None] + query                               # (b, n)
    m = torch.full((b, h, n, g), SCORE_LO, dtype=torch.long, device=dev)
    acc = torch.zeros((b, h, n, g, d), dtype=torch.long, device=dev)
    l = torch.zeros_like(m)
    for first in ([True, False] if c["mode"] == "two_pass" else [False]):
        for i in range(sinks + window):
            # a first row that the window has left behind, or a row of the window
            on = i <= place - window if i < sinks else place - window + 1 + i - sinks >= 0
            j = torch.full_like(query, i) if i < sinks else query + i
            sc = (q * kcent[kc[:, :, j].long()][:, :, :, None]).sum(-1) * kn[:, :, j][..., None] >> 24
            sc = sc.clamp(SCORE_LO, -SCORE_LO - 1)
            on = on[:, None, :, None]
            if c["mode"] != "two_pass":
                f = torch.where(on & (sc > m), weight((sc - m).clamp(min=0)), 1 << 15)
                acc = acc * f[..., None] >> 15
                l = l * f >> 15
            if first or c["mode"] != "two_pass":
                m = torch.where(on & (sc > m), sc, m)
            if first:
                continue
            p = torch.where(on, weight((m - sc).clamp(min=0)), 0)
            l = l + p
            acc = acc + ((vn[:, :, j][..., None] * p)[..., None] * vcent[vc[:, :, j].long()][:, :, :, None] >> 23)
            if c["mode"] != "two_pass":
                acc = acc.clamp(ACC_LO, ACC_HI)
    acc = acc.clamp(ACC_LO, ACC_HI).cpu().numpy()
    l = l.cpu().numpy()
    k = np.frexp(l.astype(np.float64))[1].astype(np.int64) - 32
    ln = np.where(k >= 0, l >> np.maximum(k, 0), l << np.maximum(-k, 0))
    r = (1 << 62) // np.maximum(ln, 1)
    out = acc * r[..., None] >> (47 + k)[..., None]
    return torch.from_numpy(np.ascontiguousarray(out.transpose(0, 2, 1, 3, 4)).reshape(b, n, N_Q, d).astype(np.int32))


def work(case):
    c = case
    d = c["d"]
    row = d * (c["key_bits"] + c["value_bits"]) // 8 + 4
    if c["kind"] != "window":
        heads = c["batch"] * c["n"] * c["n_kv"]
        size = 4 if c["type"] == "fp32" else 2
        # butterflies; a comparison a bit of a code, or a product
        flops = heads * d * (2 * (d.bit_length() - 1) + c["key_bits"] + c["value_bits"])
        return {"bytes": heads * (2 * d * size + row), "flops": flops}
    rows, seen = 0, 0
    for ctx in _lengths(c):
        end = ctx + c["n"]
        first = max(0, ctx - c["window"] + 1)                # of the first query's window
        rows += end - first + min(c["sinks"], first)
        for p in range(ctx, end):
            lo = max(0, p - c["window"] + 1)
            seen += p + 1 - lo + min(c["sinks"], lo)
    return {"bytes": rows * c["n_kv"] * row + 2 * 4 * c["batch"] * c["n"] * N_Q * d, "flops": 4 * seen * N_Q * d}
