"""GPU: tree attends whose row tiles ask for a few runs more than a tile holds (4,096 beside the spans' first
ones, where few tiles share the scratch). Rows of one tile differ: most of them find their runs and are put
together from them, while others ask too late and go token by token. Every row is the oracle's, whichever they are."""

import numpy as np
import pytest

from oracle import native

from test_gpu_tree import FORMATS, N_KV, _cache, _check, _fill

pytestmark = pytest.mark.gpu

EXTRA, NODES, SPANS_IN_ONE = 4096, 4, 8


def _span(rows):
    """Tokens a wave walks: an eighth of a context of one launch, 64 of a longer one."""
    return -(-(-(-rows // SPANS_IN_ONE)) // 16) * 16 if rows <= 512 else 64


def _demand(s, n):
    """Runs that rows of scores s (rows, tokens) ask for over n tokens and the tree's nodes behind them: an event a run,
    but in the first span. (A node's own row may be one more.)"""
    before = np.maximum.accumulate(s[:, :n], -1)
    return int((s[:, 1:n] > before[:, :-1])[:, _span(n + NODES) - 1:].sum())


@pytest.mark.parametrize("fmt", [FORMATS[0], FORMATS[5]])
@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("seed", range(12))
def test_a_tile_that_runs_out_for_some_rows(ctx, fmt, long, seed):
    from insitu_amd.attention import CompressedAttention
    d, G = fmt[0], fmt[3]
    assert NODES * G == 16                              # a KV head is one whole row tile
    rng = np.random.default_rng(seed)
    most = 1400 if long else 512 - NODES
    u = np.where(np.arange(d) % 3 == 0, -65536.0, 65536.0)
    k = u * (0.5 + 0.02 * np.arange(most + NODES))[:, None, None]
    k = k + rng.standard_normal((most + NODES, N_KV, d)) * (9000 if long or d == 64 else 2500)
    v = np.rint(rng.standard_normal((1, most + NODES, N_KV, d)) * 65536).astype(np.int64)
    # every head climbs along u, more or less steadily
    noise = rng.uniform(0.5, (18.0 if d == 64 else 9.0) if long else 3.0, (1, NODES, N_KV * G, 1)) / 32
    q = np.rint(u / 32 + rng.standard_normal((1, NODES, N_KV * G, d)) * 65536 * noise).astype(np.int64)
    # as many tokens as ask for a few runs too many of the first KV head's tile
    trial = _cache(ctx, fmt, [most])
    hosts, f = _fill(trial, fmt, [most], np.rint(k[None, :most]).astype(np.int64), v[:, :most])
    s, _ = native.scores(q[0, :, :G].reshape(-1, d), hosts[0].view(0), f)
    n = next((n for n in range(513 - NODES if long else 256, most) if _demand(s, n) > EXTRA + seed % 4), None)
    assert n is not None and _demand(s, n) <= EXTRA + 300
    rows = np.rint(np.concatenate([k[:n], -k[n:n + NODES]])[None]).astype(np.int64)
    lens = [n + NODES]
    c = _cache(ctx, fmt, lens)
    hosts, f = _fill(c, fmt, lens, rows, v)
    parents = np.full((1, NODES), -1)
    out, st = CompressedAttention(c).attend_tree(q, parents, "online")
    _check(out.cpu().numpy(), st, q, hosts, f, G, lens, parents, NODES, "online", serial=None)
    assert st.serial_fallbacks >= 1
