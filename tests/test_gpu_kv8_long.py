"""The loops that long contexts live in, against 64 bits: rings that are refilled many times, barriers whose parity flips,
block-table entries fetched anew, accumulators rescaled late, sums loaded a page ahead. Few blocks and few splits give each
warp many pages at lengths that a plain computation can check. Tolerances as in test_gpu_kv8."""
import numpy as np
import pytest

from test_gpu_kv8 import BLOCK, FMTS, TOL, TOL_LSE, attention64, build, dev, rel_err, rows_of, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("qh,kvh,d,ctx,m,window,splits", [
    (32, 8, 64, 5000, 16, 0, 1),      # 64 rows: 40 tiles of 128 keys in one block
    (16, 4, 128, 6000, 16, 0, 1),     # 47 tiles
    (8, 2, 64, 20000, 16, 0, 1),      # 157 tiles: four more rounds of block-table entries
    (8, 2, 64, 20000, 16, 9000, 3),   # a window that starts inside a page
    (8, 1, 128, 9001, 32, 0, 2),      # 256 rows
    (8, 2, 64, 20000, 1, 0, 1),       # 8 rows: 79 pages per warp, two more rounds of entries
    (8, 2, 128, 16000, 1, 0, 1),      # 42 pages per warp, one more round
    (8, 2, 64, 20000, 3, 0, 1),       # 16 rows
    (16, 4, 128, 14000, 3, 0, 1),
    (8, 2, 64, 9000, 8, 5000, 1),     # 32 rows: two groups of 16
    (16, 4, 128, 6000, 8, 0, 1),      # the same at head_dim 128: 16 pages per warp
    (16, 4, 128, 32768, 8, 0, 0),     # the default splits
])
def test_attention(la, synth, cuda, fmt, qh, kvh, d, ctx, m, window, splits):
    import torch

    K, V = rows_of(synth, ctx + m, ctx + m, kvh, d)
    q = synth.Stream(ctx + 7).normal_f16((m, qh, d))
    cache = build(la, cuda, fmt, K, V, ctx)
    lse = torch.zeros((m, qh), dtype=torch.float32, device=cuda)
    got = cache.verify(dev(q, cuda), ctx, window=window, lse=lse, splits=splits)
    la.sync()
    sealed = ctx // BLOCK * BLOCK
    want, wl = attention64(q, values(K, sealed, fmt), values(V, sealed, fmt), ctx, window)
    assert rel_err(got.cpu().numpy(), want) < TOL
    assert np.max(np.abs(lse.cpu().numpy() - wl) / np.maximum(1, np.abs(wl))) < TOL_LSE


def rising(synth, n, m, qh, kvh, d):
    """Scores that grow along the keys, V blocks of very different scales."""
    K, V = rows_of(synth, 6 + d, n, kvh, d)
    K = (K.astype(np.float32) * np.linspace(0.01, 12, n)[:, None, None]).astype(np.float16)
    scale = 10.0 ** np.random.RandomState(2).randint(-4, 3, (n + BLOCK - 1) // BLOCK)
    V = (V.astype(np.float32) * scale.repeat(BLOCK)[:n, None, None]).astype(np.float16)
    q = (synth.Stream(9 + d).normal_f16((m, qh, d)).astype(np.float32) * 4).astype(np.float16)
    return K, V, q


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("m", [1, 3, 16])
@pytest.mark.parametrize("splits", [1, 4])
def test_attention_rising_scores(la, synth, cuda, fmt, d, m, splits):
    """The running maximum moves again and again, also once accumulators hold something."""
    ctx, kvh, qh = 2500, 2, 8
    K, V, q = rising(synth, ctx + m, m, qh, kvh, d)
    cache = build(la, cuda, fmt, K, V, ctx)
    got = cache.verify(dev(q, cuda), ctx, splits=splits)
    la.sync()
    sealed = ctx // BLOCK * BLOCK
    want, _ = attention64(q, values(K, sealed, fmt), values(V, sealed, fmt), ctx)
    assert rel_err(got.cpu().numpy(), want) < TOL


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_rising_scores(la, synth, cuda, fmt, d):
    ctx, t, kvh, qh = 2000, 50, 2, 8
    K, V, q = rising(synth, ctx + t, t, qh, kvh, d)
    cache = build(la, cuda, fmt, K, V, ctx + t)
    got = cache.prefill(dev(q, cuda), ctx)
    la.sync()
    sealed = (ctx + t) // BLOCK * BLOCK
    want, _ = attention64(q, values(K, sealed, fmt), values(V, sealed, fmt), ctx)
    assert rel_err(got.cpu().numpy(), want) < TOL


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("qh,kvh,d,ctx,m,window", [
    (32, 32, 64, 20000, 1, 0),      # on 148 SMs 9 rounds of pages per warp
    (32, 32, 128, 9000, 2, 0),      # 4 rounds, a ring of two stages
    (32, 32, 64, 7456, 32, 0),      # 32 rows: three whole rounds, then pages whose rows four warps share
    (64, 32, 128, 7456, 16, 3000),
    (64, 32, 64, 12500, 16, 0),     # 32 rows, too many rounds for sharing
])
def test_key_weights(la, synth, cuda, fmt, qh, kvh, d, ctx, m, window):
    import torch

    n, g = ctx + m, qh // kvh
    K, V = rows_of(synth, n, n, kvh, d)
    q = (synth.Stream(n + 3).normal_f16((m, qh, d)).astype(np.float32) * 2).astype(np.float16)
    cache = build(la, cuda, fmt, K, V, ctx)
    qd = dev(q, cuda)
    lse = torch.empty((m, qh), dtype=torch.float32, device=cuda)
    cache.verify(qd, ctx, window=window, lse=lse)
    prev = dev(np.random.RandomState(n).rand(kvh, n).astype(np.float32), cuda)
    got = cache.key_weights(qd, lse, ctx, window=window)
    more = cache.key_weights(qd, lse, ctx, window=window, prev=prev, decay=0.25)
    la.sync()
    z = lse.cpu().numpy().astype(np.float64)
    Kv = values(K, ctx // BLOCK * BLOCK, fmt)
    pos = ctx + np.arange(m)[:, None]
    key = np.arange(n)[None, :]
    seen = (key <= pos) & ((key > pos - window) if window else True)
    want = np.zeros((kvh, n))
    for h in range(qh):
        s = q[:, h].astype(np.float64) @ Kv[:, h // g].T / np.sqrt(d)
        want[h // g] += np.where(seen, np.exp(s - z[:, h, None]), 0).sum(0)

    def off(a, b):
        return np.max(np.clip(np.abs(a - b) - 1e-4 * np.abs(b), 0, None)) / np.sqrt(np.mean(b ** 2))

    got, more, p = got.cpu().numpy(), more.cpu().numpy(), prev.cpu().numpy()
    assert off(got, want) < 2e-5
    assert np.allclose(got.sum(axis=1), m * g, rtol=1e-4)
    assert off(more, want + 0.25 * p) < 2e-5
