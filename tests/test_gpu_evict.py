"""Eviction on the GPU: which keys stay (exactly the plain rule's, ties and special values included) and their move into
a smaller 8-bit cache (codes sealed anew, bit by bit)."""
import numpy as np
import pytest

from test_gpu_kv8 import BLOCK, FMTS, TOL, attention64, build, dev, finite16, mode, quantise, rows_of, values

pytestmark = pytest.mark.gpu


def keep_plain(w, budget, sink, recent):
    """Ascending kept positions of one row: NaN is the smallest, -0 equals 0, ties go to the lower position."""
    n = len(w)
    key = np.where(np.isnan(w), -np.inf, w.astype(np.float64))
    nan = np.isnan(w)
    mid = sorted(range(sink, n - recent), key=lambda i: (nan[i], -key[i], i))[:budget - sink - recent]
    return np.array(sorted(list(range(sink)) + mid + list(range(n - recent, n))), dtype=np.int32)


def rows_for(kind, heads, n, seed):
    r = np.random.RandomState(seed)
    if kind == "skewed":
        return (r.rand(heads, n) ** 8).astype(np.float32)
    if kind == "equal":
        return np.full((heads, n), 0.25, np.float32)
    if kind == "few":   # many ties across the threshold
        return r.randint(0, 4, (heads, n)).astype(np.float32)
    if kind == "zeros":
        return np.where(r.rand(heads, n) < 0.5, 0.0, -0.0).astype(np.float32)
    w = r.randn(heads, n).astype(np.float32)   # negative values, infinities, NaN, subnormals
    for v in (np.inf, -np.inf, np.nan, 1e-40, -1e-40, -0.0):
        w[r.rand(heads, n) < 0.05] = v
    return w


@pytest.mark.parametrize("kind", ["skewed", "equal", "few", "zeros", "special"])
@pytest.mark.parametrize("heads,n,budget,sink,recent", [
    (1, 1, 1, 0, 0), (2, 7, 3, 1, 1), (3, 33, 32, 0, 32), (8, 1000, 250, 4, 64), (4, 5003, 2047, 1, 100),
    (2, 40000, 10001, 0, 0), (3, 300, 300, 5, 60), (3, 300, 65, 5, 60), (1, 70000, 69999, 0, 0), (1, 9000, 1, 0, 0)])
def test_select(la, cuda, kind, heads, n, budget, sink, recent):
    w = rows_for(kind, heads, n, n + budget)
    pad = np.full((heads, n + 5), np.float32(1e30))   # a row stride: what lies past a row is not looked at
    pad[:, :n] = w
    keep, kept = la.evict_select(dev(pad, cuda), n, budget, sink, recent)
    la.sync()
    keep, kept = keep.cpu().numpy(), kept.cpu().numpy()
    for h in range(heads):
        want = keep_plain(w[h], budget, sink, recent)
        assert np.array_equal(keep[h], want), h
        assert np.array_equal(kept[h], w[h][want], equal_nan=True)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,d,n,committed,budget,sink,recent", [
    (3, 64, 300, 300, 100, 4, 40), (4, 128, 300, 290, 64, 0, 30), (2, 64, 1000, 990, 999, 1, 50),
    (2, 128, 96, 96, 96, 0, 0), (1, 64, 40, 40, 5, 1, 2), (2, 64, 2000, 1990, 33, 1, 30)])
def test_evict_moves_values(la, synth, cuda, fmt, heads, d, n, committed, budget, sink, recent):
    K, V = rows_of(synth, n + d, n, heads, d)
    cache = build(la, cuda, fmt, K, V, committed)
    w = rows_for("skewed", heads, n, n)
    dst = build(la, cuda, fmt, K[:0], V[:0], 0, capacity=budget + 40)
    keep, _ = cache.evict(dev(w, cuda), budget, sink, recent, dst)
    gk, gv = dst.read(0, budget)
    la.sync()
    sealed = committed // BLOCK * BLOCK
    full = budget // BLOCK * BLOCK
    assert (dst.length, dst.sealed) == (budget, full)
    keep = keep.cpu().numpy()
    for got, x in ((gk, K), (gv, V)):
        x = values(x, sealed, fmt).astype(np.float32)
        for h in range(heads):
            assert np.array_equal(keep[h], keep_plain(w[h], budget, sink, recent))
            rows = x[keep[h], h]
            for b in range(full // BLOCK):
                _, c, s = quantise(rows[b * BLOCK:(b + 1) * BLOCK], fmt)
                rows[b * BLOCK:(b + 1) * BLOCK] = c * s
            assert np.array_equal(got.cpu().numpy()[:, h], rows.astype(np.float16))


@pytest.mark.parametrize("fmt", FMTS)
def test_attention_goes_on_after_eviction(la, synth, cuda, fmt):
    """attend, add up weights, evict, append at the slots after the kept ones, attend: against 64 bits over the kept
    values."""
    import torch

    heads, d, qh, n, m, budget = 2, 64, 8, 900, 4, 200
    K, V = rows_of(synth, 3, n + m, heads, d)
    q = synth.Stream(9).normal_f16((m, qh, d))
    cache = build(la, cuda, fmt, K[:n], V[:n], n - m)
    lse = torch.empty((m, qh), dtype=torch.float32, device=cuda)
    qd = dev(q, cuda)
    cache.verify(qd, n - m, lse=lse)
    w = cache.key_weights(qd, lse, n - m)
    dst = la.LayerCache8(mode(la, fmt), heads, d, budget + 64, device=cuda)
    keep, _ = cache.evict(w, budget, 4, 32, dst)
    dst.append(dev(K[n:], cuda), dev(V[n:], cuda), draft=True)
    got = dst.verify(qd, budget)
    la.sync()
    gk, gv = dst.read(0, budget)
    keep = keep.cpu().numpy()
    sealed = (n - m) // BLOCK * BLOCK
    rows = {}
    for name, x in (("k", K), ("v", V)):
        val = values(x[:n], sealed, fmt).astype(np.float32)
        kept = np.stack([val[keep[h], h] for h in range(heads)], axis=1)
        for b in range(budget // BLOCK):
            for h in range(heads):
                _, c, s = quantise(kept[b * BLOCK:(b + 1) * BLOCK, h], fmt)
                kept[b * BLOCK:(b + 1) * BLOCK, h] = c * s
        tail = kept[budget // BLOCK * BLOCK:].astype(np.float16)
        rows[name] = np.concatenate([kept[:budget // BLOCK * BLOCK], tail.astype(np.float32),
                                     finite16(x[n:])]).astype(np.float64)
    la.sync()
    want, _ = attention64(q, rows["k"], rows["v"], budget)
    err = np.max(np.abs(got.cpu().numpy() - want)) / np.sqrt(np.mean(want ** 2))
    assert err < TOL + 2.0 ** -9
    del gk, gv


def test_kernels_from_the_cubin(la, synth, cuda):
    """The committed kernel image runs the 8-bit cache and eviction with the same bits as the linked kernels."""
    import torch

    def once():
        K, V = rows_of(synth, 55, 700, 2, 64)
        q = dev(synth.Stream(56).normal_f16((4, 8, 64)), cuda)
        cache = build(la, cuda, "int8", K, V, 690)
        lse = torch.empty((4, 8), dtype=torch.float32, device=cuda)
        out = cache.verify(q, 696, lse=lse)
        w = cache.key_weights(q, lse, 696)
        dst = la.LayerCache8(la.MODE_I8BLK, 2, 64, 200, device=cuda)
        keep, kept = cache.evict(w, 150, 2, 32, dst)
        k, v = dst.read(0, 150)
        p = cache.prefill(dev(synth.Stream(57).normal_f16((60, 8, 64)), cuda), 640)
        la.sync()
        return [x.cpu() for x in (out, lse, w, keep, kept, k, v, p)]

    want = once()
    la.load_cubin()
    try:
        got = once()
        assert la.cubin_launches() >= 8
    finally:
        la.unload_cubin()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
