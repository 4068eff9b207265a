"""Attention over an 8-bit cache whose V blocks differ in scale, on the GPU, against 64 bits over the values the codes
stand for: a block's share of the softmax sum does not depend on how large its V is.

Tolerance: TOL of test_gpu_kv8 (2e-3 of the RMS beyond half an fp16 ulp). Each product of the numerator carries P's
rounding to 11 bits, at most 2^-11 of it, and so does the sum. Where one key has all the weight the two cancel; where it
has some of it, an output is off by at most 2^-11 of itself, of which half an ulp (2^-12 at the least) is the output's
own: up to 8 RMS that is below 2e-3. Where many keys count, the roundings add up at random, to some 2^-12 of the RMS, 5
deviations of which stay below the same bound."""
import numpy as np
import pytest

from test_gpu_kv8 import BLOCK, FMTS, TOL, TOL_LSE, attention64, build, dev, rel_err, rows_of, values

pytestmark = pytest.mark.gpu


def uneven(synth, kind, n, m, qh, kvh, d, seed=0):
    """(K, V, q) of n keys and m query rows, scores of deviation 1 (the sink's apart)."""
    K, V = (x.astype(np.float32) for x in rows_of(synth, 300 + n + seed, n, kvh, d))
    q = synth.Stream(400 + n + seed).normal_f16((m, qh, d)).astype(np.float32)
    block = np.arange(n) // BLOCK
    if kind == "blocks":        # any of seven magnitudes
        V *= 10.0 ** np.random.RandomState(n).randint(-4, 3, block[-1] + 1)[block, None, None]
    elif kind == "alternate":   # half of the weight on blocks whose V is next to nothing
        V *= np.where(block % 2 == 1, 1e-6, 1.0)[:, None, None]
    elif kind == "sink":        # the first key has some 0.55 of the weight, and its block a V of 100
        q[:, :, :8], K[:, :, :8] = 2, 0
        K[0, :, :8] = np.log(2 * n) * np.sqrt(d) / 16
        V[:BLOCK] *= 100
    return K.astype(np.float16), V.astype(np.float16), q.astype(np.float16)


KINDS = ["blocks", "alternate", "sink"]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("m", [1, 3, 16])   # 4, 12 and 64 rows per kv head
def test_attention(la, synth, cuda, fmt, kind, d, m):
    ctx, qh, kvh = 1500, 8, 2
    K, V, q = uneven(synth, kind, ctx + m, m, qh, kvh, d)
    cache = build(la, cuda, fmt, K, V, ctx)
    sealed = ctx // BLOCK * BLOCK
    want, _ = attention64(q, values(K, sealed, fmt), values(V, sealed, fmt), ctx)
    for splits in (0, 1, 5):   # the default (one cluster where the rows are few), one block, split partials
        got = cache.verify(dev(q, cuda), ctx, splits=splits)
        la.sync()
        assert rel_err(got.cpu().numpy(), want) < TOL, splits


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("qh,kvh,d,ctx,t,window", [
    (8, 2, 64, 900, 100, 0), (8, 2, 128, 900, 100, 0),
    (8, 2, 64, 900, 70, 300), (8, 2, 128, 900, 70, 300),
    (4, 1, 64, 3000, 40, 0), (4, 1, 128, 3000, 40, 0)])   # few query tiles: the keys are split
def test_prefill(la, synth, cuda, fmt, kind, qh, kvh, d, ctx, t, window):
    n = ctx + t
    K, V, q = uneven(synth, kind, n, t, qh, kvh, d)
    cache = build(la, cuda, fmt, K, V, n)
    got = cache.prefill(dev(q, cuda), ctx, window=window)
    la.sync()
    sealed = n // BLOCK * BLOCK
    want, _ = attention64(q, values(K, sealed, fmt), values(V, sealed, fmt), ctx, window)
    assert rel_err(got.cpu().numpy(), want) < TOL


# ------------------------------------------------------------------ pages that must not drown the others' P
# A block of zeros has a scale of 1 and the open pages are fp16: next to small V neither may push the other pages' P to
# fp16's lower end, nor may a block whose large V nobody attends to. The tolerance is the one above: P has its 11 bits for
# keys down to 2^-21 of the largest product, and what is smaller is off by 2^-32 of that product.
def small(synth, kind, n, m, qh, kvh, d):
    K, V = (x.astype(np.float32) for x in rows_of(synth, 500 + n, n, kvh, d))
    q = synth.Stream(600 + n).normal_f16((m, qh, d)).astype(np.float32)
    if kind == "small":       # every V some 1e-3, the tail's too
        V *= 1e-3
    elif kind == "tiny":
        V *= 1e-4
    elif kind == "zeros":     # a block of zeros, one of negative zeros, and a head that is all zeros
        V *= 1e-3
        V[96:128], V[160:192, 0], V[:, 1] = 0, -0.0, 0
    elif kind == "zeros, tiny":
        V *= 1e-4
        V[64:128], V[:32, 1] = 0, 0
    elif kind == "zero tail":
        V[n // BLOCK * BLOCK - BLOCK:] = 0
        V *= 1e-3
    elif kind == "outlier":   # one key of V 1e4 times the others', with no weight
        V *= 1e-2
        V[70] *= 1e4
        q[:, :, 0], K[:, :, 0], K[70, :, 0] = 4, 0, -8 * np.sqrt(d)
    elif kind == "large":     # up to the largest fp16, the infinities beyond it stored as that
        V *= 2e4
    with np.errstate(over="ignore"):
        return K.astype(np.float16), V.astype(np.float16), q.astype(np.float16)


SMALL = ["small", "tiny", "zeros", "zeros, tiny", "zero tail", "outlier", "large"]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("kind", SMALL)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("m", [1, 3, 16])
def test_attention_small_v(la, synth, cuda, fmt, kind, d, m):
    import torch

    ctx, qh, kvh = 1500, 8, 2
    K, V, q = small(synth, kind, ctx + m, m, qh, kvh, d)
    cache = build(la, cuda, fmt, K, V, ctx)
    sealed = ctx // BLOCK * BLOCK
    want, wl = attention64(q, values(K, sealed, fmt), values(V, sealed, fmt), ctx)
    for splits in (0, 1, 5):
        lse = torch.empty((m, qh), dtype=torch.float32, device=cuda)
        got = cache.verify(dev(q, cuda), ctx, splits=splits, lse=lse)
        la.sync()
        assert rel_err(got.cpu().numpy(), want) < TOL, splits
        assert np.max(np.abs(lse.cpu().numpy() - wl) / np.maximum(1, np.abs(wl))) < TOL_LSE, splits
        if kind == "zeros":
            assert not got[:, qh // 2:].any()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("kind", SMALL)
@pytest.mark.parametrize("qh,kvh,d,ctx,t,window", [
    (8, 2, 64, 900, 90, 0), (8, 2, 128, 900, 90, 0), (8, 2, 64, 900, 70, 300), (8, 2, 128, 3000, 40, 0)])
def test_prefill_small_v(la, synth, cuda, fmt, kind, qh, kvh, d, ctx, t, window):
    n = ctx + t
    K, V, q = small(synth, kind, n, t, qh, kvh, d)
    cache = build(la, cuda, fmt, K, V, n)
    got = cache.prefill(dev(q, cuda), ctx, window=window)
    la.sync()
    sealed = n // BLOCK * BLOCK
    want, _ = attention64(q, values(K, sealed, fmt), values(V, sealed, fmt), ctx, window)
    assert rel_err(got.cpu().numpy(), want) < TOL
    if kind == "zeros":
        assert not got[:, qh // 2:].any()
