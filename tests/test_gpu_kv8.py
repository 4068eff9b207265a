"""The 8-bit block cache (MODE_I8BLK, MODE_E4M3BLK) on the GPU: append and sealing, rollback, reading back, attention,
prefill and per-key attention weights, against plain restatements (codes bit by bit, attention in 64 bits over the
values the codes stand for).

Tolerances: attention output 2e-3 of its RMS beyond half an fp16 ulp, as the other verify kernels' (P is rounded to fp16:
at most 2^-11 of the largest product sum, some 5e-4); log-sum-exp 2e-5 times max(1, |lse|) (fp32 scores of up to 128
products, ex2 and log2 to about 2 ulp each); weights 2e-5 of their RMS beyond 1e-4 of each (an fp32 exponent of up to 64
is good to 2^-18)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TOL, TOL_LSE = 2e-3, 2e-5
BLOCK, TAIL = 32, 128
FMTS = ["int8", "e4m3"]


def mode(la, fmt):
    return la.MODE_I8BLK if fmt == "int8" else la.MODE_E4M3BLK


def dev(a, cuda):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).to(cuda)


def rel_err(got, want):
    want = want.astype(np.float64)
    rms = float(np.sqrt(np.mean(want ** 2)))
    half_ulp = 0.5 * np.abs(np.spacing(want.astype(np.float16))).astype(np.float64)
    return float(np.max(np.clip(np.abs(got.astype(np.float64) - want) - half_ulp, 0.0, None))) / rms


def finite16(x):
    x = np.where(np.isnan(x), np.float16(0), x)
    return np.clip(x.astype(np.float32), -65504, 65504)


def quantise(x, fmt):
    """One block and head, fp32 [32][D]: (codes as uint8, values as fp32 code values, scale)."""
    import torch

    top = np.float32(np.max(np.abs(x)))
    scale = np.float32(1) if top == 0 else np.float32(top / np.float32(127 if fmt == "int8" else 448))
    y = (x.astype(np.float32) / scale).astype(np.float32)
    if fmt == "int8":
        c = np.clip(np.rint(y), -127, 127).astype(np.int8)
        return c.view(np.uint8) ^ 0x80, c.astype(np.float32), scale   # stored plus 128
    t = torch.from_numpy(np.clip(y, -448, 448)).to(torch.float8_e4m3fn)
    return t.view(torch.uint8).numpy(), t.float().numpy(), scale


def values(x, sealed, fmt):
    """The fp64 values of fp16 rows [n][heads][D], the first `sealed` of them in 8 bits."""
    out = finite16(x).astype(np.float64)
    for b in range(sealed // BLOCK):
        for h in range(x.shape[1]):
            rows = slice(b * BLOCK, (b + 1) * BLOCK)
            _, v, s = quantise(finite16(x[rows, h]), fmt)
            out[rows, h] = (v * s).astype(np.float32)
    return out


def section_codes(sec, D):
    """The K and V codes [32][D] and the scales of a section's bytes, by the documented layout."""
    key, dim = np.arange(BLOCK)[:, None], np.arange(D)[None, :]
    k = (((key // 16 * 2 + key // 8 % 2) * (D // 64) + dim // 64) * 32 + key % 8 * 4 + dim // 16 % 4) * 16 + dim % 16
    v = ((key // 16 * (D // 32) + dim // 32) * 32 + dim % 8 * 4 + key % 8 // 2) * 16 + dim // 16 % 2 * 8 \
        + dim // 8 % 2 * 4 + key // 8 % 2 * 2 + key % 2
    return sec[32 + k], sec[32 + 32 * D + v], sec[:8].copy().view(np.float32)


def attention64(q, K, V, ctx, window=0, gate=None):
    """(out, lse) of q [m][qh][D] at ctx.. over fp64 K, V [n][heads][D]."""
    m, qh, d = q.shape
    g = qh // K.shape[1]
    out, lse = np.zeros((m, qh, d)), np.zeros((m, qh))
    for t in range(m):
        lo = max(0, ctx + t - window + 1) if window else 0
        for h in range(qh):
            s = K[lo:ctx + t + 1, h // g] @ q[t, h].astype(np.float64) / np.sqrt(d)
            p = np.exp(s - s.max())
            lse[t, h] = s.max() + np.log(p.sum())
            out[t, h] = p / p.sum() @ V[lo:ctx + t + 1, h // g]
    if gate is not None:
        out = out / (1 + np.exp(-gate.astype(np.float64)))[:, :, None]
    return out, lse


def rows_of(synth, seed, n, heads, d):
    s = synth.Stream(seed)
    return s.normal_f16((n, heads, d)), s.normal_f16((n, heads, d))


def build(la, cuda, fmt, K, V, committed, capacity=None, permute=True, poison=True):
    """A cache of the rows, `committed` of them final, on a permuted block table; unused pool and tail bytes poisoned."""
    import torch

    n, heads, d = K.shape
    capacity = capacity or n + 64
    logical = (capacity + BLOCK - 1) // BLOCK
    table = torch.from_numpy(np.random.RandomState(n).permutation(logical + 3)[:logical].astype(np.int32)).to(cuda) \
        if permute else None
    cache = la.LayerCache8(mode(la, fmt), heads, d, capacity, device=cuda, block_table=table, pool_blocks=logical + 3)
    if poison:   # NaN in the tail, NaN scales and codes in the pool
        cache.pool.fill_(0xff)
        cache.tail.fill_(0xff)
    if committed:
        cache.append(dev(K[:committed], cuda), dev(V[:committed], cuda))
    if n > committed:
        cache.append(dev(K[committed:], cuda), dev(V[committed:], cuda), draft=True)
    return cache


# ------------------------------------------------------------------ append, seal, read
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,d", [(3, 64), (4, 128)])
def test_append_bytes(la, synth, cuda, fmt, heads, d):
    """Chunks of odd lengths (one of them sealing tokens of the tail while later ones reuse its slots): every sealed
    code and scale, and the values read back, bit by bit; special rows: zeros, one large value, infinities, NaN."""
    steps = [1, 30, 5, 64, 300, 31, 128, 7]
    n = sum(steps)
    K, V = rows_of(synth, 900 + d, n, heads, d)
    K[64:96] = 0
    V[96:128, 1] = np.float16(0)
    V[100, 1, 3] = np.float16(-6e-8)
    K[130, 0, :4] = [np.inf, -np.inf, np.nan, 60000]
    V[n - 1, 0, :3] = [np.nan, np.inf, -np.inf]
    cache = build(la, cuda, fmt, K[:0], V[:0], 0, capacity=n)
    at = 0
    for s in steps:
        cache.append(dev(K[at:at + s], cuda), dev(V[at:at + s], cuda))
        at += s
    la.sync()
    assert cache.length == n and cache.sealed == n // BLOCK * BLOCK
    pool, table = cache.pool.cpu().numpy(), cache.table.cpu().numpy()
    lay = cache.layout
    for b in range(cache.sealed // BLOCK):
        for h in range(heads):
            at = int(table[b]) * lay.block_bytes + h * lay.head_bytes
            kc, vc, sc = section_codes(pool[at:at + lay.head_bytes], d)
            rows = slice(b * BLOCK, (b + 1) * BLOCK)
            for got, s, x in ((kc, sc[0], K), (vc, sc[1], V)):
                want, _, scale = quantise(finite16(x[rows, h]), fmt)
                assert s == scale and np.array_equal(got, want), (b, h)
    for pos0, count in ((0, n), (cache.sealed - 3, n - cache.sealed + 3), (n - 1, 1), (17, 40)):
        gk, gv = cache.read(pos0, count)
        la.sync()
        for got, x in ((gk, K), (gv, V)):
            want = values(x, cache.sealed, fmt)[pos0:pos0 + count].astype(np.float16)
            assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d", [64, 128])
def test_append_norm_rope_matches_f16_cache(la, synth, cuda, fmt, d):
    """k-norm, RoPE and a strided source: the K that is quantised is the fp16 K of the MODE_F16 cache."""
    heads, n = 4, 77
    stream = synth.Stream(31)
    raw = dev(stream.normal_f16((n, heads * d * 2 + 8)), cuda)
    kn = dev(stream.normal_f16((d,)), cuda)
    rope = dev(la.rope_table(1e6, 0.5 if d == 128 else 1.0, d, n).view(np.float16), cuda)
    k, v = raw[:, :heads * d], raw[:, heads * d:2 * heads * d]
    f16 = la.LayerCache(la.MODE_F16, heads, d, n, device=cuda)
    f16.append(k, v, 0, rope=rope, k_norm=kn, token_stride=raw.stride(0))
    cache = la.LayerCache8(mode(la, fmt), heads, d, n, device=cuda)
    cache.append(k[:50], v[:50], rope=rope, k_norm=kn, token_stride=raw.stride(0))
    cache.append(k[50:], v[50:], rope=rope, k_norm=kn, token_stride=raw.stride(0))
    la.sync()
    K = f16.logical()["K"].view(np.float16)
    V = f16.logical()["V"].view(np.float16)
    gk, gv = cache.read(0, n)
    la.sync()
    assert np.array_equal(gk.cpu().numpy(), values(K, 64, fmt).astype(np.float16))
    assert np.array_equal(gv.cpu().numpy(), values(V, 64, fmt).astype(np.float16))


@pytest.mark.parametrize("fmt", FMTS)
def test_rollback_leaves_no_trace(la, synth, cuda, fmt):
    """Rounds of drafts with rejections: sealed bytes and live values are those of the accepted tokens alone."""
    heads, d, total = 2, 64, 230
    K, V = rows_of(synth, 77, total, heads, d)
    junkK, junkV = rows_of(synth, 78, 64, heads, d)
    cache = build(la, cuda, fmt, K[:40], V[:40], 40, capacity=300, permute=False, poison=False)
    rng = np.random.RandomState(5)
    at = 40
    while at < total - 32:
        m = int(rng.randint(1, 33))
        keep = int(rng.randint(1, m + 1))
        dk, dv = junkK[:m].copy() * np.float16(50), junkV[:m].copy() * np.float16(50)
        dk[:keep], dv[:keep] = K[at:at + keep], V[at:at + keep]
        cache.append(dev(dk, cuda), dev(dv, cuda), draft=True)
        cache.truncate(at + keep)
        at += keep
    cache.append(dev(K[at:total], cuda), dev(V[at:total], cuda))
    plain = build(la, cuda, fmt, K, V, total, capacity=300, permute=False, poison=False)
    la.sync()
    assert cache.sealed == plain.sealed == total // BLOCK * BLOCK
    used = cache.sealed // BLOCK * cache.layout.block_bytes
    assert np.array_equal(cache.pool.cpu().numpy()[:used], plain.pool.cpu().numpy()[:used])
    for a, b in zip(cache.read(0, total), plain.read(0, total)):
        assert np.array_equal(a.cpu().numpy(), b.cpu().numpy())


# ------------------------------------------------------------------ attention
GEOMS = [(32, 8, 64), (16, 4, 128)]
ATTEND = [
    # q_heads, kv_heads, D, ctx, m, window, gate, splits
    (32, 8, 64, 0, 1, 0, False, 0),
    (32, 8, 64, 31, 1, 0, True, 0),
    (16, 4, 128, 32, 1, 0, False, 0),
    (32, 8, 64, 777, 1, 0, False, 0),
    (16, 4, 128, 1500, 2, 0, False, 0),
    (32, 8, 64, 1023, 3, 0, True, 0),
    (16, 4, 128, 999, 4, 0, True, 3),
    (32, 8, 64, 2100, 5, 0, False, 0),
    (16, 4, 128, 700, 8, 0, True, 0),
    (32, 8, 64, 1311, 8, 0, False, 5),
    (32, 8, 64, 650, 16, 0, False, 0),
    (16, 4, 128, 517, 16, 0, False, 0),
    (32, 8, 64, 95, 32, 0, False, 0),
    (16, 4, 128, 200, 32, 0, True, 2),
    (16, 4, 128, 600, 8, 100, False, 0),    # window edges inside pages
    (32, 8, 64, 500, 1, 1, False, 0),       # a token that sees itself alone
    (32, 8, 64, 500, 4, 3, False, 4),       # a window shorter than the round; splits that some rows never see
    (32, 8, 64, 300, 16, 64, False, 0),
    (6, 6, 64, 333, 7, 0, False, 0),        # no sharing
    (14, 2, 128, 150, 3, 0, False, 0),      # 7 query heads per kv head
    (8, 1, 64, 400, 32, 0, True, 0),        # multi-query: 256 rows
    (32, 8, 64, 5000, 1, 0, False, 1),      # one split, several ring turns per warp
    (16, 4, 128, 5000, 9, 0, False, 1),
    (16, 4, 128, 3000, 1, 0, False, 90),    # more splits than usual, one page each
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("qh,kvh,d,ctx,m,window,gated,splits", ATTEND)
def test_attention(la, synth, cuda, fmt, qh, kvh, d, ctx, m, window, gated, splits):
    import torch

    K, V = rows_of(synth, ctx + m, ctx + m, kvh, d)
    q = synth.Stream(ctx + 7).normal_f16((m, qh, d))
    gate = synth.Stream(ctx + 8).normal_f16((m, qh)) if gated else None
    cache = build(la, cuda, fmt, K, V, ctx)
    wide = torch.zeros((m, qh * d + 8), dtype=torch.float16, device=cuda)   # rows with a stride
    wide[:, :qh * d] = dev(q, cuda).reshape(m, -1)
    lse = torch.zeros((m, qh), dtype=torch.float32, device=cuda)
    got = cache.verify(wide[:, :qh * d].unflatten(1, (qh, d)), ctx, window=window, lse=lse, splits=splits,
                       gate=None if gate is None else dev(gate, cuda))
    la.sync()
    sealed = ctx // BLOCK * BLOCK
    want, wl = attention64(q, values(K, sealed, fmt), values(V, sealed, fmt), ctx, window, gate)
    assert rel_err(got.cpu().numpy(), want) < TOL
    assert np.max(np.abs(lse.cpu().numpy() - wl) / np.maximum(1, np.abs(wl))) < TOL_LSE


@pytest.mark.parametrize("fmt", FMTS)
def test_attention_sealed_queries(la, synth, cuda, fmt):
    """A short chunk whose own tokens are sealed already, and later tokens beside them: causal masks inside pages."""
    ctx, m, n, qh, kvh, d = 50, 20, 150, 8, 2, 64
    K, V = rows_of(synth, 4, n, kvh, d)
    q = synth.Stream(5).normal_f16((m, qh, d))
    cache = build(la, cuda, fmt, K, V, n)
    got = cache.verify(dev(q, cuda), ctx)
    la.sync()
    want, _ = attention64(q, values(K, 128, fmt), values(V, 128, fmt), ctx)
    assert rel_err(got.cpu().numpy(), want) < TOL


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d", [64, 128])
def test_attention_rising_and_large_scores(la, synth, cuda, fmt, d):
    """Scores that grow along the keys (the running maximum moves often), V blocks of very different scales, scores
    far beyond fp32's exponent range once exponentiated."""
    ctx, m, kvh, qh = 1000, 3, 2, 8
    K, V = rows_of(synth, 6, ctx + m, kvh, d)
    K = (K.astype(np.float32) * np.linspace(0.01, 12, ctx + m)[:, None, None]).astype(np.float16)
    V = (V.astype(np.float32) * 10.0 ** np.random.RandomState(1).randint(-4, 3, (ctx + m + 31) // 32).repeat(32)[:ctx + m, None, None]).astype(np.float16)
    q = (synth.Stream(9).normal_f16((m, qh, d)).astype(np.float32) * 4).astype(np.float16)
    cache = build(la, cuda, fmt, K, V, ctx)
    for splits in (1, 4):
        got = cache.verify(dev(q, cuda), ctx, splits=splits)
        la.sync()
        sealed = ctx // BLOCK * BLOCK
        want, _ = attention64(q, values(K, sealed, fmt), values(V, sealed, fmt), ctx)
        assert rel_err(got.cpu().numpy(), want) < TOL


@pytest.mark.parametrize("fmt", FMTS)
def test_attention_nan_row_stays_alone(la, synth, cuda, fmt):
    ctx, m, kvh, qh, d = 300, 4, 2, 8, 64
    K, V = rows_of(synth, 16, ctx + m, kvh, d)
    q = synth.Stream(17).normal_f16((m, qh, d))
    q[1, 2, 5] = np.nan
    cache = build(la, cuda, fmt, K, V, ctx)
    got = cache.verify(dev(q, cuda), ctx).cpu().numpy()
    la.sync()
    assert np.isnan(got[1, 2]).all()
    q[1, 2, 5] = 0
    want, _ = attention64(q, values(K, 288, fmt), values(V, 288, fmt), ctx)
    other = np.ones((m, qh), dtype=bool)
    other[1, 2] = False
    assert rel_err(got[other], want[other]) < TOL


@pytest.mark.parametrize("fmt", FMTS)
def test_attention_other_stream_and_repeat(la, synth, cuda, fmt):
    """On a stream of its own, twice: the same bits (no atomics, no order of execution in the sums)."""
    import torch

    ctx, m, kvh, qh, d = 9000, 8, 4, 16, 128
    K, V = rows_of(synth, 26, ctx + m, kvh, d)
    q = dev(synth.Stream(27).normal_f16((m, qh, d)), cuda)
    cache = build(la, cuda, fmt, K, V, ctx)
    a = cache.verify(q, ctx)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = cache.verify(q, ctx)
    side.synchronize()
    la.sync()
    assert torch.equal(a, b)


# ------------------------------------------------------------------ prefill
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("qh,kvh,d,ctx,t,window", [
    (32, 8, 64, 0, 33, 0), (16, 4, 128, 0, 100, 0), (32, 8, 64, 45, 257, 0), (16, 4, 128, 300, 64, 0),
    (16, 4, 128, 500, 129, 100), (8, 2, 64, 61, 70, 33), (8, 2, 64, 40, 9, 0), (4, 4, 64, 20, 70, 0),
    (16, 2, 128, 10, 50, 40), (8, 2, 64, 1, 1, 0), (8, 2, 128, 2000, 40, 0)])
def test_prefill(la, synth, cuda, fmt, qh, kvh, d, ctx, t, window):
    n = ctx + t
    K, V = rows_of(synth, n, n, kvh, d)
    q = synth.Stream(n + 1).normal_f16((t, qh, d))
    cache = build(la, cuda, fmt, K, V, n)
    got = cache.prefill(dev(q, cuda), ctx, window=window)
    la.sync()
    sealed = n // BLOCK * BLOCK
    want, _ = attention64(q, values(K, sealed, fmt), values(V, sealed, fmt), ctx, window)
    assert rel_err(got.cpu().numpy(), want) < TOL


# ------------------------------------------------------------------ weights
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("qh,kvh,d,ctx,m,window", [
    (32, 8, 64, 0, 1, 0), (32, 8, 64, 500, 1, 0), (16, 4, 128, 333, 8, 0), (16, 4, 128, 90, 32, 0),
    (32, 8, 64, 200, 16, 70), (6, 6, 64, 100, 5, 0), (8, 1, 64, 77, 32, 0), (14, 2, 128, 3000, 3, 0)])
def test_key_weights(la, synth, cuda, fmt, qh, kvh, d, ctx, m, window):
    import torch

    n = ctx + m
    K, V = rows_of(synth, n, n, kvh, d)
    q = (synth.Stream(n + 3).normal_f16((m, qh, d)).astype(np.float32) * 2).astype(np.float16)
    cache = build(la, cuda, fmt, K, V, ctx)
    qd = dev(q, cuda)
    lse = torch.empty((m, qh), dtype=torch.float32, device=cuda)
    cache.verify(qd, ctx, window=window, lse=lse)
    prev = dev(np.random.RandomState(n).rand(kvh, n + 6).astype(np.float32), cuda)
    got = cache.key_weights(qd, lse, ctx, window=window)
    more = prev.clone()
    cache.key_weights(qd, lse, ctx, window=window, prev=more, decay=0.5, out=more)   # in place, a longer row stride
    la.sync()
    z = lse.cpu().numpy().astype(np.float64)
    Kv = values(K, ctx // BLOCK * BLOCK, fmt)
    want = np.zeros((kvh, n))
    g = qh // kvh
    for t in range(m):
        lo = max(0, ctx + t - window + 1) if window else 0
        for h in range(qh):
            s = Kv[lo:ctx + t + 1, h // g] @ q[t, h].astype(np.float64) / np.sqrt(d)
            want[h // g, lo:ctx + t + 1] += np.exp(s - z[t, h])
    got = got.cpu().numpy()

    def off(a, b):
        return np.max(np.clip(np.abs(a - b) - 1e-4 * np.abs(b), 0, None)) / np.sqrt(np.mean(b ** 2))

    assert off(got, want) < 2e-5
    assert np.allclose(got.sum(axis=1), m * g, rtol=1e-4)   # each row's weights sum to 1
    p = prev.cpu().numpy()
    assert off(more.cpu().numpy()[:, :n], want + 0.5 * p[:, :n]) < 2e-5
    assert np.array_equal(more.cpu().numpy()[:, n:], p[:, n:])
