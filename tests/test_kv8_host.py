"""Host side of the 8-bit block cache and eviction, without a GPU: layouts, sizes, split counts, refusals (each before any
launch)."""
import ctypes

import pytest


@pytest.mark.parametrize("mode", [2, 3])
@pytest.mark.parametrize("h,d,head", [(8, 64, 4128), (4, 128, 8224)])
def test_layout(la, mode, h, d, head):
    lay = la.layout(mode, h, d)
    assert (lay.head_bytes, lay.block_bytes) == (head, head * h)
    assert la.lib().lfm3a_kv8_tail_bytes(ctypes.byref(lay)) == 2 * h * 128 * d * 2
    assert la.lib().lfm3a_kv8_tail_bytes(ctypes.byref(la.layout(0, h, d))) == 0


def test_section_layout_is_a_bijection():
    for D in (64, 128):
        k, v = set(), set()
        for key in range(32):
            for dim in range(D):
                k.add((((key // 16 * 2 + key // 8 % 2) * (D // 64) + dim // 64) * 32 + key % 8 * 4 + dim // 16 % 4) * 16
                      + dim % 16)
                v.add(((key // 16 * (D // 32) + dim // 32) * 32 + dim % 8 * 4 + key % 8 // 2) * 16 + dim // 16 % 2 * 8
                      + dim // 8 % 2 * 4 + key // 8 % 2 * 2 + key % 2)
        assert k == v == set(range(32 * D))


def view(la, mode=2, h=8, d=64, pool=64, tail=64):
    return la.Kv8View(la.KvView(pool, 64, 10, la.layout(mode, h, d)), tail)


def test_modes_do_not_mix(la):
    lib = la.lib()
    v8, f16 = view(la), la.KvView(64, 64, 10, la.layout(0, 8, 64))
    assert lib.lfm3a_kv_append(ctypes.byref(v8.kv), 64, 64, 0, 0, 1, None, None, None) == la.ENOTSUP
    assert lib.lfm3a_kv_truncate(ctypes.byref(v8.kv), 5, None) == la.ENOTSUP
    assert lib.lfm3a_verify_attention(ctypes.byref(v8.kv), 64, 1, 32, 10, 0, None, 64, None, 0, 1, None) == la.ENOTSUP
    assert lib.lfm3a_prefill_attention(ctypes.byref(v8.kv), 64, 10, 32, 0, 0, 1, 64, None, 0, None) == la.ENOTSUP
    bad = la.Kv8View(f16, 64)
    assert lib.lfm3a_kv8_append(ctypes.byref(bad), 64, 64, 0, 0, 1, 0, 0, None, None, None) == la.ENOTSUP
    with pytest.raises(la.LFM3AError):
        la.LayerCache8(la.MODE_F16, 8, 64, 100)


def test_append_refusals(la):
    lib = la.lib()

    def call(v, k=64, stride=0, pos0=0, n=1, sealed=0, seal_to=0):
        return lib.lfm3a_kv8_append(ctypes.byref(v), k, 64, stride, pos0, n, sealed, seal_to, None, None, None)

    assert lib.lfm3a_kv8_append(None, 64, 64, 0, 0, 1, 0, 0, None, None, None) == la.EINVAL
    assert call(view(la, tail=0)) == la.EINVAL
    assert call(view(la, tail=72)) == la.EINVAL          # misaligned
    v = view(la)
    assert call(v, k=None) == la.EINVAL
    assert call(v, n=-1) == la.EINVAL
    assert call(v, pos0=-1) == la.EINVAL
    assert call(v, stride=100) == la.EINVAL              # shorter than a token
    assert call(v, pos0=64, sealed=96) == la.EINVAL      # below the sealed tokens
    assert call(v, pos0=64, sealed=33, seal_to=64) == la.EINVAL
    assert call(v, pos0=64, n=4, seal_to=69) == la.EINVAL
    assert call(v, pos0=64, sealed=64, seal_to=32) == la.EINVAL
    assert call(v, pos0=200, sealed=32, seal_to=200) == la.EINVAL   # the tail holds 128 tokens
    assert call(v, pos0=100, n=60, sealed=0, seal_to=0) == la.EINVAL   # would leave more than 128 open
    assert call(v, pos0=2 ** 31 - 40, n=30, sealed=2 ** 31 - 64, seal_to=2 ** 31 - 64) == la.EINVAL
    assert b"2^31" in lib.lfm3a_last_error()


def test_attention_refusals(la):
    lib = la.lib()

    def call(v=None, q=64, stride=0, m=1, qh=32, ctx=100, sealed=96, window=0, out=64, ws=None, ws_bytes=0, splits=1):
        return lib.lfm3a_kv8_attention(ctypes.byref(v or view(la)), q, stride, m, qh, ctx, sealed, window, None, out,
                                       None, ws, ws_bytes, splits, None)

    assert call(q=None) == la.EINVAL
    assert call(out=None) == la.EINVAL
    assert call(m=0) == la.EINVAL
    assert call(m=33) == la.ENOTSUP
    assert call(v=view(la, h=1), m=32, qh=9) == la.ENOTSUP   # 288 rows
    assert call(qh=33) == la.EINVAL
    assert call(stride=2052) == la.EINVAL
    assert call(stride=1024) == la.EINVAL
    assert call(q=72) == la.EINVAL
    assert call(sealed=90) == la.EINVAL
    assert call(ctx=300, sealed=96) == la.EINVAL             # 205 tokens past the sealed ones
    assert call(window=-1) == la.EINVAL
    assert call(ctx=1000, sealed=992, splits=4) == la.EINVAL   # no workspace
    assert call(ctx=1000, sealed=992, splits=4, ws=64, ws_bytes=100) == la.EWORKSPACE


def test_prefill_weights_eviction_refusals(la):
    lib = la.lib()
    v = view(la)
    r = ctypes.byref(v)
    assert lib.lfm3a_kv8_prefill(r, 64, 0, 100, 32, 0, 96, 0, 64, None, 0, None) == la.EINVAL
    assert lib.lfm3a_kv8_prefill(r, 64, 0, 100, 32, 0, 96, 0, 64, 64, 1000, None) == la.EWORKSPACE
    assert lib.lfm3a_kv8_prefill(r, 64, 0, 100, 30, 0, 96, 0, 64, 64, 1000, None) == la.EINVAL
    assert lib.lfm3a_kv8_prefill(r, 64, 0, 0, 32, 0, 0, 0, 64, None, 0, None) == la.OK      # nothing to do
    assert lib.lfm3a_kv8_read(r, 0, 10, 16, 64, 64, None) == la.EINVAL
    assert lib.lfm3a_kv8_read(r, 0, 0, 0, None, None, None) == la.OK

    def weights(q=64, m=1, lse=64, prev=None, prev_stride=0, out=64, out_stride=200):
        return lib.lfm3a_kv8_weights(r, q, 0, m, 32, 100, 96, 0, lse, prev, prev_stride, 1.0, out, out_stride, None)

    assert weights(lse=None) == la.EINVAL
    assert weights(out_stride=100) == la.EINVAL
    assert weights(prev=64, prev_stride=100) == la.EINVAL
    assert weights(m=33) == la.ENOTSUP

    def select(w=64, stride=100, heads=2, n=100, sink=1, recent=2, budget=10, keep=64):
        return lib.lfm3a_evict_select(w, stride, heads, n, sink, recent, budget, keep, None, 0, None)

    assert select(w=None) == la.EINVAL
    assert select(stride=99) == la.EINVAL
    assert select(budget=101) == la.EINVAL
    assert select(budget=0) == la.EINVAL
    assert select(sink=8, recent=3) == la.EINVAL
    assert select(sink=-1) == la.EINVAL
    assert lib.lfm3a_evict_select(64, 100, 2, 100, 1, 2, 10, 64, 64, 9, None) == la.EINVAL
    other = view(la, d=128, h=4)
    assert lib.lfm3a_kv8_compact(r, 100, 96, 64, 10, ctypes.byref(other), None) == la.EINVAL
    assert lib.lfm3a_kv8_compact(r, 100, 96, 64, 10, r, None) == la.EINVAL   # into itself
    ok = view(la, tail=1024)
    assert lib.lfm3a_kv8_compact(r, 100, 96, 64, 101, ctypes.byref(ok), None) == la.EINVAL
    assert lib.lfm3a_kv8_compact(r, 100, 90, 64, 10, ctypes.byref(ok), None) == la.EINVAL


def test_split_counts(la):
    lib = la.lib()
    for d, h, qh in ((64, 8, 32), (128, 4, 16)):
        lay = la.layout(2, h, d)
        for m in (1, 2, 4, 8, 16, 32):
            last = 0
            for ctx in (0, 31, 300, 5000, 131072, 1 << 30):
                s = lib.lfm3a_kv8_splits(ctypes.byref(lay), qh, ctx, m, 0, 148)
                assert 1 <= s <= 1024 and s >= last
                last = s
    assert lib.lfm3a_kv8_splits(None, 32, 0, 1, 0, 148) == la.EINVAL
