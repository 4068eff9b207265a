"""More of what LayerCache8 refuses before any launch, because a kernel would read or write outside the tensors given."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture()
def cache(la, cuda):
    import torch

    c = la.LayerCache8(la.MODE_I8BLK, 2, 64, 256, device=cuda)
    x = torch.randn(100, 2, 64, device=cuda).half()
    c.append(x, x)
    return c


def refused(la, f):
    with pytest.raises(la.LFM3AError) as e:
        f()
    assert e.value.code == la.EINVAL


def test_append_token_strides(la, cuda, cache):
    """A stride of 0 (expand), one below a row, one that the tensors do not have."""
    import torch

    one = torch.randn(1, 2, 64, device=cuda).half()
    x = torch.randn(8, 2, 64, device=cuda).half()
    flat = torch.randn(2000, device=cuda).half()
    wide = torch.randn(8, 6, 64, device=cuda).half()
    overlap = flat.as_strided((8, 2, 64), (64, 64, 1))
    for k, v in ((one.expand(8, 2, 64), one.expand(8, 2, 64)), (x, one.expand(8, 2, 64)), (one.expand(8, 2, 64), x),
                 (overlap, overlap), (wide[:, :2], x)):
        refused(la, lambda: cache.append(k, v))
    for stride in (64, 4096, -128):
        refused(la, lambda: cache.append(x, x, token_stride=stride))
    refused(la, lambda: cache.append(wide[:, :2], wide[:, 2:4], token_stride=128))
    assert (cache.length, cache.sealed) == (100, 96)
    cache.append(wide[:, :2], wide[:, 2:4], token_stride=384)
    cache.append(one.expand(1, 2, 64), wide[:1, 2:4])   # a single token has no stride
    k, v = cache.read(100, 9)
    la.sync()
    assert torch.equal(k, torch.cat([wide[:, :2], one])) and torch.equal(v, torch.cat([wide[:, 2:4], wide[:1, 2:4]]))


def test_query_token_strides(la, cuda, cache):
    import torch

    one = torch.randn(1, 8, 64, device=cuda).half()
    flat = torch.randn(4000, device=cuda).half()
    lse = torch.zeros(4, 8, device=cuda)
    for q in (one.expand(4, 8, 64), flat.as_strided((4, 8, 64), (64, 64, 1))):
        refused(la, lambda: cache.verify(q, 96))
        refused(la, lambda: cache.prefill(q, 96))
        refused(la, lambda: cache.key_weights(q, lse, 96))
    a, b = cache.verify(one.expand(1, 8, 64), 99), cache.verify(one.clone(), 99)
    la.sync()
    assert torch.equal(a, b)


def test_append_rope_and_norm(la, cuda, cache):
    """A RoPE table has a row for every position up to the last new one; a norm has head_dim weights."""
    import torch

    x = torch.randn(8, 2, 64, device=cuda).half()
    table = torch.from_numpy(la.rope_table(1e6, 1.0, 64, 216)).view(torch.float16).to(cuda)
    rope = table[:108]
    for bad in (table[:107], table[:0], table[::2], rope.float(), rope.view(torch.int16), rope.cpu(), rope[:, :32],
                rope.flatten(), table.view(108, 128), rope.t().contiguous().t()):
        refused(la, lambda: cache.append(x, x, rope=bad))
        refused(la, lambda: cache.append(x, x, rope=bad, draft=True))
    norm = torch.ones(64, device=cuda).half()
    for bad in (norm[:32], norm.float(), norm.cpu(), torch.ones(128, device=cuda).half()[::2]):
        refused(la, lambda: cache.append(x, x, k_norm=bad))
    assert (cache.length, cache.sealed) == (100, 96)
    cache.append(x, x, rope=rope, k_norm=norm, draft=True)   # the table's last row is the last token's
    k, _ = cache.read(100, 8)
    cache.append(x, x, pos0=100, rope=table, k_norm=norm, draft=True)
    k2, _ = cache.read(100, 8)
    la.sync()
    assert torch.equal(k, k2)


def test_memory_of_another_device(la, cuda, cache, monkeypatch):
    """Tensors on the host, and on a GPU that is not the cache's (here the cache takes itself to be on GPU 1)."""
    import torch

    def make(**kw):
        return la.LayerCache8(la.MODE_I8BLK, 2, 64, 256, **kw)

    refused(la, lambda: make(device=cuda, block_table=torch.arange(8, dtype=torch.int32)))
    refused(la, lambda: make(device="cpu"))
    refused(la, lambda: make(device="cpu", pool=cache, block_table=torch.arange(8, dtype=torch.int32, device=cuda)))
    q = torch.randn(4, 8, 64, device=cuda).half()
    ws = torch.empty(1 << 22, dtype=torch.uint8, device=cuda)
    for bad in (ws.cpu(), ws.view(2048, 2048).t()):
        refused(la, lambda: cache.verify(q, 96, workspace=bad))
        refused(la, lambda: cache.prefill(q, 96, workspace=bad))

    x = torch.randn(8, 2, 64, device=cuda).half()
    rope = torch.zeros(108, 64, device=cuda).half()
    lse, w = torch.zeros(4, 8, device=cuda), torch.zeros(2, 100, device=cuda)
    dst, other = make(device=cuda), make(device=cuda)
    calls = [lambda c: c.append(x, x), lambda c: c.append(x, x, rope=rope), lambda c: c.append(x, x, k_norm=rope[0]),
             lambda c: c.read(0, 4), lambda c: c.verify(q, 96), lambda c: c.verify(q, 96, workspace=ws),
             lambda c: c.prefill(q, 96), lambda c: c.key_weights(q, lse, 96), lambda c: c.evict(w, 40, 1, 2, dst)]
    monkeypatch.setattr(other, "_gpu", 1)
    other.length, other.sealed = cache.length, cache.sealed
    side = torch.cuda.Stream()
    for call in calls:
        refused(la, lambda: call(other))
    refused(la, lambda: cache.evict(w, 40, 1, 2, other))
    refused(la, lambda: other.read(0, 4, stream=side))
    refused(la, lambda: other.read(0, 4, stream=side.cuda_stream))
    assert (other.length, dst.length) == (100, 0)
    for call in calls:   # the same calls are right on the cache's own GPU
        call(cache)
        cache.truncate(100)
    la.sync()


def test_current_device(la, cuda, cache, monkeypatch):
    """A call while another GPU is the current one would launch there."""
    import torch

    w = torch.zeros(2, 100, device=cuda)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    refused(la, lambda: cache.read(0, 4))
    refused(la, lambda: cache.read(0, 4, stream=0))
    refused(la, lambda: la.evict_select(w, 100, 40, 1, 2))
