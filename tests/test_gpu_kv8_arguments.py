"""What LayerCache8 refuses before any launch: tensors whose type, shape, strides or device the kernels would misread."""
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


def test_append_arguments(la, cuda, cache):
    import torch

    x = torch.randn(8, 2, 64, device=cuda).half()
    for k, v in ((x.float(), x), (x, x.float()), (x, x[:4]), (x[:, :1], x[:, :1]), (x.cpu(), x.cpu()),
                 (x.transpose(1, 2).contiguous().transpose(1, 2), x), (x.flatten(1)[:, :100], x.flatten(1)[:, :100]),
                 (torch.cat([x, x], 1)[:, :2], x)):
        refused(la, lambda: cache.append(k, v))
    assert (cache.length, cache.sealed) == (100, 96)
    refused(la, lambda: cache.append(x, x, pos0=101))
    refused(la, lambda: cache.append(x.repeat(20, 1, 1), x.repeat(20, 1, 1)))   # past the capacity


def test_append_takes_the_strides_of_its_tensors(la, cuda, cache):
    import torch

    wide = torch.randn(40, 6, 64, device=cuda).half()
    cache.append(wide[:, 1:3], wide[:, 3:5])
    k, v = cache.read(100, 40)
    other = la.LayerCache8(la.MODE_I8BLK, 2, 64, 256, device=cuda)
    x = torch.cat([torch.zeros(100, 2, 64, device=cuda).half(), wide[:, 1:3]])
    y = torch.cat([torch.zeros(100, 2, 64, device=cuda).half(), wide[:, 3:5]])
    other.append(x, y)
    k2, v2 = other.read(128, 12)   # one whole page past the first cache's older tokens: the tail's values
    la.sync()
    assert torch.equal(k[28:], k2) and torch.equal(v[28:], v2)
    assert torch.equal(k[28:], wide[28:, 1:3]) and torch.equal(v[28:], wide[28:, 3:5])


def test_attention_arguments(la, cuda, cache):
    import torch

    q = torch.randn(4, 8, 64, device=cuda).half()
    lse = torch.empty(4, 8, device=cuda)
    for bad in (q.float(), q.cpu(), q[:, :, :32], q.transpose(0, 1)):
        refused(la, lambda: cache.verify(bad, 92))
        refused(la, lambda: cache.prefill(bad, 92))
        refused(la, lambda: cache.key_weights(bad, lse, 92))
    refused(la, lambda: cache.verify(q, 97))   # tokens that are not appended
    for other in (q.float(), q[:2], q.transpose(0, 1).contiguous().transpose(0, 1), q.cpu()):
        refused(la, lambda: cache.verify(q, 96, gate=other[..., 0]))
        refused(la, lambda: cache.verify(q, 96, out=other))
        refused(la, lambda: cache.prefill(q, 96, out=other))
    for bad in (lse.half(), lse[:3], lse.t().contiguous().t(), lse.cpu()):
        refused(la, lambda: cache.verify(q, 96, lse=bad))
        refused(la, lambda: cache.key_weights(q, bad, 96))
    w = torch.zeros(2, 120, device=cuda)
    for bad in (w[:, :99], w[:1], w.half(), w.cpu(), w.t().contiguous().t()):
        refused(la, lambda: cache.key_weights(q, lse, 96, prev=bad))
        refused(la, lambda: cache.key_weights(q, lse, 96, out=bad))


def test_eviction_arguments(la, cuda, cache):
    import torch

    dst = la.LayerCache8(la.MODE_I8BLK, 2, 64, 64, device=cuda)
    w = torch.rand(2, 100, device=cuda)
    for bad in (w[:1], w[:, :99], w.half(), w.cpu(), w.t().contiguous().t()):
        refused(la, lambda: cache.evict(bad, 40, 1, 2, dst))
    refused(la, lambda: cache.evict(w, 65, 1, 2, dst))    # more than dst holds
    refused(la, lambda: cache.evict(w, 40, 30, 20, dst))
    refused(la, lambda: cache.evict(w, 40, 1, 2, cache))
    refused(la, lambda: cache.evict(w, 40, 1, 2, la.LayerCache8(la.MODE_E4M3BLK, 2, 64, 64, device=cuda)))
    refused(la, lambda: cache.evict(w, 40, 1, 2, la.LayerCache8(la.MODE_I8BLK, 2, 128, 64, device=cuda)))
    assert dst.length == 0
    for table in (torch.arange(1, device=cuda).int(), torch.arange(8, device=cuda)):
        refused(la, lambda: la.LayerCache8(la.MODE_I8BLK, 2, 64, 64, device=cuda, block_table=table))
