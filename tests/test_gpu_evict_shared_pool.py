"""Eviction into another cache of the same pool: blocks that are still being read are refused, others give what a pool of
its own gives."""
import pytest

pytestmark = pytest.mark.gpu

N, BUDGET = 300, 100


def source(la, cuda, pool_blocks, seed=3):
    import torch

    gen = torch.Generator(device=cuda).manual_seed(seed)
    cache = la.LayerCache8(la.MODE_I8BLK, 2, 64, 320, device=cuda, pool_blocks=pool_blocks)
    k, v = (torch.randn(N, 2, 64, generator=gen, device=cuda).half() for _ in range(2))
    cache.append(k, v)   # 288 tokens in the blocks 0 .. 8, 12 in the tail
    return cache, torch.rand(2, N, generator=gen, device=cuda)


def smaller(la, cuda, cache, blocks):
    import torch

    table = None if blocks is None else torch.tensor(blocks, dtype=torch.int32, device=cuda)
    return la.LayerCache8(la.MODE_I8BLK, 2, 64, 128, device=cuda, pool=cache, block_table=table)


@pytest.mark.parametrize("blocks", [None, [12, 8, 13, 14], [12, -1, 13, 14], [0, 12, 13, 14]])
def test_blocks_in_use_are_refused(la, cuda, blocks):
    import torch

    cache, w = source(la, cuda, 16)
    dst = smaller(la, cuda, cache, blocks)   # None: the default table, the source's own first blocks; -1 is taken as 0
    before = cache.pool.clone()
    with pytest.raises(la.LFM3AError) as e:
        cache.evict(w, BUDGET, 4, 32, dst)
    assert e.value.code == la.EINVAL
    la.sync()
    assert dst.length == 0 and torch.equal(cache.pool, before)


@pytest.mark.parametrize("blocks", [[12, 10, 15, 14], [9, 11, 99, 0]])   # 99 is taken as 15; the last is not written
def test_other_blocks_of_the_pool(la, cuda, blocks):
    import torch

    cache, w = source(la, cuda, 16)
    alone = la.LayerCache8(la.MODE_I8BLK, 2, 64, 128, device=cuda)
    dst = smaller(la, cuda, cache, blocks)
    whole = cache.read(0, N)
    a, b = cache.evict(w, BUDGET, 4, 32, dst), cache.evict(w, BUDGET, 4, 32, alone)
    la.sync()
    for x, y in zip((*a, *dst.read(0, BUDGET), *cache.read(0, N)), (*b, *alone.read(0, BUDGET), *whole)):
        assert torch.equal(x, y)
