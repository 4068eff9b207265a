"""LayerCache8 on a machine without a GPU: a pool, block table or tail on the host is refused (the kernels would be given
host addresses)."""
import pytest


def test_host_memory(la):
    import torch

    for kw in ({}, {"block_table": torch.arange(8, dtype=torch.int32)}):
        with pytest.raises(la.LFM3AError) as e:
            la.LayerCache8(la.MODE_I8BLK, 2, 64, 256, device="cpu", **kw)
        assert e.value.code == la.EINVAL
