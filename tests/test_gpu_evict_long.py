"""Selection where a block's share of the keys no longer fits shared memory (more than 8 x 49152 candidates of a kv head),
just below that, and where a cluster takes over from one block (16384), against the plain rule, exactly."""
import numpy as np
import pytest

from test_gpu_evict import keep_plain, rows_for
from test_gpu_kv8 import dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["skewed", "few", "special"])
@pytest.mark.parametrize("heads,n,budget,sink,recent", [
    (2, 400003, 100001, 3, 64), (1, 393216, 393215, 0, 0), (1, 393217, 1, 0, 0), (2, 16384, 5000, 0, 0),
    (2, 16385, 5000, 0, 0), (1, 16385 + 40, 16385, 30, 10)])
def test_select(la, cuda, kind, heads, n, budget, sink, recent):
    w = rows_for(kind, heads, n, n + budget)
    keep, kept = la.evict_select(dev(w, cuda), n, budget, sink, recent)
    la.sync()
    keep, kept = keep.cpu().numpy(), kept.cpu().numpy()
    for h in range(heads):
        want = keep_plain(w[h], budget, sink, recent)
        assert np.array_equal(keep[h], want), h
        assert np.array_equal(kept[h], w[h][want], equal_nan=True)
