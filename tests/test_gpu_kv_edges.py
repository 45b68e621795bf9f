"""Edges of the paged cache's operators on a B200: units of one tile, values that
are not finite, what is reported where."""
import numpy as np
import pytest

from test_gpu_kv import DTYPES, Cache, Trees, sync_ok

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group,nodes", [(4, 3), (7, 4), (7, 9)])
def test_units_of_one_tile(lrs, backend, dtype, group, nodes):
    """Units whose only tile sets every row's maximum, several a CTA and softmax
    groups with and without rows: right, and the same bits each time."""
    import torch
    s = [(13 * i % 115, 1 + i % nodes) for i in range(150)]
    cache = Cache(lrs, dtype, 4, 64, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, group)
    trees.run(backend)
    sync_ok(backend)
    first = trees.out.clone()
    trees.check()
    for _ in range(30):
        trees.out.fill_(-5.0)
        trees.run(backend)
        sync_ok(backend)
        assert torch.equal(first, trees.out)
