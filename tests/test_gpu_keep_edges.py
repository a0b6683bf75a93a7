"""lp_kv_keep on the GPU without layers: the lengths alone."""
import numpy as np
import pytest

import llmpager_amd as lp
from test_gpu_tree import Mem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [1, 5, 1000])
@pytest.mark.parametrize("max_depth", [0, 5, 100])
def test_lengths_without_layers(cuda, batch, max_depth):
    m, K = Mem(cuda), lp.Kernels(cuda)
    rng = np.random.default_rng(batch)
    new = rng.integers(0, 130, batch)
    past = rng.integers(0, 9000, batch)
    kept = rng.integers(-1, max_depth + 3, batch)
    path = np.tile(np.arange(max_depth + 1, dtype=np.int32) * 2, (batch, 1))
    starts = np.concatenate(([3], 3 + np.cumsum(new))).astype(np.int32)
    do = m.up(np.full(batch, 7, np.int32))
    args = [m.up(path), max_depth, m.up(kept.astype(np.int32)), m.up(starts), m.up((past + new).astype(np.int32))]
    K.kv_keep([], *args, 0, batch)  # nothing to do
    assert (cuda.download(do, (batch,), np.int32) == 7).all()
    K.kv_keep([], *args, do, batch)
    want = past + np.clip(kept, 0, np.minimum(new, max_depth + 1))
    assert np.array_equal(cuda.download(do, (batch,), np.int32), want)
    m.free()
