"""lp_verify_tree on the GPU at the ends of what its description allows, against its definition
in 64 bits (tests/_tree.py); paths and tokens are whole numbers and have to be equal."""
import numpy as np
import pytest

import llmpager_amd as lp
from _tree import verify
from test_gpu_tree import Mem
from test_gpu_verify import Case, _path_alone, _same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(cuda):
    return lp.Kernels(cuda)


# ---- calls without tokens -----------------------------------------------------------


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("batch,max_depth", [(1, 0), (3, 5), (70, 70), (1300, 2)])
@pytest.mark.parametrize("tokens,max_q,starts", [(0, 5, 0), (0, 5, 2), (9, 0, 0), (9, 0, 1), (0, 0, 0)])
def test_without_tokens(cuda, K, sampled, batch, max_depth, tokens, max_q, starts):
    """No sequence has a token, whatever the starts say (they rise by `starts`): nothing kept
    and no next token, over what a step before has left there, without a workspace."""
    m = Mem(cuda)
    x = m.up(np.zeros(9 * 50, np.float32))
    i = m.up(np.zeros(9, np.int32))
    ds = m.up(np.arange(batch + 1, dtype=np.int32) * starts)
    shapes = ((batch, max_depth + 1), (batch,), (batch,))
    out = [m.up(np.full(s, 7, np.int32)) for s in shapes]
    assert K.verify_tree_ws_bytes(50, batch, tokens, max_q, max_depth, sampled) == 0
    for stream in (None, cuda.stream()):
        if stream is not None:
            for d, s in zip(out, shapes):
                cuda.htod_async(d, np.full(s, 7, np.int32), stream)
        K.verify_tree(x, 50, 50, i, i, ds, batch, tokens, max_q, max_depth, 0, x if sampled else 0, 50, x, *out, 0, stream, ws_bytes=0)
        path, kept, after = (cuda.download(d, s, np.int32, stream) for d, s in zip(out, shapes))
        assert (path == -1).all() and (kept == 0).all() and (after == -1).all()
        if stream is not None:
            cuda.destroy_stream(stream)
    m.free()
