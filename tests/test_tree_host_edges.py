"""What the entry points of a step with drafted tokens refuse, or take, at the ends of their
arguments: on the CPU, before any device call."""
import ctypes as C

import pytest

import llmpager_amd as lp
from test_paged_host import INVALID, P, _cache, _said


@pytest.mark.parametrize("caches", [None, (lp.KvCache * 0)(), (lp.KvCache * 1)()])
@pytest.mark.parametrize("lens_out", [0, 2 * P])
def test_keeps_without_layers_look_at_no_cache(caches, lens_out):
    """A null list, an empty one, and one whose first entry no call would take."""
    at = caches if caches is not None else C.POINTER(lp.KvCache)()
    assert lp.lib().lp_kv_keep(None, at, 0, P, 3, P, P, P, lens_out, 2, None) == INVALID
    assert "null context" in _said(), _said()
