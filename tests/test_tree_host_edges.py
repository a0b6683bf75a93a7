"""What the entry points of a step with drafted tokens refuse, or take, at the ends of their
arguments: on the CPU, before any device call."""
import ctypes as C

import pytest

import llmpager_amd as lp
from test_paged_host import INVALID, P, _cache, _said
from test_tree_host import _keep


@pytest.mark.parametrize("caches", [None, (lp.KvCache * 0)(), (lp.KvCache * 1)()])
@pytest.mark.parametrize("lens_out", [0, 2 * P])
def test_keeps_without_layers_look_at_no_cache(caches, lens_out):
    """A null list, an empty one, and one whose first entry no call would take."""
    at = caches if caches is not None else C.POINTER(lp.KvCache)()
    assert lp.lib().lp_kv_keep(None, at, 0, P, 3, P, P, P, lens_out, 2, None) == INVALID
    assert "null context" in _said(), _said()


SPREAD = dict(path=P, kept=2 * P, q_starts=3 * P, seq_lens=4 * P)  # of 2 sequences, 4 entries of a path


@pytest.mark.parametrize("lens_out", [P, P + 28, P - 4, 2 * P, 2 * P + 4, 2 * P - 4, 3 * P, 3 * P + 8, 3 * P - 4, 4 * P, 4 * P + 4, 4 * P - 4])
@pytest.mark.parametrize("layers", [0, 1])
def test_lengths_over_what_is_read_are_refused(lens_out, layers):
    assert _keep(lens_out=lens_out, layers=layers, **SPREAD) == INVALID and "overlap" in _said(), _said()


@pytest.mark.parametrize("lens_out", [0, P + 32, P - 8, 2 * P + 8, 2 * P - 8, 3 * P + 12, 4 * P + 8, 5 * P])
def test_lengths_beside_what_is_read_are_taken(lens_out):
    assert _keep(lens_out=lens_out, **SPREAD) == INVALID and "null context" in _said(), _said()
