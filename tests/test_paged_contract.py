"""What lp_kv_cache, lp_kv_append_paged, lp_attn_paged and lp_logprobs state in
include/llmpager_hip.h, on the CPU."""
import numpy as np
import pytest

import llmpager_amd as lp
from _paged import q4
from test_paged_host import INVALID, P, UNSUPPORTED, _attn, _cache, _logprobs, _said


def test_scales_that_a_q4_page_may_hold():
    """Every scale of 7 significant bits within 2^-17 .. 896: 72 of it and its
    multiples -8 .. 7 are fp16 numbers, so n s - 72 s is exact; some scale of 11 bits is
    off by s / 29 and none by more than s / 28, and from 910 on 72 of it is no number."""
    s = np.array([m * 2.0 ** e for e in range(-23, 10) for m in range(64, 128) if 2.0 ** -17 <= m * 2.0 ** e <= 896.0])
    for n in [72.0] + list(range(-8, 8)):
        assert np.array_equal((n * s).astype(np.float16).astype(np.float64), n * s)
    h = np.arange(1, 1 << 15, dtype=np.uint16).view(np.float16).astype(np.float64)
    h = h[(h >= 2.0 ** -10) & (h < 909.0)]
    off = np.abs((72.0 * h).astype(np.float16).astype(np.float64) - 72.0 * h) / h
    assert 1 / 29 < off.max() < 1 / 28
    with np.errstate(over="ignore"):
        assert np.isinf(np.float16(72.0 * 910.0)) and np.isfinite(np.float16(72.0 * 896.0))


def test_scales_as_the_append_makes_them():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((4000, 64)) * 10.0 ** rng.uniform(-8, 6, (4000, 1))
    x[0], x[1, 3] = 0.0, np.inf
    _, s = q4(x)
    m, _ = np.frexp(s)
    assert s.min() == 2.0 ** -17 and s.max() == 896.0 and np.array_equal(m * 128, np.rint(m * 128))
    assert np.array_equal(s.astype(np.float16).astype(np.float64), s)


@pytest.mark.parametrize("kv,heads,batch,tokens,max_q,taken", [
    (2, 64, 64, 4096, 2048, True),           # 64 sequences, of which one has 2,048 tokens
    (8, 64, 4096, 8192, 4096, False),        # 8,388,608 blocks of 128 query rows
    (8, 64, 4095, 8192, 4096, True),
    (2, 8, 4096, 1 << 30, 1 << 30, False),
    (1, 1 << 20, 4, 1 << 20, 1 << 11, False),  # 2^31 query rows
    (1, 4, 4096, 4096, 1, True),
])
def test_bounds_of_the_query_rows(kv, heads, batch, tokens, max_q, taken):
    c = _cache(kv_heads=kv)
    kw = dict(heads=heads, batch=batch, tokens=tokens, max_q=max_q, q_stride=heads * 128, out_stride=heads * 128)
    if taken:
        assert _attn(c, **kw) == INVALID and "null context" in _said(), _said()
    else:
        assert _attn(c, **kw) == UNSUPPORTED and "query rows" in _said(), _said()
        assert lp.lib().lp_attn_paged_ws_bytes(c, heads, batch, tokens, max_q, 60) == 0


@pytest.mark.parametrize("kw", [dict(tokens=0), dict(max_q=0), dict(batch=0), dict(tokens=0, batch=0)])
def test_a_call_without_queries_needs_no_workspace(kw):
    c = _cache(max_pages=4096)
    n = dict(batch=2, tokens=3, max_q=2)
    n.update(kw)
    assert lp.lib().lp_attn_paged_ws_bytes(c, 4, n["batch"], n["tokens"], n["max_q"], 60000) == 0
    assert _attn(c, workspace=0, ws_bytes=0, max_seq=60000, **kw) == INVALID and "null context" in _said(), _said()


@pytest.mark.parametrize("kw,attn", [
    (dict(), True), (dict(tokens=900, max_q=900, q_stride=1024), True), (dict(tokens=20000, max_q=20000, batch=50), False)])
def test_workspaces_of_calls_that_need_one(kw, attn):
    """What test_workspaces_checked looks at where a workspace is needed, and calls
    that are known to need one."""
    c = _cache(max_pages=4096)
    n = dict(batch=2, tokens=3, max_q=2, max_seq=60000)
    n.update(kw)
    need = lp.lib().lp_attn_paged_ws_bytes(c, 4, n["batch"], n["tokens"], n["max_q"], 60000)
    assert (need > 0) == attn
    kw = dict(n, ws_bytes=need)
    assert _attn(c, **kw) == INVALID and "null context" in _said()
    if attn:
        assert _attn(c, **dict(kw, ws_bytes=need - 1)) == INVALID and "workspace" in _said()
        assert _attn(c, **dict(kw, workspace=0)) == INVALID and "null workspace" in _said()
        assert _attn(c, **dict(kw, workspace=P + 64)) == UNSUPPORTED and "workspace" in _said()


def test_log_probabilities_that_need_a_workspace():
    need = lp.lib().lp_logprobs_ws_bytes(2, 151936, 5)
    assert need > 0 and lp.lib().lp_logprobs_ws_bytes(3000, 151936, 5) == 0
    kw = dict(vocab=151936, stride=151936)
    assert _logprobs(ws_bytes=need, **kw) == INVALID and "null context" in _said()
    assert _logprobs(ws_bytes=need - 1, **kw) == INVALID and "workspace" in _said()
    assert _logprobs(workspace=0, **kw) == INVALID and "null workspace" in _said()
    assert _logprobs(workspace=P + 64, **kw) == UNSUPPORTED and "workspace" in _said()
