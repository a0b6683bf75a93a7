"""What the paged cache and log probability entry points refuse, and the sizes
they state: on the CPU, before any device call (a null context is refused last,
so a call that is right otherwise says just that)."""
import ctypes as C
import os
import re

import pytest

import llmpager_amd as lp
from test_abi import HEADER, ROOT, _c_struct_fields

INVALID, UNSUPPORTED = -1, -2
P = 1 << 32  # an aligned address that nothing reads


def _cache(**kw):
    d = dict(k_pages=P, v_pages=P, table=P, pages=8, page_rows=16, max_pages=4, kv_heads=2, head_dim=128, format=lp.KV_Q4)
    d.update(kw)
    return lp.KvCache(**d)


def _append(cache=None, **kw):
    d = dict(q=P, q_stride=512, k=P, k_stride=256, v=P, v_stride=256, q_norm=0, k_norm=0, eps=1e-6, inv_freq=P, mscale=1.0,
             q_out=P, q_out_stride=512, k_out=0, v_out=0, heads=4, q_starts=P, seq_lens=P, batch=2, tokens=3)
    d.update(kw)
    return lp.lib().lp_kv_append_paged(None, cache if cache is not None else _cache(), *d.values(), None)


def _attn(cache=None, **kw):
    d = dict(q=P, q_stride=512, out=2 * P, out_stride=512, heads=4, q_starts=P, seq_lens=P, batch=2, tokens=3, max_q=2,
             max_seq=60, scale=0.1, workspace=P, ws_bytes=1 << 40)
    d.update(kw)
    return lp.lib().lp_attn_paged(None, cache if cache is not None else _cache(), *d.values(), None)


def _logprobs(**kw):
    d = dict(logits=P, stride=100, rows=2, vocab=100, targets=P, logp=P, entropy=P, top=5, ids=P, top_logp=P, workspace=P,
             ws_bytes=1 << 40)
    d.update(kw)
    return lp.lib().lp_logprobs(None, *d.values(), None)


def _said():
    return lp.lib().lp_last_error().decode()


def test_right_calls_need_a_context_only():
    for call in (_append, _attn, _logprobs):
        assert call() == INVALID and "null context" in _said()
    assert _append(q_norm=P, k_norm=P, k_out=P, v_out=P) == INVALID and "null context" in _said()
    assert _append(q_stride=1024, k=P + 2048, k_stride=1024, v=P + 3 * 1024, v_stride=1024) == INVALID and "null context" in _said()
    assert _logprobs(targets=0, logp=0, entropy=0, top=0, ids=0, top_logp=0) == INVALID and "null context" in _said()


CACHES = [
    (dict(format=2), INVALID), (dict(format=-1), INVALID), (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=256), UNSUPPORTED),
    (dict(page_rows=8), UNSUPPORTED), (dict(page_rows=48), UNSUPPORTED), (dict(page_rows=512), UNSUPPORTED),
    (dict(pages=0), INVALID), (dict(max_pages=0), INVALID), (dict(kv_heads=0), INVALID), (dict(kv_heads=-2), INVALID),
    (dict(max_pages=(1 << 26) + 1), UNSUPPORTED), (dict(k_pages=0), INVALID), (dict(v_pages=0), INVALID),
    (dict(table=0), INVALID), (dict(k_pages=P + 8), INVALID), (dict(v_pages=P + 2), INVALID), (dict(table=P + 2), INVALID),
]


@pytest.mark.parametrize("kw,code", CACHES)
def test_caches_refused(kw, code):
    for call, who in ((_append, "kv_append_paged"), (_attn, "attn_paged")):
        assert call(_cache(**kw)) == code and _said().startswith(who), _said()
    assert lp.lib().lp_attn_paged_ws_bytes(_cache(**kw), 4, 2, 3, 2, 60) == 0


def test_null_cache_refused():
    null = C.POINTER(lp.KvCache)()
    assert _append(null) == INVALID and "null cache" in _said()
    assert _attn(null) == INVALID and "null cache" in _said()
    assert lp.lib().lp_attn_paged_ws_bytes(null, 4, 2, 3, 2, 60) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(heads=0), INVALID), (dict(heads=3), INVALID), (dict(heads=-4), INVALID), (dict(batch=-1), INVALID),
    (dict(tokens=-1), INVALID), (dict(batch=4097), UNSUPPORTED), (dict(q_starts=0), INVALID), (dict(seq_lens=0), INVALID),
    (dict(q_starts=P + 1), INVALID), (dict(q=0), INVALID), (dict(q=P + 4), UNSUPPORTED), (dict(q_stride=508), INVALID),
    (dict(q_stride=514), UNSUPPORTED), (dict(q_stride=-512), INVALID)])
def test_batches_and_queries_refused(kw, code):
    for call in (_append, _attn):
        assert call(**kw) == code and "null context" not in _said(), _said()


@pytest.mark.parametrize("kw,code", [
    (dict(k=0), INVALID), (dict(v=0), INVALID), (dict(k=P + 8), UNSUPPORTED), (dict(v_stride=252), INVALID),
    (dict(q_out=0), INVALID), (dict(q_out_stride=4), INVALID), (dict(inv_freq=0), INVALID), (dict(inv_freq=P + 4), INVALID),
    (dict(q_norm=P + 4), INVALID), (dict(k_norm=P + 2), INVALID), (dict(k_out=P + 4), INVALID), (dict(v_out=P + 8), INVALID)])
def test_appends_refused(kw, code):
    assert _append(**kw) == code and "null context" not in _said(), _said()


@pytest.mark.parametrize("kw,code", [
    (dict(out=0), INVALID), (dict(out=P), INVALID), (dict(out=P + 4), UNSUPPORTED), (dict(out_stride=500), INVALID),
    (dict(max_q=-1), INVALID), (dict(max_seq=-1), INVALID)])
def test_attention_refused(kw, code):
    assert _attn(**kw) == code and "null context" not in _said(), _said()


@pytest.mark.parametrize("kw,code", [
    (dict(logits=0), INVALID), (dict(logits=P + 2), INVALID), (dict(rows=-1), INVALID), (dict(vocab=0), INVALID),
    (dict(stride=99), INVALID), (dict(top=-1), INVALID), (dict(top=101), INVALID), (dict(top=65), UNSUPPORTED),
    (dict(targets=0), INVALID), (dict(logp=0), INVALID), (dict(ids=0), INVALID), (dict(top_logp=0), INVALID),
    (dict(entropy=P + 1), INVALID), (dict(ids=P + 2), INVALID), (dict(logp=P + 3), INVALID)])
def test_logprobs_refused(kw, code):
    assert _logprobs(**kw) == code and "null context" not in _said(), _said()


def test_workspaces_checked():
    """Where a call needs a workspace, one that is null, misaligned or a byte
    short is refused; one that is as large as stated is taken."""
    c = _cache(max_pages=4096)
    need = lp.lib().lp_attn_paged_ws_bytes(c, 4, 2, 3, 2, 60000)
    if need:
        kw = dict(max_seq=60000)
        assert _attn(c, ws_bytes=need, **kw) == INVALID and "null context" in _said()
        assert _attn(c, ws_bytes=need - 1, **kw) == INVALID and "workspace" in _said()
        assert _attn(c, workspace=0, **kw) == INVALID and "workspace" in _said()
        assert _attn(c, workspace=P + 64, **kw) == UNSUPPORTED and "workspace" in _said()
    need = lp.lib().lp_logprobs_ws_bytes(2, 151936, 5)
    if need:
        kw = dict(vocab=151936, stride=151936)
        assert _logprobs(ws_bytes=need, **kw) == INVALID and "null context" in _said()
        assert _logprobs(ws_bytes=need - 1, **kw) == INVALID and "workspace" in _said()
        assert _logprobs(workspace=0, **kw) == INVALID and "workspace" in _said()
        assert _logprobs(workspace=P + 64, **kw) == UNSUPPORTED and "workspace" in _said()


@pytest.mark.parametrize("rows", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", [64, 128])
def test_page_bytes(rows, dim):
    """An fp16 page's rows, and a q4 region of them (group 32)."""
    assert lp.kv_page_bytes(rows, dim, lp.KV_F16) == rows * dim * 2
    assert lp.kv_page_bytes(rows, dim, lp.KV_Q4) == lp.q4_bytes(rows, dim, 32)
    assert lp.kv_page_bytes(rows, dim, lp.KV_Q4) % 16 == 0
    assert lp.kv_page_bytes(rows + 1, dim, lp.KV_Q4) == lp.kv_page_bytes(rows, dim, 2) == lp.kv_page_bytes(rows, 80, 0) == 0


def test_kv_cache_struct_follows_the_header():
    hdr = open(HEADER).read()
    fields = _c_struct_fields(hdr, "lp_kv_cache")
    assert fields == [f for f, _ in lp.KvCache._fields_] and C.sizeof(lp.KvCache) == 48
    rs = open(os.path.join(ROOT, "rust", "llmpager-hip", "src", "ffi.rs")).read()
    body = re.search(r"pub struct lp_kv_cache \{(.*?)\n\}", rs, flags=re.S).group(1)
    assert re.findall(r"pub ([a-z0-9_]+):", body) == fields
