"""What the entry points of a step with drafted tokens refuse, and the sizes they
state: on the CPU, before any device call (a null context is refused last, so a
call that is right otherwise says just that).  And the formulas themselves: that a
verified token has the target's distribution."""
import ctypes as C

import numpy as np
import pytest

import llmpager_amd as lp
from _tree import ancestors, random_tree, verify_one
from test_paged_host import CACHES, INVALID, P, UNSUPPORTED, _cache, _said


def _layout(**kw):
    d = dict(parents=P, q_starts=P, batch=2, tokens=9, max_q=6, depths=P, masks=P)
    d.update(kw)
    return lp.lib().lp_tree_layout(None, *d.values(), None)


def _append(cache=None, **kw):
    d = dict(q=P, q_stride=512, k=P, k_stride=256, v=P, v_stride=256, q_norm=0, k_norm=0, eps=1e-6, inv_freq=P, mscale=1.0,
             q_out=P, q_out_stride=512, k_out=0, v_out=0, heads=4, q_starts=P, seq_lens=P, depths=P, batch=2, tokens=3)
    d.update(kw)
    return lp.lib().lp_kv_append_tree(None, cache if cache is not None else _cache(), *d.values(), None)


def _attn(cache=None, **kw):
    d = dict(q=P, q_stride=512, out=2 * P, out_stride=512, heads=4, q_starts=P, seq_lens=P, masks=P, batch=2, tokens=3,
             max_q=2, max_seq=60, scale=0.1, workspace=P, ws_bytes=1 << 40)
    d.update(kw)
    return lp.lib().lp_attn_tree(None, cache if cache is not None else _cache(), *d.values(), None)


def _verify(**kw):
    d = dict(logits=P, stride=100, vocab=100, drafts=P, parents=P, q_starts=P, batch=2, tokens=9, max_q=6, max_depth=3,
             temperatures=P, probs=P, probs_stride=100, uniforms=P, path=P, kept=P, next=P, workspace=P, ws_bytes=1 << 40)
    d.update(kw)
    return lp.lib().lp_verify_tree(None, *d.values(), None)


def _keep(caches=None, **kw):
    d = dict(path=P, max_depth=3, kept=P, q_starts=P, seq_lens=P, lens_out=2 * P, batch=2)
    d.update(kw)
    caches = caches if caches is not None else [_cache()]
    n = d.pop("layers", len(caches))
    return lp.lib().lp_kv_keep(None, (lp.KvCache * len(caches))(*caches), n, *d.values(), None)


def test_right_calls_need_a_context_only():
    for call in (_layout, _append, _attn, _verify, _keep):
        assert call() == INVALID and "null context" in _said(), _said()
    for kw in (dict(temperatures=0), dict(probs=0, probs_stride=0), dict(max_depth=0), dict(batch=0), dict(tokens=0)):
        assert _verify(**kw) == INVALID and "null context" in _said(), _said()
    assert _keep(lens_out=0) == INVALID and "null context" in _said()
    assert _keep(layers=0) == INVALID and "null context" in _said()
    assert _layout(max_q=1024) == INVALID and "null context" in _said()


@pytest.mark.parametrize("kw,code", CACHES)
def test_caches_refused(kw, code):
    for call, who in ((lambda: _append(_cache(**kw)), "kv_append_tree"), (lambda: _attn(_cache(**kw)), "attn_tree"),
                      (lambda: _keep([_cache(**kw)]), "kv_keep")):
        assert call() == code and _said().startswith(who), _said()
    assert lp.lib().lp_attn_tree_ws_bytes(_cache(**kw), 4, 2, 3, 2, 60) == 0


def test_null_caches_refused():
    null = C.POINTER(lp.KvCache)()
    assert _append(null) == INVALID and "null cache" in _said()
    assert _attn(null) == INVALID and "null cache" in _said()
    assert lp.lib().lp_kv_keep(None, null, 2, P, 3, P, P, P, 0, 2, None) == INVALID and "null cache" in _said()


@pytest.mark.parametrize("kw,code", [
    (dict(parents=0), INVALID), (dict(depths=0), INVALID), (dict(masks=0), INVALID), (dict(masks=P + 4), INVALID),
    (dict(parents=P + 2), INVALID), (dict(depths=P + 1), INVALID), (dict(batch=-1), INVALID), (dict(tokens=-1), INVALID),
    (dict(batch=4097), UNSUPPORTED), (dict(max_q=-1), INVALID), (dict(max_q=1025), UNSUPPORTED), (dict(q_starts=0), INVALID),
    (dict(q_starts=P + 2), INVALID)])
def test_layouts_refused(kw, code):
    assert _layout(**kw) == code and _said().startswith("tree_layout"), _said()


@pytest.mark.parametrize("kw,code", [
    (dict(heads=0), INVALID), (dict(heads=3), INVALID), (dict(batch=-1), INVALID), (dict(tokens=-1), INVALID),
    (dict(batch=4097), UNSUPPORTED), (dict(q_starts=0), INVALID), (dict(seq_lens=0), INVALID), (dict(q=0), INVALID),
    (dict(q=P + 4), UNSUPPORTED), (dict(q_stride=508), INVALID), (dict(q_stride=514), UNSUPPORTED)])
def test_batches_refused(kw, code):
    for call, who in ((_append, "kv_append_tree"), (_attn, "attn_tree")):
        assert call(**kw) == code and _said().startswith(who), _said()


@pytest.mark.parametrize("kw,code", [
    (dict(depths=0), INVALID), (dict(depths=P + 2), INVALID), (dict(k=0), INVALID), (dict(v_stride=252), INVALID),
    (dict(inv_freq=0), INVALID), (dict(q_out=0), INVALID), (dict(k_out=P + 4), INVALID)])
def test_appends_refused(kw, code):
    assert _append(**kw) == code and _said().startswith("kv_append_tree"), _said()


@pytest.mark.parametrize("kw,code", [
    (dict(masks=0), INVALID), (dict(masks=P + 4), INVALID), (dict(out=0), INVALID), (dict(out=P), INVALID),
    (dict(max_q=-1), INVALID), (dict(max_seq=-1), INVALID), (dict(max_q=1025), UNSUPPORTED), (dict(out_stride=500), INVALID)])
def test_attention_refused(kw, code):
    assert _attn(**kw) == code and _said().startswith("attn_tree"), _said()
    if "max_q" in kw:
        assert lp.lib().lp_attn_tree_ws_bytes(_cache(), 4, 2, 3, kw["max_q"], 60) == 0


@pytest.mark.parametrize("kw,code", [
    ({n: 0}, INVALID) for n in ("logits", "drafts", "parents", "q_starts", "uniforms", "path", "kept", "next")] + [
    ({n: P + 2}, INVALID) for n in ("logits", "drafts", "parents", "q_starts", "temperatures", "probs", "uniforms", "path",
                                    "kept", "next")] + [
    (dict(vocab=0), INVALID), (dict(stride=99), INVALID), (dict(probs_stride=99), INVALID), (dict(max_depth=-1), INVALID),
    (dict(max_depth=1024), UNSUPPORTED), (dict(max_q=-1), INVALID), (dict(max_q=1025), UNSUPPORTED), (dict(batch=-1), INVALID),
    (dict(batch=4097), UNSUPPORTED), (dict(tokens=-1), INVALID), (dict(tokens=1 << 23), UNSUPPORTED),
    (dict(vocab=(1 << 19) + 1, stride=1 << 20, probs_stride=1 << 20), UNSUPPORTED)])
def test_verifications_refused(kw, code):
    assert _verify(**kw) == code and _said().startswith("verify_tree"), _said()


@pytest.mark.parametrize("kw,code", [
    (dict(path=0), INVALID), (dict(kept=0), INVALID), (dict(path=P + 2), INVALID), (dict(kept=P + 1), INVALID),
    (dict(lens_out=P + 2), INVALID), (dict(lens_out=P), INVALID), (dict(q_starts=0), INVALID), (dict(seq_lens=0), INVALID),
    (dict(max_depth=-1), INVALID), (dict(max_depth=1024), UNSUPPORTED), (dict(batch=-1), INVALID), (dict(batch=4097), UNSUPPORTED),
    (dict(layers=-1), INVALID)])
def test_keeps_refused(kw, code):
    assert _keep(**kw) == code and _said().startswith("kv_keep"), _said()


@pytest.mark.parametrize("kw", [dict(table=2 * P), dict(pages=9), dict(page_rows=32), dict(max_pages=5), dict(kv_heads=1),
                                dict(head_dim=64), dict(format=lp.KV_F16)])
def test_layers_that_differ_are_refused(kw):
    assert _keep([_cache(), _cache(k_pages=2 * P, v_pages=3 * P)]) == INVALID and "null context" in _said()
    assert _keep([_cache(), _cache(**kw)]) == INVALID and "share" in _said()


@pytest.mark.parametrize("probs", [0, 1])
@pytest.mark.parametrize("vocab,batch,tokens,max_q,max_depth", [
    (100, 2, 9, 6, 3), (151936, 32, 1900, 60, 8), (151936, 1, 26, 26, 5), (1, 1, 1, 1, 0), (1 << 19, 4096, 5000, 1024, 1023)])
def test_workspaces_checked(probs, vocab, batch, tokens, max_q, max_depth):
    """A workspace that is null, misaligned or a byte short is refused, one that is
    as large as stated is taken; a call without tokens needs none."""
    need = lp.lib().lp_verify_tree_ws_bytes(vocab, batch, tokens, max_q, max_depth, probs)
    assert need > 0
    kw = dict(vocab=vocab, stride=vocab, probs=probs * P, probs_stride=vocab, batch=batch, tokens=tokens, max_q=max_q,
              max_depth=max_depth, ws_bytes=need)
    assert _verify(**kw) == INVALID and "null context" in _said()
    assert _verify(**dict(kw, ws_bytes=need - 1)) == INVALID and "workspace" in _said()
    assert _verify(**dict(kw, workspace=0)) == INVALID and "null workspace" in _said()
    assert _verify(**dict(kw, workspace=P + 64)) == UNSUPPORTED and "workspace" in _said()
    for none in (dict(batch=0), dict(tokens=0), dict(max_q=0)):
        assert _verify(**dict(kw, workspace=0, ws_bytes=0, **none)) == INVALID and "null context" in _said()


def test_attention_workspaces_checked():
    c = _cache(max_pages=4096)
    for heads, batch, q, seq in ((4, 2, 2, 60000), (64, 1, 26, 1500), (64, 16, 32, 6000), (64, 4, 1024, 60000)):
        kw = dict(heads=heads, q_stride=heads * 128, out_stride=heads * 128, batch=batch, tokens=batch * q, max_q=q, max_seq=seq)
        need = lp.lib().lp_attn_tree_ws_bytes(c, heads, batch, batch * q, q, seq)
        assert _attn(c, ws_bytes=need, **kw) == INVALID and "null context" in _said()
        if need:
            assert _attn(c, ws_bytes=need - 1, **kw) == INVALID and "workspace" in _said()
            assert _attn(c, workspace=0, **kw) == INVALID and "null workspace" in _said()
            assert _attn(c, workspace=P + 64, **kw) == UNSUPPORTED and "workspace" in _said()
    assert lp.lib().lp_attn_tree_ws_bytes(c, 64, 16, 512, 32, 6000) > 0
    assert _attn(c, workspace=0, ws_bytes=0, max_q=0, max_seq=60000) == INVALID and "null context" in _said()


# ---- the formulas -------------------------------------------------------------------


def test_ancestors():
    deep, masks = ancestors([-1, 0, 0, 1, 3, 7, -5, 5])
    assert deep == [0, 1, 1, 2, 3, 0, 0, 1]
    assert masks == [1, 3, 5, 11, 27, 32, 64, 160]


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("temp", [1.0, 0.7])
def test_verified_tokens_have_the_targets_distribution(sampled, temp):
    """The first two tokens that come out of trees of five nodes, 20,000 times: their
    frequencies against the target's probabilities.  Each is a binomial count; of the 30 that
    are looked at none may be off by more than 5 of its standard deviations."""
    rng = np.random.default_rng(5 if sampled else 6)
    V, n = 5, 20000
    # the target's rows after each context: none, or one token
    first = rng.standard_normal(V) * 1.2
    second = rng.standard_normal((V, V)) * 1.2
    p1 = np.exp(first / temp) / np.exp(first / temp).sum()
    p2 = np.exp(second / temp) / np.exp(second / temp).sum(1, keepdims=True)
    q1 = np.array([0.4, 0.3, 0.2, 0.05, 0.05], np.float32)
    q2 = np.array([0.1, 0.2, 0.3, 0.2, 0.2], np.float32)
    up = [-1, 0, 0, 1, 1]
    ones, twos = np.zeros(V), np.zeros((V, V))
    for _ in range(n):
        if sampled:  # drawn from q, one by one
            d = np.concatenate(([0], rng.choice(V, 2, p=q1 / q1.sum(dtype=np.float64)), rng.choice(V, 2, p=q2 / q2.sum(dtype=np.float64))))
        else:        # whatever was chosen
            d = np.array([0, 1, 3, 2, 0])
        x = np.stack([first, second[d[1]], second[d[2]], np.zeros(V), np.zeros(V)]).astype(np.float64)
        q = np.stack([q1, q2, q2, q2, q2]) if sampled else None
        path, z = verify_one(x, d, up, temp, rng.random(5), q, 2)
        got = [int(d[i]) for i in path[1:]] + [z]
        ones[got[0]] += 1
        if len(got) > 1:
            twos[got[0], got[1]] += 1
    assert (np.abs(ones - n * p1) <= 5 * np.sqrt(n * p1 * (1 - p1))).all(), (ones / n, p1)
    for a in range(V):
        m = twos[a].sum()
        if m > 500:
            assert (np.abs(twos[a] - m * p2[a]) <= 5 * np.sqrt(m * p2[a] * (1 - p2[a]))).all(), (a, twos[a] / m, p2[a])


def test_random_trees_are_trees():
    rng = np.random.default_rng(0)
    for n in (1, 2, 70):
        up = random_tree(rng, n, 4)
        assert up[0] == -1 and all(0 <= p < i for i, p in enumerate(up) if i) and max(ancestors(up)[0]) <= 4
