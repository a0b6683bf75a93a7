"""The paged KV cache on the GPU: lp_kv_append_paged and lp_attn_paged against
the same formulas in 64 bits (tests/_paged.py), at one token and many, odd and
ragged lengths, pages that end inside a tile, strided rows, padding, empty rows
and pages that are not there; then one behind the other as a program runs them.

Tolerances count roundings.  Appended rows: 64-bit values rounded once (f32:
2^-24 of the value, fp16: 2^-11); their angles are exact to 2^-50 turns, 4-bit
codes are equal.  Attention (fp32 with fp16 hi + lo images of its fp32 operands):
an image leaves 2^-22 of the operand, a score is off by that of its size, |s| <=
|q| |k| scale, and its probability by as much; with |s| up to 16 here that is 2^-18 =
3.8e-6, the fp32 sums of up to 8192 terms in blocks of 64 and less add below
2^-24 x 64 = 3.8e-6: 1e-5 of the largest |v| a row sees."""
import numpy as np
import pytest

import llmpager_amd as lp
from _paged import Batch, HipGraph, q4

pytestmark = pytest.mark.gpu

EPS = 1e-6
ATTN_TOL = 1e-5


@pytest.fixture(scope="module")
def K(cuda):
    return lp.Kernels(cuda)


def _f32(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def _append_inputs(B, pad_cols=0):
    """q, k, v as columns of one projection's output, norms."""
    n = (B.heads + 2 * B.kv) * B.dim + pad_cols
    x = _f32(B.rng, B.tokens, n)
    a, b = B.heads * B.dim, (B.heads + B.kv) * B.dim
    return x, x[:, :a], x[:, a:b], x[:, b:b + B.kv * B.dim], _f32(B.rng, B.dim) + 1, _f32(B.rng, B.dim) + 1


def _append(K, B, x, qw, kw, mscale=1.0, out=True, stream=None):
    """Launch; (q_out, k_out, v_out) device rows preset to 7."""
    W, D = x.shape[1], B.dim
    dx = B.up(x)
    dq = B.up(np.full((B.tokens, B.heads * D), 7, np.float32))
    dko, dvo = (B.up(np.full((B.tokens, B.kv * D), 7, np.float32)) for _ in range(2))
    K.kv_append_paged(B.cache, dx, W, dx + B.heads * D * 4, W, dx + (B.heads + B.kv) * D * 4, W,
                      0 if qw is None else B.up(qw), 0 if kw is None else B.up(kw), EPS, B.up(B.freq), mscale, dq,
                      B.heads * D, dko if out else 0, dvo if out else 0, B.heads, B.dstarts, B.dlens, B.batch, B.tokens,
                      stream)
    return dq, dko, dvo


def _check_append(K, B, mscale=1.0, norms=True, pad_cols=0, out=True):
    x, q, k, v, qw, kw = _append_inputs(B, pad_cols)
    if not norms:
        qw = kw = None
    B.device()
    dq, dko, dvo = _append(K, B, x, qw, kw, mscale, out)
    wq, wk, wv, pools = B.append(q, k, v, qw, kw, EPS, mscale)
    D, n = B.dim, B.live
    got = B.cuda.download(dq, (B.tokens, B.heads, D), np.float32)
    # pairs' products cancel: a rounding of the pair's length, not of the result
    tol = 2.0 ** -23 * np.hypot(wq[..., :D // 2], wq[..., D // 2:])
    assert (np.abs(got[:n] - wq[:n]) <= np.concatenate((tol, tol), -1)[:n]).all()
    assert (got[n:] == 7).all()
    for d, w in ((dko, wk), (dvo, wv)):
        g = B.cuda.download(d, (B.tokens, B.kv, D), np.float32)
        if not out:
            assert (g == 7).all()
            continue
        assert (g[n:] == 7).all()
        if B.fmt == lp.KV_Q4:
            assert np.array_equal(g[:n], w[:n].astype(np.float32))
        else:
            assert np.allclose(g[:n], w[:n], rtol=2.0 ** -10, atol=2.0 ** -24)  # a step, where 64 bits sit on a border
    for d, w in zip((B.dk, B.dv), pools):
        g = B.cuda.download(d, w.shape, np.uint8)
        if B.fmt == lp.KV_Q4:
            assert np.array_equal(g, w)
        else:
            steps = g.view(np.int16).astype(np.int32) - w.view(np.int16)
            assert np.abs(steps).max() <= 1 and (steps != 0).mean() < 1e-3
    B.free()


@pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])
@pytest.mark.parametrize("new,past,heads,kv,dim,page,pad", [
    ([1], [0], 1, 1, 64, 16, 0),                       # the first token of all
    ([1], [1500], 32, 4, 128, 64, 0),
    ([1, 1, 1], [15, 16, 31], 5, 1, 128, 16, 2),       # a page's last, first and last row; padding
    ([17, 1, 64, 3], [0, 250, 5, 13], 6, 2, 64, 32, 1),
    ([0, 9, 0, 2], [8, 3, 0, 60], 4, 4, 128, 256, 0),  # sequences without a new token
    ([40], [131000], 3, 3, 64, 128, 0),                # angles of far positions
])
def test_append(cuda, K, fmt, new, past, heads, kv, dim, page, pad):
    _check_append(K, Batch(cuda, new, past, heads, kv, dim, page, fmt, seed=len(new) + dim, pad=pad))


@pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])
def test_append_without_norms_scaled_strided(cuda, K, fmt):
    _check_append(K, Batch(cuda, [5, 2], [30, 7], 8, 2, 128, 16, fmt, seed=2), mscale=1.25, norms=False, pad_cols=20, out=False)


@pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])
def test_append_many_sequences(cuda, K, fmt):
    """More sequences than lanes: a token finds its own."""
    n = 201
    _check_append(K, Batch(cuda, [1 + (b % 3 == 0) for b in range(n)], [b % 37 for b in range(n)], 2, 1, 64, 16, fmt, seed=n))


@pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])
def test_append_where_no_page_is(cuda, K, fmt):
    """Table entries that name no page, and positions past the table's width:
    the other tokens' rows arrive, nothing else changes."""
    B = Batch(cuda, [40, 40, 5], [0, 8, 70], 4, 2, 64, 16, fmt, seed=8, cols=4)
    B.table[0, 1] = -1
    B.table[1, 0], B.table[1, 2] = B.pages, 2 ** 31 - 1
    _check_append(K, B)


def test_append_in_place(cuda, K):
    """q_out = q and k_out = k."""
    B = Batch(cuda, [3, 4], [5, 40], 4, 4, 128, 32, lp.KV_Q4, seed=4).device()
    q, k, v = (_f32(B.rng, B.tokens, 4 * 128) for _ in range(3))
    dq, dk, dv, f = B.up(q), B.up(k), B.up(v), B.up(B.freq)
    K.kv_append_paged(B.cache, dq, 512, dk, 512, dv, 512, 0, 0, EPS, f, 1.0, dq, 512, dk, dv, 4, B.dstarts, B.dlens, 2,
                      B.tokens)
    wq, wk, wv, _ = B.append(q, k, v, None, None, EPS)
    assert np.allclose(cuda.download(dq, wq.shape, np.float32), wq, atol=2e-6)
    assert np.array_equal(cuda.download(dk, wk.shape, np.float32), wk.astype(np.float32))
    assert np.array_equal(cuda.download(dv, wv.shape, np.float32), wv.astype(np.float32))
    B.free()


def test_append_q4_extremes(cuda, K):
    """Rows of zeros, of one value, of tiny, huge, infinite and NaN values and of
    values on the border of two codes: what the page holds are numbers."""
    B = Batch(cuda, [8], [3], 1, 1, 64, 16, lp.KV_Q4, seed=5).device()
    v = np.zeros((8, 64), np.float32)
    v[1, 5] = 3.0
    v[2] = 1e-9 * np.arange(64)
    v[3] = 1e6 * (np.arange(64) - 30)
    v[4, ::7], v[4, 1::7] = np.inf, -np.inf
    v[5] = np.arange(64)
    v[5, ::9] = np.nan
    v[6] = np.where(np.arange(64) % 32 == 0, 7.0, np.arange(64) % 14 * 0.5 - 3.25)  # scale 1: k + 1/4, k + 3/4
    v[7] = np.where(np.arange(64) % 32 == 0, 7.0, np.arange(64) % 12 - 5.5)         # halves: to the even code
    q = np.zeros((8, 64), np.float32)
    dq, dk, dv = B.up(q), B.up(q), B.up(v)
    do = B.alloc(8 * 64 * 4)
    K.kv_append_paged(B.cache, dq, 64, dk, 64, dv, 64, 0, 0, EPS, B.up(B.freq), 1.0, dq, 64, 0, do, 1, B.dstarts, B.dlens,
                      1, 8)
    codes, s = q4(v.astype(np.float64)[:, None])
    want = ((codes - 8.0).reshape(8, 2, 32) * s.reshape(8, 2, 1)).reshape(8, 64)
    got = cuda.download(do, (8, 64), np.float32)
    assert np.isfinite(got).all() and np.array_equal(got, want.astype(np.float32))
    assert np.array_equal(np.abs(got[4, ::7]), np.full(10, 7 * 896.0))
    B.free()


# ---- attention -----------------------------------------------------------------


def _attn(K, B, q, max_q=None, max_seq=None, out_stride=0, stream=None, ws=None):
    """out [tokens, heads D] over rows preset to 7."""
    W = B.heads * B.dim
    ow = W + out_stride
    dq, do = B.up(q), B.up(np.full((B.tokens, ow), 7, np.float32))
    mq, ms = max_q or max(B.new + [1]), max_seq or max(B.lens + [1])
    n = K.attn_paged_ws_bytes(B.cache, B.heads, B.batch, B.tokens, mq, ms)
    ws = ws or B.alloc(n)
    K.attn_paged(B.cache, dq, q.shape[1], do, ow, B.heads, B.dstarts, B.dlens, B.batch, B.tokens, mq, ms,
                 1.0 / np.sqrt(B.dim), ws, stream, ws_bytes=ws.nbytes)
    return B.cuda.download(do, (B.tokens, ow), np.float32, stream)


def _queries(B, std=1.0, cols=0):
    return (_f32(B.rng, B.tokens, B.heads * B.dim + cols) * std).astype(np.float32)


def _close(got, want, tol=ATTN_TOL):
    fine = np.abs(want[np.isfinite(want)])
    size = fine.max() if fine.size else 0.0
    bad = ~(np.abs(got - want) <= tol * max(size, 1.0)) & ~(np.isnan(got) & np.isnan(want)) & ~(got == want)
    assert not bad.any(), (np.argwhere(bad)[:5], np.nanmax(np.abs(got - want)))


def _check_attn(K, B, **kw):
    cols = kw.pop("cols", 0)
    q = _queries(B, cols=cols)
    B.device()
    W = B.heads * B.dim
    got = _attn(K, B, q, out_stride=cols, **kw)
    want = B.attention(q[:, :W].reshape(B.tokens, B.heads, B.dim), 1.0 / np.sqrt(B.dim), kw.get("max_seq"))
    _close(got[:B.live, :W].reshape(B.live, B.heads, B.dim), want[:B.live])
    assert (got[B.live:] == 7).all() and (got[:, W:] == 7).all()
    B.free()


FORMATS = pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])


@FORMATS
@pytest.mark.parametrize("new,past,heads,kv,dim,page,pad", [
    ([1], [0], 1, 1, 64, 16, 0),                        # one row in all
    ([1], [1500], 32, 4, 128, 64, 0),
    ([1, 1, 1, 1], [62, 63, 64, 65], 8, 2, 128, 16, 3),  # around a tile's end
    ([1] * 5, [0, 700, 15, 16, 2047], 5, 1, 64, 256, 0),
    ([1] * 9, [40 * b for b in range(9)], 24, 8, 64, 32, 1),
    ([1, 1], [3000, 1], 48, 1, 128, 128, 0),            # more heads on one KV head than a tile's rows
    ([1], [8191], 64, 4, 128, 64, 0),
    ([1, 1], [511, 20000], 4, 4, 128, 32, 0),           # a long context
])
def test_attention_of_single_tokens(cuda, K, fmt, new, past, heads, kv, dim, page, pad):
    _check_attn(K, Batch(cuda, new, past, heads, kv, dim, page, fmt, seed=sum(past) + dim, pad=pad))


@FORMATS
@pytest.mark.parametrize("new,past,heads,kv,dim,page,pad", [
    ([2], [0], 1, 1, 64, 16, 0),
    ([5, 3, 1], [600, 0, 63], 16, 2, 128, 64, 0),       # guesses
    ([8, 8], [100, 4000], 16, 1, 64, 16, 2),
    ([17], [0], 4, 4, 128, 32, 0),                      # short prompts, alone in their pages
    ([33, 1, 64, 65], [0, 5, 31, 64], 8, 2, 64, 16, 1),
    ([130, 7], [1, 300], 32, 4, 128, 64, 0),
    ([257], [1000], 6, 2, 128, 128, 0),
    ([300, 0, 200], [0, 50, 77], 5, 1, 64, 256, 5),     # a sequence without a new token, padding
    ([70], [2500], 7, 7, 64, 32, 0),
])
def test_attention_of_several_tokens(cuda, K, fmt, new, past, heads, kv, dim, page, pad):
    _check_attn(K, Batch(cuda, new, past, heads, kv, dim, page, fmt, seed=sum(new) + dim, pad=pad))


@FORMATS
@pytest.mark.parametrize("new,past", [([1, 1, 1], [40, 300, 3]), ([20, 3], [77, 0]), ([200], [130])])
def test_attention_bounds_wider_than_the_batch(cuda, K, fmt, new, past):
    """max_q and max_seq far above what is there, strided rows."""
    _check_attn(K, Batch(cuda, new, past, 8, 2, 128, 32, fmt, seed=77), max_q=max(new) + 300, max_seq=9000, cols=12)


@FORMATS
@pytest.mark.parametrize("new,past", [([1, 1], [500, 90]), ([12, 4], [200, 64]), ([150], [70])])
def test_attention_leaves_absent_pages_out(cuda, K, fmt, new, past):
    """Entries that name no page in the middle, at the start and at the end; a
    sequence none of whose pages is there has zeros."""
    B = Batch(cuda, new, past, 6, 2, 64, 16, fmt, seed=9)
    B.table[0, 2], B.table[0, 5], B.table[0, 0] = -1, B.pages, -2 ** 31
    B.table[0, (B.lens[0] - 1) // 16] = 2 ** 31 - 1
    if len(new) > 1:
        B.table[1] = -1
    _check_attn(K, B)


@FORMATS
@pytest.mark.parametrize("new", [[4, 1], [40, 2], [3, 140]])
def test_attention_of_tokens_without_rows(cuda, K, fmt, new):
    """Lengths below the new tokens' number: the first tokens stand before row 0
    and see nothing, so they get zeros; a length of 0 or less leaves all empty."""
    B = Batch(cuda, new, [0, 0], 4, 2, 128, 16, fmt, seed=3)
    B.lens = [new[0] - 2, -1]
    _check_attn(K, B)


@FORMATS
def test_attention_cut_at_its_bounds(cuda, K, fmt):
    """A length over max_seq, or over the table's width, is taken as that."""
    _check_attn(K, Batch(cuda, [1, 5], [300, 100], 4, 2, 64, 16, fmt, seed=6), max_seq=117)
    B = Batch(cuda, [2], [60], 4, 2, 64, 16, fmt, seed=6, cols=4)
    B.lens = [90]
    _check_attn(K, B)
    # tokens past a sequence's first max_q are left as they were
    B = Batch(cuda, [6, 2], [30, 8], 4, 2, 64, 16, fmt, seed=6)
    q = _queries(B)
    B.device()
    got = _attn(K, B, q, max_q=4).reshape(B.tokens, 4, 64)
    want = B.attention(q.reshape(B.tokens, 4, 64), 1.0 / 8)
    _close(got[[0, 1, 2, 3, 6, 7]], want[[0, 1, 2, 3, 6, 7]])
    assert (got[4:6] == 7).all()
    B.free()


@pytest.mark.parametrize("new,past,heads", [([1], [200], 4), ([6], [70], 4), ([90], [40], 4), ([90], [40], 2)])
def test_attention_hidden_rows_may_hold_anything(cuda, K, new, past, heads):
    """NaN and infinities in rows that a token does not see (the rows behind the
    last in its page, and the later tokens' own) leave its output as it is; the
    tokens that see them get what the formula gives."""
    B = Batch(cuda, new, past, heads, 2, 64, 16, lp.KV_F16, seed=11)
    n, L = new[0], B.lens[0]
    P = B.pools[0].view(np.float16).reshape(B.pages, 2, 16, 64), B.pools[1].view(np.float16).reshape(B.pages, 2, 16, 64)
    for pool in P:  # behind the last row
        pool[B.table[0, (L - 1) // 16], :, (L - 1) % 16 + 1:] = np.nan
    bad = np.full((2, 64), np.nan, np.float16)
    if n > 2:
        B.put(L - 2, bad, bad)
        B.put(L - 1, None, np.where(np.arange(64) % 2, np.inf, -np.inf).astype(np.float16))
    _check_attn(K, B)


def test_attention_large_scores(cuda, K):
    """Scores hundreds apart: one row takes everything, none overflows."""
    B = Batch(cuda, [1, 70], [333, 10], 4, 2, 128, 16, lp.KV_F16, seed=12)
    q = _queries(B, std=60.0)
    B.device()
    got = _attn(K, B, q).reshape(B.tokens, 4, 128)
    want = B.attention(q.reshape(B.tokens, 4, 128), 1.0 / np.sqrt(128.0))
    # |s| up to 60 x 128^.5 x 4 = 2,700: 2^-22 of it moves a probability by 7e-4
    _close(got, want, 2e-3)
    B.free()


def test_attention_other_stream_and_two_at_once(cuda, K):
    """Two calls with a workspace each on two streams, neither the null stream."""
    Bs = [Batch(cuda, n, p, 8, 2, 128, 32, f, seed=20 + i) for i, (n, p, f) in enumerate(
        [([1, 1], [4000, 900], lp.KV_Q4), ([3, 40], [1000, 100], lp.KV_F16)])]
    qs, outs, streams = [], [], [cuda.stream(), cuda.stream()]
    for B in Bs:
        qs.append(_queries(B))
        B.device()
    cuda.sync()
    W = 8 * 128
    args = []
    for B, q in zip(Bs, qs):
        n = K.attn_paged_ws_bytes(B.cache, 8, B.batch, B.tokens, max(B.new), max(B.lens))
        args.append((B.up(q), B.alloc(B.tokens * W * 4), B.alloc(n)))
    cuda.sync()
    for _ in range(5):
        for B, s, (dq, do, ws) in zip(Bs, streams, args):
            K.attn_paged(B.cache, dq, W, do, W, 8, B.dstarts, B.dlens, B.batch, B.tokens, max(B.new), max(B.lens),
                         1.0 / np.sqrt(128.0), ws, s, ws_bytes=ws.nbytes)
    cuda.sync()
    for B, q, (_, do, _) in zip(Bs, qs, args):
        _close(cuda.download(do, (B.tokens, 8, 128), np.float32),
               B.attention(q.reshape(B.tokens, 8, 128), 1.0 / np.sqrt(128.0)))
    for s in streams:
        cuda.destroy_stream(s)
    for B in Bs:
        B.free()


@FORMATS
@pytest.mark.parametrize("new,past", [([1, 1, 1], [900, 30, 2]), ([4, 150], [70, 0])])
def test_attention_same_call_same_bits(cuda, K, fmt, new, past):
    B = Batch(cuda, new, past, 16, 2, 128, 16, fmt, seed=30)
    q = _queries(B)
    B.device()
    first = _attn(K, B, q)
    for _ in range(3):
        assert np.array_equal(_attn(K, B, q), first)
    B.free()


# ---- one behind the other ----------------------------------------------------------


@FORMATS
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (6, 1, 64)])
def test_prompts_then_tokens(cuda, K, fmt, heads, kv, dim):
    """Prompts in two chunks, then single tokens, each append behind the last:
    what a serving program runs, against the formulas over the same pages."""
    prompt, chunk, steps = [70, 23, 131], [40, 23, 64], 3
    qw, kw = None, None
    have = [0, 0, 0]
    rng = np.random.default_rng(40)
    pages = Batch(cuda, [p + steps for p in prompt], [0, 0, 0], heads, kv, dim, 16, fmt, seed=41)
    table, pools = pages.table, pages.pools
    rounds = [chunk, [p - c for p, c in zip(prompt, chunk)]] + [[1, 1, 1]] * steps
    qw, kw = _f32(rng, dim) + 1, _f32(rng, dim) + 1
    for i, new in enumerate(rounds):
        B = Batch(cuda, new, have, heads, kv, dim, 16, fmt, seed=50 + i, spare=3)
        B.pages, B.cols, B.table, B.pools = pages.pages, pages.cols, table, pools
        x, q, k, v, _, _ = _append_inputs(B)
        B.device()
        dq, _, _ = _append(K, B, x, qw, kw, out=False)
        _, _, _, want = B.append(q, k, v, qw, kw, EPS)
        got = [cuda.download(d, want[0].shape, np.uint8) for d in (B.dk, B.dv)]
        if fmt == lp.KV_Q4:
            assert all(np.array_equal(g, w) for g, w in zip(got, want))
        B.pools = pools = got
        W = heads * dim
        do, n = B.alloc(B.tokens * W * 4), K.attn_paged_ws_bytes(B.cache, heads, 3, B.tokens, max(new), max(B.lens))
        ws = B.alloc(n)
        K.attn_paged(B.cache, dq, W, do, W, heads, B.dstarts, B.dlens, 3, B.tokens, max(new), max(B.lens),
                     1.0 / np.sqrt(dim), ws, ws_bytes=ws.nbytes)
        out = cuda.download(do, (B.tokens, heads, dim), np.float32)
        q = cuda.download(dq, (B.tokens, heads, dim), np.float32)
        _close(out, B.attention(q, 1.0 / np.sqrt(dim)))
        have = B.lens
        B.free()


@FORMATS
def test_captured_step_replayed_with_other_lengths(cuda, K, fmt):
    """Append and attention captured once; replays take the lengths, tables and
    rows that are in device memory then, with eager work between them."""
    heads, kv, dim, page, batch, most = 8, 2, 128, 16, 4, 600
    s = cuda.stream()
    B = Batch(cuda, [1] * batch, [most - 1] * batch, heads, kv, dim, page, fmt, seed=60).device()
    W = heads * dim
    dx, dq, do = B.alloc(batch * (heads + 2 * kv) * dim * 4), B.alloc(batch * W * 4), B.alloc(batch * W * 4)
    df = B.up(B.freq)
    row = (heads + 2 * kv) * dim
    ws = B.alloc(K.attn_paged_ws_bytes(B.cache, heads, batch, batch, 1, most))
    cuda.sync()

    def launch(stream):
        K.kv_append_paged(B.cache, dx, row, dx + W * 4, row, dx + (heads + kv) * dim * 4, row, 0, 0, EPS, df, 1.0, dq, W,
                          0, 0, heads, B.dstarts, B.dlens, batch, batch, stream)
        K.attn_paged(B.cache, dq, W, do, W, heads, B.dstarts, B.dlens, batch, batch, 1, most, 1.0 / np.sqrt(dim), ws,
                     stream, ws_bytes=ws.nbytes)

    cuda.capture_begin(s)
    launch(s)
    g = cuda.capture_end(s)
    rng = np.random.default_rng(61)
    for lens in ([600, 1, 64, 300], [2, 17, 65, 599], [33, 34, 35, 36], [600, 600, 600, 600]):
        x = _f32(rng, batch, row)
        cuda.htod_async(dx, x, s)
        cuda.htod_async(B.dlens, np.asarray(lens, np.int32), s)
        cuda.sync_stream(s)
        g.launch(s)
        out = cuda.download(do, (batch, heads, dim), np.float32, s)
        B.pools = [cuda.download(d, B.pools[0].shape, np.uint8, s) for d in (B.dk, B.dv)]
        q = cuda.download(dq, (batch, heads, dim), np.float32, s)
        B.lens, B.past = lens, [n - 1 for n in lens]
        _close(out, B.attention(q, 1.0 / np.sqrt(dim)))
        # the same, eagerly
        launch(s)
        assert np.array_equal(cuda.download(do, (batch, heads, dim), np.float32, s), out)
    g.close()
    cuda.destroy_stream(s)
    B.free()


@FORMATS
@pytest.mark.parametrize("new,past,heads,kv", [
    ([1] * 70, [11 * b for b in range(70)], 4, 2),          # more sequences than lanes
    ([1 + b % 3 for b in range(130)], [b for b in range(130)], 8, 1),
    ([1] * 1030, [b % 90 for b in range(1030)], 2, 1),      # more than share their contexts out
    ([1] * 600, [b % 50 for b in range(600)], 4, 4),        # more (sequence, KV head)s than have counters
    ([20 + b % 7 for b in range(66)], [3 * b for b in range(66)], 8, 2),
])
def test_attention_many_sequences(cuda, K, fmt, new, past, heads, kv):
    _check_attn(K, Batch(cuda, new, past, heads, kv, 64, 16, fmt, seed=len(new)))


@FORMATS
@pytest.mark.parametrize("new,past", [([9, 40], [3000, 1500]), ([70, 33], [4100, 64]), ([64], [6000]), ([128], [191])])
def test_attention_many_rows_of_long_contexts(cuda, K, fmt, new, past):
    """Contexts in spans that end inside a sequence and behind the shorter one."""
    _check_attn(K, Batch(cuda, new, past, 8, 2, 128, 32, fmt, seed=40))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,past", [([48], [2000]), ([130], [500])])
def test_attention_seen_rows_that_are_no_numbers(cuda, K, dim, new, past):
    """Infinities in a value row that the later tokens see and the earlier do not,
    among them two of one column with opposite signs; a value row of NaN that all
    see in some columns."""
    B = Batch(cuda, new, past, 8, 2, dim, 16, lp.KV_F16, seed=41)
    v = np.ones((2, dim), np.float16)
    v[:, 3], v[:, 7] = np.inf, -np.inf
    B.put(past[0] + 20, None, v)
    w = np.zeros((2, dim), np.float16)
    w[:, 7] = np.inf
    B.put(past[0] + 30, None, w)
    u = np.zeros((2, dim), np.float16)
    u[0, 5] = np.nan
    B.put(100, None, u)
    _check_attn(K, B)


@pytest.mark.parametrize("new,past", [([1, 1], [3000, 40]), ([3, 30], [900, 70])])
def test_graphs_of_one_stream_replayed_at_once(cuda, K, new, past):
    """Two graphs that the program captured itself from one stream, replayed on two
    others beside eager calls on that stream: three workspaces, nothing else shared."""
    Bs = [Batch(cuda, new, past, 8, 2, 128, 32, lp.KV_Q4, seed=50 + i) for i in range(3)]
    qs = [_queries(B) for B in Bs]
    W, mq, ms = 8 * 128, max(new), max(Bs[0].lens)
    args = []
    for B, q in zip(Bs, qs):
        B.device()
        args.append((B.up(q), B.alloc(B.tokens * W * 4), B.alloc(K.attn_paged_ws_bytes(B.cache, 8, B.batch, B.tokens, mq, ms))))
    cuda.sync()

    def launch(i, stream):
        B, (dq, do, ws) = Bs[i], args[i]
        for _ in range(3):
            K.attn_paged(B.cache, dq, W, do, W, 8, B.dstarts, B.dlens, B.batch, B.tokens, mq, ms, 1.0 / np.sqrt(128.0), ws,
                         stream, ws_bytes=ws.nbytes)

    s, s0, s1 = (cuda.stream() for _ in range(3))
    g0, g1 = (HipGraph(s, lambda st, i=i: launch(i, st)) for i in range(2))
    want = [B.attention(q.reshape(B.tokens, 8, 128), 1.0 / np.sqrt(128.0)) for B, q in zip(Bs, qs)]
    for _ in range(4):
        for B, (_, do, _) in zip(Bs, args):
            cuda.htod_async(do, np.full((B.tokens, W), 7, np.float32), s)
        cuda.sync()
        for _ in range(5):
            g0.launch(s0)
            g1.launch(s1)
            launch(2, s)
        for st in (s, s0, s1):
            cuda.sync_stream(st)
        for B, (_, do, _), w in zip(Bs, args, want):
            _close(cuda.download(do, (B.tokens, 8, 128), np.float32), w)
    g0.close()
    g1.close()
    for st in (s, s0, s1):
        cuda.destroy_stream(st)
    for B in Bs:
        B.free()


def test_attention_on_more_streams_than_have_counters(cuda, K):
    """The same bits on 70 streams, whether the counters are a stream's or the
    workspace's."""
    B = Batch(cuda, [1, 1], [2500, 300], 8, 2, 128, 16, lp.KV_Q4, seed=52)
    q = _queries(B)
    B.device()
    streams = [cuda.stream() for _ in range(70)]
    outs = [_attn(K, B, q, stream=s) for s in streams]
    _close(outs[0].reshape(2, 8, 128), B.attention(q.reshape(2, 8, 128), 1.0 / np.sqrt(128.0)))
    for o in outs[1:]:
        assert np.array_equal(o, outs[0])
    for s in streams:
        cuda.destroy_stream(s)
    B.free()


@FORMATS
@pytest.mark.parametrize("new,past,heads,kv,dim", [
    ([2, 1], [3000, 700], 32, 2, 128),      # 32 query rows of a KV head, and 16 of them
    ([4], [2000], 6, 1, 128),
    ([3, 3, 1], [900, 4000, 0], 8, 1, 64),
    ([1, 1], [2000, 130], 12, 1, 128),
    ([1], [9000], 17, 1, 64),
    ([8, 2, 5], [1500, 6000, 31], 16, 4, 128),
])
def test_attention_of_two_tiles_in_parts(cuda, K, fmt, new, past, heads, kv, dim):
    """9 to 32 query rows of a KV head over contexts in parts: every share of the
    threads that join them."""
    _check_attn(K, Batch(cuda, new, past, heads, kv, dim, 16, fmt, seed=heads))
