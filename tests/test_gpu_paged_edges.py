"""lp_kv_append_paged and lp_attn_paged where they are most easily wrong: part of a
batch's sequences, one row far above thousands of others, values that are no finite
numbers in any place."""
import numpy as np
import pytest

import llmpager_amd as lp
from _paged import GROUP, Batch, q4
from test_gpu_paged import ATTN_TOL, EPS, FORMATS, _append_inputs, _attn, _close, _f32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(cuda):
    return lp.Kernels(cuda)


# ---- part of a batch's sequences ------------------------------------------------


def _of_sequences(B, b0):
    """The cache as sequences b0 .. of the batch have it."""
    return lp.KvCache(k_pages=B.dk, v_pages=B.dv, table=B.dtable + b0 * B.cols * 4, pages=B.pages, page_rows=B.page,
                      max_pages=B.cols, kv_heads=B.kv, head_dim=B.dim, format=B.fmt)


@FORMATS
@pytest.mark.parametrize("new,past,b0,b1", [
    ([5, 3, 1], [40, 95, 7], 1, 3),
    ([5, 3, 1], [40, 95, 7], 2, 3),                       # one sequence behind eight tokens
    ([4, 4, 4, 4], [30, 33, 200, 64], 1, 3),              # and tokens behind them
    ([3] * 140, [10 + b % 50 for b in range(140)], 70, 138),
])
def test_append_of_some_sequences(cuda, K, fmt, new, past, b0, b1):
    """q_starts + b0: tokens before that sequence's first belong to none; their rows
    and every page of theirs stay as they are, byte for byte."""
    B = Batch(cuda, new, past, 4, 2, 64, 16, fmt, seed=70 + b0, pad=2)
    x, q, k, v, qw, kw = _append_inputs(B)
    B.device()
    W, D = x.shape[1], 64
    dx, df, dqw, dkw = B.up(x), B.up(B.freq), B.up(qw), B.up(kw)
    dq, dko, dvo = (B.up(np.full((B.tokens, n * D), 7, np.float32)) for n in (4, 2, 2))
    K.kv_append_paged(_of_sequences(B, b0), dx, W, dx + 4 * D * 4, W, dx + 6 * D * 4, W, dqw, dkw, EPS, df, 1.0, dq, 4 * D,
                      dko, dvo, 4, B.dstarts + b0 * 4, B.dlens + b0 * 4, b1 - b0, B.tokens)
    wq, wk, wv, pools = B.append(q, k, v, qw, kw, EPS)
    t0, t1 = int(B.starts[b0]), int(B.starts[b1])
    mine = np.zeros(B.pages, bool)
    for b in range(b0, b1):
        mine[B.table[b, :-(-B.lens[b] // 16)]] = True
    for d, w, was in zip((B.dk, B.dv), pools, B.pools):
        got = cuda.download(d, w.shape, np.uint8)
        assert np.array_equal(got[~mine], was[~mine])
        if fmt == lp.KV_Q4:
            assert np.array_equal(got[mine], w[mine])
        else:
            assert np.abs(got[mine].view(np.int16).astype(np.int32) - w[mine].view(np.int16)).max() <= 1
    for d, w in ((dq, wq), (dko, wk), (dvo, wv)):
        got = cuda.download(d, w.shape, np.float32)
        assert (got[:t0] == 7).all() and (got[t1:] == 7).all()
        assert np.allclose(got[t0:t1], w[t0:t1], rtol=2.0 ** -10, atol=1e-5)
    B.free()


@FORMATS
@pytest.mark.parametrize("new,past,b0,b1", [
    ([5, 3, 1], [40, 95, 7], 1, 3), ([1, 1, 1, 1], [900, 33, 2000, 64], 1, 3), ([50, 40, 3, 60], [30, 700, 5, 64], 1, 3)])
def test_attention_of_some_sequences(cuda, K, fmt, new, past, b0, b1):
    B = Batch(cuda, new, past, 4, 2, 64, 16, fmt, seed=80 + b0)
    q = _f32(B.rng, B.tokens, 4 * 64)
    B.device()
    dq, do = B.up(q), B.up(np.full((B.tokens, 256), 7, np.float32))
    c, n = _of_sequences(B, b0), b1 - b0
    mq, ms = max(new[b0:b1]), max(B.lens[b0:b1])
    ws = B.alloc(K.attn_paged_ws_bytes(c, 4, n, B.tokens, mq, ms))
    K.attn_paged(c, dq, 256, do, 256, 4, B.dstarts + b0 * 4, B.dlens + b0 * 4, n, B.tokens, mq, ms, 0.125, ws,
                 ws_bytes=ws.nbytes)
    got = cuda.download(do, (B.tokens, 4, 64), np.float32)
    t0, t1 = int(B.starts[b0]), int(B.starts[b1])
    assert (got[:t0] == 7).all() and (got[t1:] == 7).all()
    _close(got[t0:t1], B.attention(q.reshape(B.tokens, 4, 64), 0.125)[t0:t1])
    B.free()


# ---- one row far above the others ------------------------------------------------
# In units of the largest probability: an image's smallest step is 2^-24 of 2^9, so a
# small probability is off by 2^-34 at most, N of them, all alike, by N 2^-34 (2.3e-5 at
# 400,000); an fp32 sum that holds the large one is rounded by 2^-24 of it a matrix product
# of 16 or 32 rows and image, for 1,024 rows or fewer before it is put aside: 2^7 2^-24 =
# 7.6e-6; the sums put aside are one addition per 1,024 rows, of either sign as the values
# vary: a quarter of 2^-24 x 200 = 3e-6.  Together 3.4e-5 of the mean |v|, which is below a
# third of the largest here: 1e-5 of that.


class Shared:
    """`seqs` sequences over one context of `rows` rows, `new` query tokens each: rows
    `at` have `gap` nats more than the others, values a common part."""

    def __init__(self, cuda, fmt, dim, rows, at, gap, seqs, new, heads, pad=0, spread=0.0, seed=0):
        page = 256
        B = self.B = Batch(cuda, [new], [page], heads, 1, dim, page, fmt, seed=seed)
        rng = B.rng
        cols = -(-rows // page)
        B.pages, B.cols, B.batch = cols, cols, seqs
        order = rng.permutation(cols).astype(np.int32)
        B.table = np.tile(order, (seqs, 1))
        B.lens, B.new = [rows] * seqs, [new] * seqs
        B.live, B.tokens = seqs * new, seqs * new + pad
        B.starts = (np.arange(seqs + 1) * new).astype(np.int32)
        k = rng.standard_normal((cols * page, dim), np.float32) * np.float32(spread)
        k[at] = gap / np.sqrt(dim)
        v = 1 + rng.standard_normal((cols * page, dim), np.float32) / 2
        B.pools, self.held = [], []
        for x in (k, v):
            if fmt == lp.KV_F16:
                y = x.astype(np.float16)
                held, raw = y.astype(np.float64), y.view(np.uint8).reshape(cols, -1)
            else:
                codes, s = q4(x.astype(np.float64))
                held = ((codes - 8.0).reshape(len(x), -1, GROUP) * s[..., None]).reshape(len(x), -1)
                raw = np.concatenate((s.astype(np.float16).view(np.uint8).reshape(cols, -1),
                                      (codes[:, 0::2] | codes[:, 1::2] << 4).reshape(cols, -1)), 1)
            pool = np.empty((cols, 1, raw.shape[1]), np.uint8)
            pool[order, 0] = raw
            B.pools.append(pool)
            self.held.append(held[:rows])
        # every sequence asks the same
        self.q = (1.0 + 0.01 * rng.standard_normal((new, heads, dim))).astype(np.float32)
        self.rows = rows

    def check(self, K, **kw):
        B, n, H = self.B, len(self.q), self.B.heads
        q = np.zeros((B.tokens, H * B.dim), np.float32)
        q[:B.live] = np.tile(self.q.reshape(n, -1), (B.batch, 1))
        B.device()
        got = _attn(K, B, q, max_seq=self.rows, **kw)
        k, v = self.held
        want = np.empty((n, H, B.dim))
        for i in range(n):
            L = self.rows - n + 1 + i
            s = self.q[i].astype(np.float64) @ k[:L].T / np.sqrt(B.dim)
            p = np.exp(s - s.max(-1, keepdims=True))
            want[i] = p @ v[:L] / p.sum(-1, keepdims=True)
        got = got[:B.live].reshape(B.batch, n, H, B.dim)
        err = np.abs(got - want).max()
        print("largest error", err, "of", np.abs(v).max())
        assert err <= ATTN_TOL * np.abs(v).max()
        B.free()


@FORMATS
@pytest.mark.parametrize("dim,rows,gap,at,spread", [
    (128, 8192, 12.0, 0, 0.0), (64, 8192, 15.0, 0, 0.3), (128, 8192, 17.0, 0, 0.0), (64, 8192, 18.0, 4000, 0.0),
    (128, 8192, 18.0, 8100, 0.2), (64, 100003, 12.0, 0, 0.0), (128, 100003, 17.0, 5, 0.0), (64, 100003, 19.0, 0, 0.3),
    (128, 100003, 20.0, 70000, 0.0), (128, 100003, 24.0, 3, 0.0)])
def test_one_row_above_many_many_query_rows(cuda, K, fmt, dim, rows, gap, at, spread):
    """40 query rows that walk the whole context (bounds as if there were 512 tiles)."""
    Shared(cuda, fmt, dim, rows, at, gap, 1, 5, 8, pad=8192, spread=spread, seed=int(gap)).check(K, max_q=8192)


@FORMATS
@pytest.mark.parametrize("rows,gap", [(8192, 17.0), (100003, 17.0), (100003, 19.0)])
def test_one_row_above_many_in_spans(cuda, K, fmt, rows, gap):
    Shared(cuda, fmt, 128, rows, 9, gap, 1, 5, 8, seed=int(gap)).check(K)


@FORMATS
@pytest.mark.parametrize("dim,seqs,heads,new,rows,gap,at", [
    (64, 512, 2, 1, 32768, 12.0, 0), (128, 512, 2, 1, 32768, 17.0, 0), (64, 512, 5, 4, 32768, 18.0, 20000),
    (128, 256, 9, 2, 32768, 17.0, 32000), (64, 512, 2, 1, 400003, 13.0, 7), (64, 512, 2, 1, 400003, 17.0, 0),
    (64, 512, 5, 4, 400003, 19.0, 3), (128, 512, 2, 1, 400003, 17.0, 300000), (128, 256, 9, 2, 400003, 18.0, 0),
    (128, 512, 2, 1, 400003, 24.0, 0)])
def test_one_row_above_many_few_query_rows(cuda, K, fmt, dim, seqs, heads, new, rows, gap, at):
    """As many sequences as workgroups: each walks a whole context, its waves a quarter
    of it each."""
    Shared(cuda, fmt, dim, rows, at, gap, seqs, new, heads, seed=int(gap)).check(K)


RISING = (np.array([100, 3000, 6000, 20000]), np.array([[13.0], [17.0], [24.0], [33.0]]))
FALLING = (np.array([100, 3000, 6000, 20000]), np.array([[33.0], [30.0], [22.0], [19.0]]))


@FORMATS
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("at,gap", [RISING, FALLING])
@pytest.mark.parametrize("seqs,new,heads,pad", [(1, 5, 8, 8192), (512, 1, 2, 0)])
def test_rows_above_what_came_before(cuda, K, fmt, dim, at, gap, seqs, new, heads, pad):
    """Four large rows one behind the other: sums put aside at one base and met at
    another, by many query rows and by few."""
    Shared(cuda, fmt, dim, 33001, at, gap, seqs, new, heads, pad=pad, seed=dim).check(K, max_q=8192 if pad else None)


@FORMATS
@pytest.mark.parametrize("rows,gap", [(8192, 17.0), (100003, 18.0)])
def test_one_row_above_many_in_parts(cuda, K, fmt, rows, gap):
    Shared(cuda, fmt, 128, rows, 1, gap, 1, 1, 8, seed=int(gap)).check(K)


# ---- values that are no finite numbers ---------------------------------------------


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,past,heads,kv", [
    ([1], [700], 4, 2), ([1, 1, 1], [4000, 33, 300], 16, 2), ([3], [900], 8, 2), ([7, 2], [2000, 600], 8, 2)])
def test_few_rows_see_no_numbers(cuda, K, dim, new, past, heads, kv):
    """Infinities that every query sees, in chunks that are whole and in the last one:
    of the row with the largest score, of one with hardly any probability, two of
    opposite signs in one column, a NaN."""
    B = Batch(cuda, new, past, heads, kv, dim, 16, lp.KV_F16, seed=90 + dim)
    q = _f32(B.rng, B.tokens, heads * dim)
    for b, L in enumerate(B.lens):
        rows = B.rng.permutation(min(L, past[b]))[:6]
        first = q[int(B.starts[b])].reshape(kv, -1, dim)[:, 0]
        B.put(int(rows[0]), first.astype(np.float16), None, b)              # the largest score
        B.put(int(rows[1]), (-2 * first).astype(np.float16), None, b)       # about 34 nats below
        for i, (c, x) in enumerate([(3, np.inf), (7, -np.inf), (9, np.inf), (9, -np.inf), (11, np.nan), (13, -np.inf)]):
            v = B.rng.standard_normal((kv, dim)).astype(np.float16)
            v[:, c] = x
            B.put(int(rows[i]), None, v, b)
        w = np.ones((kv, dim), np.float16)
        w[:, 17] = np.inf
        B.put(L - new[b], None, w, b)  # in the last chunk
    B.device()
    got = _attn(K, B, q).reshape(B.tokens, heads, dim)
    want = B.attention(q.reshape(B.tokens, heads, dim), 1.0 / np.sqrt(dim))
    assert np.isinf(want).any() and np.isnan(want).any()
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True)
    _close(got[fine], want[fine])
    B.free()


# ---- one prompt's bound for many sequences ---------------------------------------------


@FORMATS
def test_a_prompt_and_many_single_tokens(cuda, K, fmt):
    """64 sequences, one with 150 new tokens and the others with one, bounds of 2,048
    new tokens: 65,536 blocks of 128 query rows, almost all of them empty."""
    B = Batch(cuda, [1] * 20 + [150] + [1] * 43, [30 * b % 700 for b in range(64)], 64, 4, 64, 16, fmt, seed=7, pad=2048 - 213)
    q = _f32(B.rng, B.tokens, 64 * 64)
    B.device()
    got = _attn(K, B, q, max_q=2048, max_seq=1000)
    _close(got[:B.live].reshape(-1, 64, 64), B.attention(q.reshape(-1, 64, 64), 0.125)[:B.live])
    assert (got[B.live:] == 7).all()
    B.free()
