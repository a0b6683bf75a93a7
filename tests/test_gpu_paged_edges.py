"""lp_kv_append_paged and lp_attn_paged where they are most easily wrong: part of a
batch's sequences."""
import numpy as np
import pytest

import llmpager_amd as lp
from _paged import Batch
from test_gpu_paged import EPS, FORMATS, _append_inputs, _close, _f32

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
