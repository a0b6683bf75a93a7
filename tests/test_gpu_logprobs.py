"""lp_logprobs on the GPU against 64 bits (tests/_paged.py).

Tolerances: a term e^(x - M) is off by the rounding of x - M (2^-24 of it), of the
exponential's argument and of itself, under 2^-22 (1 + |x - M|) in all; terms that
matter to a sum have |x - M| < 20, so sums and log S are off by at most 20 x 2^-22 =
5e-6 and, as the terms' errors are of either sign, by far less; the result is
rounded to fp32 (2^-24 of up to 40).  1e-5 covers both."""
import numpy as np
import pytest

import llmpager_amd as lp
from _paged import HipGraph, logprobs

pytestmark = pytest.mark.gpu

TOL = 1e-5


@pytest.fixture(scope="module")
def K(cuda):
    return lp.Kernels(cuda)


def _run(cuda, K, x, targets, top, stride=None, entropy=True, stream=None, launches=1):
    R, V = x.shape
    stride = stride or V
    wide = np.full((R, stride), 1e30, np.float32)  # what stands between the rows
    wide[:, :V] = x
    dx = cuda.upload(wide)
    dt = cuda.upload(np.asarray(targets, np.int32)) if targets is not None else 0
    dl, de = (cuda.upload(np.full(R, 7, np.float32)) for _ in range(2))
    di, dp = (cuda.upload(np.full((R, max(top, 1)), 7, t)) for t in (np.int32, np.float32))
    ws = cuda.alloc_device(max(256, K.logprobs_ws_bytes(R, V, top)))
    cuda.sync()
    for _ in range(launches):
        K.logprobs(dx, stride, R, V, dt, dl if dt else 0, de if entropy else 0, top, di, dp, ws, stream,
                   ws_bytes=ws.nbytes)
    got = [cuda.download(d, s, t, stream) for d, s, t in
           ((dl, (R,), np.float32), (de, (R,), np.float32), (di, (R, max(top, 1)), np.int32), (dp, (R, max(top, 1)), np.float32))]
    for p in (dx, dl, de, di, dp, ws) + ((dt,) if dt else ()):
        cuda.free_device(p)
    return got


def _same(got, want, tol=TOL):
    ok = np.isclose(got, want, rtol=tol, atol=tol, equal_nan=True) | (got == want)
    assert ok.all(), (np.argwhere(~ok)[:5], got[~ok][:5], want[~ok][:5])


def _check(cuda, K, x, targets, top, **kw):
    logp, ent, ids, tp = _run(cuda, K, x, targets, top, **kw)
    wl, we, wi, wt = logprobs(x, np.asarray(targets), top)
    _same(logp, wl)
    _same(ent, we)
    if top:
        assert np.array_equal(ids, wi)
        _same(tp, wt)


@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (1, 2, 0), (3, 63, 5), (2, 64, 64), (5, 65, 1), (1, 255, 20), (4, 257, 8), (7, 1000, 64), (2, 4099, 20),
    (1, 151936, 20), (3, 151936, 0), (33, 32003, 5), (300, 2049, 3), (1, 200001, 64)])
def test_logprobs(cuda, K, rows, vocab, top):
    rng = np.random.default_rng(rows * vocab + top)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    _check(cuda, K, x, rng.integers(0, vocab, rows), top)


@pytest.mark.parametrize("vocab", [1000, 4099, 100003])
def test_strided_rows_and_targets_outside(cuda, K, vocab):
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((6, vocab)).astype(np.float32)
    _check(cuda, K, x, [0, vocab - 1, -1, vocab, 2 ** 31 - 1, 5], 7, stride=vocab + 3)


@pytest.mark.parametrize("vocab", [70, 3001, 151936])
def test_equal_logits_lowest_id_first(cuda, K, vocab):
    """Few distinct values (signed zeros among them), one for all, and blocks of
    the largest at the row's ends."""
    rng = np.random.default_rng(vocab)
    x = rng.integers(-2, 3, (4, vocab)).astype(np.float32)
    x[0][x[0] == 0] = np.where(np.arange((x[0] == 0).sum()) % 2, 0.0, -0.0)
    x[1] = 1.25
    x[2, :40], x[2, -40:] = 9.0, 9.0
    x[3] = -np.arange(vocab)[::-1] // 3
    _check(cuda, K, x, [3, 0, vocab - 1, vocab // 2], 64)


@pytest.mark.parametrize("order", ["rising", "falling"])
def test_sorted_rows(cuda, K, order):
    x = np.arange(20011, dtype=np.float32)[None] * 1e-3
    _check(cuda, K, x if order == "rising" else x[:, ::-1].copy(), [77], 64)


@pytest.mark.parametrize("vocab", [500, 50021])
def test_masked_and_sure_rows(cuda, K, vocab):
    """-inf for most tokens, for all but one and the type's lowest value; rows
    that are all but certain, whose entropy is in the small terms."""
    rng = np.random.default_rng(vocab)
    x = (rng.standard_normal((6, vocab)) * 2).astype(np.float32)
    x[0, rng.random(vocab) < 0.99] = -np.inf
    x[0, 3] = 1.0
    x[1] = -np.inf
    x[1, vocab - 2] = -5.0
    x[2, rng.random(vocab) < 0.5] = np.finfo(np.float32).min
    x[3, 17] += 25.0
    x[4] *= 1e4
    x[5] = -1e30
    _check(cuda, K, x, [3, vocab - 2, 9, 17, int(x[4].argmax()), 0], 20)
    # a masked token's own log probability
    logp = _run(cuda, K, x[1:2], [0], 0)[0]
    assert logp[0] == -np.inf
    # an entropy of e^-10 or so, to fp32's precision of it
    y = np.zeros((1, vocab), np.float32) - 20.0
    y[0, 5] = 0.0
    _, ent, _, _ = _run(cuda, K, y, [5], 0)
    want = logprobs(y, np.array([5]), 0)[1]
    assert abs(ent[0] / want[0] - 1) < 1e-5


@pytest.mark.parametrize("vocab", [300, 40009])
def test_rows_without_probabilities(cuda, K, vocab):
    """NaN, +inf or nothing but -inf: NaN for what cannot be said, ids of the
    numbers there are."""
    x = np.random.default_rng(1).standard_normal((4, vocab)).astype(np.float32)
    x[0, ::2] = np.nan
    x[1, 7] = np.inf
    x[2] = -np.inf
    x[3] = np.nan
    x[3, 10] = 1.0
    logp, ent, ids, tp = _run(cuda, K, x, [1, 2, 3, 10], 4)
    assert np.isnan(logp).all() and np.isnan(ent).all() and np.isnan(tp).all()
    want = np.argsort(-np.where(np.isnan(x[0]), -np.inf, x[0]), kind="stable")[:4]
    assert np.array_equal(ids[0], want) and ids[1, 0] == 7
    assert np.array_equal(ids[2], [0, 1, 2, 3]) and np.array_equal(ids[3], [10, -1, -1, -1])


def test_parts_not_wanted(cuda, K):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((3, 5003)).astype(np.float32)
    wl, we, wi, wt = logprobs(x, np.array([1, 2, 3]), 6)
    logp, ent, ids, tp = _run(cuda, K, x, None, 6, entropy=False)
    assert (logp == 7).all() and (ent == 7).all() and np.array_equal(ids, wi)
    logp, ent, ids, tp = _run(cuda, K, x, [1, 2, 3], 0)
    _same(logp, wl)
    _same(ent, we)
    assert (ids == 7).all() and (tp == 7).all()


def test_other_stream_again_and_again(cuda, K):
    s = cuda.stream()
    rng = np.random.default_rng(6)
    x = rng.standard_normal((2, 151936)).astype(np.float32)
    _check(cuda, K, x, [5, 6], 20, stream=s, launches=4)
    cuda.destroy_stream(s)


def test_captured(cuda, K):
    """Replays read the logits and targets that are there then."""
    rng = np.random.default_rng(7)
    R, V, top = 3, 60013, 10
    s = cuda.stream()
    dx, dt = cuda.alloc_device(R * V * 4), cuda.alloc_device(R * 4)
    dl, de, di, dp = (cuda.alloc_device(n) for n in (R * 4, R * 4, R * top * 4, R * top * 4))
    ws = cuda.alloc_device(max(256, K.logprobs_ws_bytes(R, V, top)))
    cuda.sync()
    cuda.capture_begin(s)
    K.logprobs(dx, V, R, V, dt, dl, de, top, di, dp, ws, s, ws_bytes=ws.nbytes)
    g = cuda.capture_end(s)
    for i in range(4):
        x, t = (rng.standard_normal((R, V)) * (i + 1)).astype(np.float32), rng.integers(0, V, R).astype(np.int32)
        cuda.htod_async(dx, x, s)
        cuda.htod_async(dt, t, s)
        cuda.sync_stream(s)
        g.launch(s)
        wl, we, wi, wt = logprobs(x, t, top)
        _same(cuda.download(dl, (R,), np.float32, s), wl)
        _same(cuda.download(de, (R,), np.float32, s), we)
        assert np.array_equal(cuda.download(di, (R, top), np.int32, s), wi)
        _same(cuda.download(dp, (R, top), np.float32, s), wt)
    g.close()
    cuda.destroy_stream(s)
    for p in (dx, dt, dl, de, di, dp, ws):
        cuda.free_device(p)


@pytest.mark.parametrize("rows,vocab,top", [(2100, 4200, 2), (1024, 8300, 1), (1025, 9000, 64), (64, 33000, 64)])
def test_many_rows(cuda, K, rows, vocab, top):
    """Rows in parts and whole, around the number that have counters."""
    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    _check(cuda, K, x, rng.integers(0, vocab, rows), top)


@pytest.mark.parametrize("top", [1, 20, 64])
def test_best_logits_in_one_place(cuda, K, top):
    """The largest all in one lane's logits, in one block, and in a row's last part."""
    rng = np.random.default_rng(top)
    x = rng.standard_normal((4, 70001)).astype(np.float32)
    x[0, 8192:8192 + 4 * 64 * 16:256] += 50   # one lane's, 16 blocks
    x[1, 4096:4096 + 100] += np.arange(100, dtype=np.float32)
    x[2, -80:] = 30
    x[3, :] = np.float32(-2.5)                # all equal
    _check(cuda, K, x, [8192, 4196, 70000, 0], top)


def test_graphs_of_one_stream_replayed_at_once(cuda, K):
    """Two graphs that the program captured itself from one stream, replayed on two
    others beside eager calls on that stream."""
    rng = np.random.default_rng(8)
    R, V, top = 3, 90001, 12
    xs = [rng.standard_normal((R, V)).astype(np.float32) for _ in range(3)]
    mem = []
    for x in xs:
        mem.append([cuda.upload(x), cuda.upload(np.arange(R, dtype=np.int32))] +
                   [cuda.alloc_device(n) for n in (R * 4, R * 4, R * top * 4, R * top * 4, K.logprobs_ws_bytes(R, V, top))])
    cuda.sync()

    def launch(i, stream):
        dx, dt, dl, de, di, dp, ws = mem[i]
        for _ in range(3):
            K.logprobs(dx, V, R, V, dt, dl, de, top, di, dp, ws, stream, ws_bytes=ws.nbytes)

    s, s0, s1 = (cuda.stream() for _ in range(3))
    g0, g1 = (HipGraph(s, lambda st, i=i: launch(i, st)) for i in range(2))
    for _ in range(4):
        for m in mem:
            cuda.htod_async(m[4], np.full((R, top), 7, np.int32), s)
        cuda.sync()
        for _ in range(5):
            g0.launch(s0)
            g1.launch(s1)
            launch(2, s)
        for st in (s, s0, s1):
            cuda.sync_stream(st)
        for x, m in zip(xs, mem):
            wl, we, wi, wt = logprobs(x, np.arange(R), top)
            _same(cuda.download(m[2], (R,), np.float32), wl)
            _same(cuda.download(m[3], (R,), np.float32), we)
            assert np.array_equal(cuda.download(m[4], (R, top), np.int32), wi)
            _same(cuda.download(m[5], (R, top), np.float32), wt)
    g0.close()
    g1.close()
    for st in (s, s0, s1):
        cuda.destroy_stream(st)
    for m in mem:
        for p in m:
            cuda.free_device(p)
