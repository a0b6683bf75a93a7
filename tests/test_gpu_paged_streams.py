"""lp_attn_paged and lp_logprobs beside the calls that need a stream's arrival
counters, on many streams."""
import threading

import numpy as np
import pytest

import llmpager_amd as lp
from _paged import Batch, logprobs
from test_gpu_logprobs import _run, _same
from test_gpu_paged import _attn, _close, _queries

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(cuda):
    return lp.Kernels(cuda)


def test_counters_are_not_taken_from_other_calls(cuda, K):
    """Paged attention and log probabilities on 70 streams; then calls that are refused
    on a stream without counters run on 20 more, and a capture begins."""
    rng = np.random.default_rng(0)
    B = Batch(cuda, [1, 1], [2500, 300], 8, 2, 128, 16, lp.KV_Q4, seed=1)
    q = _queries(B)
    B.device()
    x = rng.standard_normal((2, 40000)).astype(np.float32)
    wl, _, wi, _ = logprobs(x, np.array([3, 4]), 5)
    rows, cols = 8, 64
    w, v, h = (rng.standard_normal(n).astype(np.float32) for n in ((rows, cols), cols, rows))
    w = w.view(np.uint32) & 0xffff0000  # bf16 values
    d = [cuda.upload(a) for a in ((w >> 16).astype(np.uint16), v, np.ones(rows, np.float32))]
    want = h + w.view(np.float32) @ v
    streams = [cuda.stream() for _ in range(70)]
    more = [cuda.stream() for _ in range(20)]
    try:
        outs = [_attn(K, B, q, stream=s) for s in streams]
        for o in outs[1:]:
            assert np.array_equal(o, outs[0])
        for s in streams:
            logp, _, ids, _ = _run(cuda, K, x, [3, 4], 5, stream=s)
            _same(logp, wl)
            assert np.array_equal(ids, wi)
        for s in more:
            dh, dn = cuda.upload(h), cuda.alloc_device(256)
            cuda.sync()
            K.gemv_add_rmsnorm(d[0], d[1], rows, cols, dh, d[2], 1e-6, dn, s)
            got = cuda.download(dh, (rows,), np.float32, s)
            ok = np.allclose(got, want, rtol=1e-4, atol=1e-4)
            assert ok
            for p in (dh, dn):
                cuda.free_device(p)
        cuda.capture_begin(more[0])
        cuda.capture_end(more[0]).close()
    finally:
        for s in streams + more:
            cuda.destroy_stream(s)
        for p in d:
            cuda.free_device(p)
        B.free()


def test_streams_and_graphs_give_their_counters_back(cuda, K):
    """More streams, and more graphs, one behind the other than there are sets."""
    B = Batch(cuda, [1, 1], [2500, 300], 8, 2, 128, 16, lp.KV_Q4, seed=2)
    q = _queries(B)
    B.device()
    W = 8 * 128
    dq, do = B.up(q), B.alloc(2 * W * 4)
    ws = B.alloc(K.attn_paged_ws_bytes(B.cache, 8, 2, 2, 1, 2501))
    want = B.attention(q.reshape(2, 8, 128), 1.0 / np.sqrt(128.0))

    def launch(s):
        K.attn_paged(B.cache, dq, W, do, W, 8, B.dstarts, B.dlens, 2, 2, 1, 2501, 1.0 / np.sqrt(128.0), ws, s,
                     ws_bytes=ws.nbytes)

    for i in range(70):
        s = cuda.stream()
        if i % 2:
            cuda.capture_begin(s)
            launch(s)
            g = cuda.capture_end(s)
            for _ in range(3):
                g.launch(s)
                launch(s)
            cuda.sync_stream(s)
            g.close()
        else:
            launch(s)
        _close(cuda.download(do, (2, 8, 128), np.float32, s), want)
        cuda.destroy_stream(s)
    B.free()


PER_THREAD = 2  # hipStreamPerThread: one handle, a stream for each host thread


def test_threads_on_their_own_streams_by_one_handle(cuda, K):
    """Four host threads, each with its workspaces, on the handle that names a stream
    of each of them."""
    Bs, jobs = [], []
    for i in range(4):
        B = Batch(cuda, [1, 1], [2500 + 300 * i, 300], 8, 2, 128, 16, lp.KV_Q4, seed=10 + i)
        q = _queries(B)
        B.device()
        x = B.rng.standard_normal((2, 50021)).astype(np.float32)
        Bs.append(B)
        jobs.append((B.up(q), B.alloc(2 * 4096), B.alloc(K.attn_paged_ws_bytes(B.cache, 8, 2, 2, 1, max(B.lens))),
                     B.up(x), B.up(np.array([3, 4], np.int32)), B.alloc(256), B.alloc(256), B.alloc(256),
                     B.alloc(K.logprobs_ws_bytes(2, 50021, 5)),
                     B.attention(q.reshape(2, 8, 128), 1.0 / np.sqrt(128.0)), logprobs(x, np.array([3, 4]), 5)))
    cuda.sync()
    start, failed = threading.Barrier(4), []

    def run(B, job):
        dq, do, ws, dx, dt, dl, di, dp, ws2, att, (wl, _, wi, wp) = job
        try:
            cuda.bind_thread()
            start.wait()
            for _ in range(5):
                for _ in range(20):
                    K.attn_paged(B.cache, dq, 1024, do, 1024, 8, B.dstarts, B.dlens, 2, 2, 1, max(B.lens),
                                 1.0 / np.sqrt(128.0), ws, PER_THREAD, ws_bytes=ws.nbytes)
                    K.logprobs(dx, 50021, 2, 50021, dt, dl, 0, 5, di, dp, ws2, PER_THREAD, ws_bytes=ws2.nbytes)
                _close(cuda.download(do, (2, 8, 128), np.float32, PER_THREAD), att)
                _same(cuda.download(dl, (2,), np.float32, PER_THREAD), wl)
                assert np.array_equal(cuda.download(di, (2, 5), np.int32, PER_THREAD), wi)
                _same(cuda.download(dp, (2, 5), np.float32, PER_THREAD), wp)
        except BaseException as e:  # to the test's own thread
            failed.append(e)

    threads = [threading.Thread(target=run, args=a) for a in zip(Bs, jobs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for B in Bs:
        B.free()
    if failed:
        raise failed[0]
