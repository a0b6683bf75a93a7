"""Trees of drafted tokens over the paged KV cache on the GPU: lp_tree_layout,
lp_kv_append_tree, lp_attn_tree and lp_kv_keep against the same formulas in 64 bits
(tests/_tree.py).

Tolerances: layouts and moved rows are equal.  Appended rows: 64-bit values rounded
once (f32: 2^-24 of a pair's length, fp16: 2^-11; 4-bit codes are equal).  Attention
has the products and sums of lp_attn_paged: an image of a query leaves 2^-22 of it,
a score is off by that of its size, up to 16 here, 2^-18 = 3.8e-6, and its probability by as
much; the fp32 sums add below 2^-24 x 64 = 3.8e-6: 1e-5 of the largest |v| a row sees."""
import numpy as np
import pytest

import llmpager_amd as lp
from _paged import HipGraph
from _tree import Trees, ancestors, random_tree, words_of

pytestmark = pytest.mark.gpu

EPS = 1e-6
ATTN_TOL = 1e-5


@pytest.fixture(scope="module")
def K(cuda):
    return lp.Kernels(cuda)


def _f32(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


class Mem:
    """Device buffers of one test."""

    def __init__(self, cuda):
        self.cuda, self.ptrs = cuda, []

    def up(self, a):
        p = self.cuda.upload(np.ascontiguousarray(a))
        self.ptrs.append(p)
        return p

    def alloc(self, n):
        p = self.cuda.alloc_device(max(n, 256))
        self.ptrs.append(p)
        return p

    def free(self):
        self.cuda.sync()
        for p in self.ptrs:
            self.cuda.free_device(p)


# ---- layout -----------------------------------------------------------------------


def _layout(cuda, K, trees, max_q=None, pad=0, front=0):
    m = Mem(cuda)
    rng = np.random.default_rng(len(trees))
    T = front + sum(map(len, trees)) + pad
    parents = np.concatenate([np.full(front, 0)] + [np.asarray(t, np.int64) for t in trees] + [np.zeros(pad)]).astype(np.int32)
    starts = front + np.concatenate(([0], np.cumsum([len(t) for t in trees]))).astype(np.int32)
    q = max_q or max([len(t) for t in trees] + [1])
    W = (q + 63) // 64
    d0, m0 = rng.integers(0, 99, T).astype(np.int32), rng.integers(0, 1 << 62, (T, W)).astype(np.uint64)
    dd, dm = m.up(d0), m.up(m0)
    K.tree_layout(m.up(parents), m.up(starts), len(trees), T, q, dd, dm)
    for b, t in enumerate(trees):
        deep, masks = ancestors(t[:q])
        at = starts[b]
        d0[at:at + len(deep)] = deep
        m0[at:at + len(deep)] = words_of(masks, W)
    assert np.array_equal(cuda.download(dd, d0.shape, np.int32), d0)
    assert np.array_equal(cuda.download(dm, m0.shape, np.uint64), m0)
    m.free()


def test_layout_small(cuda, K):
    _layout(cuda, K, [[-1]])
    _layout(cuda, K, [[-1, 0, 0, 1, 3, 4, 4, 2]], pad=3, front=2)
    _layout(cuda, K, [[], [-1, 0], [], [-1], []], max_q=7)


def test_layout_parents_that_are_none(cuda, K):
    """A node's own number, a higher one, a negative one, one out of range: a root."""
    _layout(cuda, K, [[0, 0, 2, 9, 3, 4, 2 ** 31 - 1, -2 ** 31, 5, 5]])


@pytest.mark.parametrize("n", [63, 64, 65, 128, 200, 256, 257, 1000, 1024])
def test_layout_sizes(cuda, K, n):
    rng = np.random.default_rng(n)
    _layout(cuda, K, [random_tree(rng, n), [-1] + list(range(n - 1)), [-1] + [0] * (n // 2), [-1]], pad=1)


def test_layout_tokens_past_max_q(cuda, K):
    rng = np.random.default_rng(3)
    _layout(cuda, K, [random_tree(rng, 90), random_tree(rng, 5), random_tree(rng, 64)], max_q=64)


def test_layout_many_sequences(cuda, K):
    rng = np.random.default_rng(4)
    _layout(cuda, K, [random_tree(rng, int(n)) for n in rng.integers(0, 12, 1500)], max_q=70)


# ---- append -----------------------------------------------------------------------


def _append(K, B, x, qw, kw, mscale=1.0, stream=None):
    W, D = x.shape[1], B.dim
    dx = B.up(x)
    dq = B.up(np.full((B.tokens, B.heads * D), 7, np.float32))
    dko, dvo = (B.up(np.full((B.tokens, B.kv * D), 7, np.float32)) for _ in range(2))
    K.kv_append_tree(B.cache, dx, W, dx + B.heads * D * 4, W, dx + (B.heads + B.kv) * D * 4, W,
                     0 if qw is None else B.up(qw), 0 if kw is None else B.up(kw), EPS, B.up(B.freq), mscale, dq, B.heads * D,
                     dko, dvo, B.heads, B.dstarts, B.dlens, B.up(B.depths), B.batch, B.tokens, stream)
    return dq, dko, dvo


def _check_append(K, B, norms=True, mscale=1.0):
    x = _f32(B.rng, B.tokens, (B.heads + 2 * B.kv) * B.dim)
    a, b, D, n = B.heads * B.dim, (B.heads + B.kv) * B.dim, B.dim, B.live
    qw, kw = (_f32(B.rng, D) + 1, _f32(B.rng, D) + 1) if norms else (None, None)
    B.device()
    dq, dko, dvo = _append(K, B, x, qw, kw, mscale)
    wq, wk, wv, pools = B.append_tree(x[:, :a], x[:, a:b], x[:, b:], qw, kw, EPS, mscale)
    got = B.cuda.download(dq, (B.tokens, B.heads, D), np.float32)
    tol = 2.0 ** -23 * np.hypot(wq[..., :D // 2], wq[..., D // 2:])
    assert (np.abs(got[:n] - wq[:n]) <= np.concatenate((tol, tol), -1)[:n]).all()
    assert (got[n:] == 7).all()
    for d, w in ((dko, wk), (dvo, wv)):
        g = B.cuda.download(d, (B.tokens, B.kv, D), np.float32)
        assert (g[n:] == 7).all()
        if B.fmt == lp.KV_Q4:
            assert np.array_equal(g[:n], w[:n].astype(np.float32))
        else:
            assert np.allclose(g[:n], w[:n], rtol=2.0 ** -10, atol=2.0 ** -24)
    for d, w in zip((B.dk, B.dv), pools):
        g = B.cuda.download(d, w.shape, np.uint8)
        if B.fmt == lp.KV_Q4:
            assert np.array_equal(g, w)
        else:
            steps = g.view(np.int16).astype(np.int32) - w.view(np.int16)
            assert np.abs(steps).max() <= 1 and (steps != 0).mean() < 1e-3
    B.free()


@pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])
@pytest.mark.parametrize("sizes,past,heads,kv,dim,page,pad", [
    ([1], [0], 1, 1, 64, 16, 0),
    ([26], [1500], 32, 4, 128, 64, 0),
    ([7, 1, 40], [15, 16, 250], 5, 1, 128, 16, 2),
    ([0, 9, 0, 70], [8, 3, 0, 60], 4, 4, 64, 256, 0),
    ([12], [131000], 3, 3, 64, 128, 0),
])
def test_append(cuda, K, fmt, sizes, past, heads, kv, dim, page, pad):
    rng = np.random.default_rng(sum(sizes))
    _check_append(K, Trees(cuda, [random_tree(rng, n) if n else [] for n in sizes], past, heads, kv, dim, page, fmt, seed=dim, pad=pad))


@pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])
def test_append_depths_of_the_callers_own(cuda, K, fmt):
    """Any whole numbers, negative and large ones; scaled, without norms."""
    B = Trees(cuda, [[-1] + [0] * 8, [-1, 0]], [40, 3], 4, 2, 64, 16, fmt, seed=1)
    B.depths = np.array([0, 1, -1, -40, 1000, 99999, 7, 7, 0, -3, 2], np.int32)
    _check_append(K, B, norms=False, mscale=1.25)


def test_append_of_a_chain_is_the_paged_one(cuda, K):
    """The same bits, in queries and pages, as lp_kv_append_paged where nodes follow one another."""
    for fmt in (lp.KV_F16, lp.KV_Q4):
        B = Trees(cuda, [[-1] + list(range(30)), [-1, 0]], [77, 5], 8, 2, 128, 32, fmt, seed=2)
        x = _f32(B.rng, B.tokens, 12 * 128)
        B.device()
        dq, _, _ = _append(K, B, x, None, None)
        got = [cuda.download(dq, (B.tokens, 1024), np.float32)] + [cuda.download(p, B.pools[0].shape, np.uint8) for p in (B.dk, B.dv)]
        dx = B.up(x)
        C = Trees(cuda, B.trees, B.past, 8, 2, 128, 32, fmt, seed=2).device()
        do = C.alloc(B.tokens * 4096)
        K.kv_append_paged(C.cache, dx, 1536, dx + 4096, 1536, dx + 5120, 1536, 0, 0, EPS, C.up(C.freq), 1.0, do, 1024, 0, 0, 8,
                          C.dstarts, C.dlens, 2, C.tokens)
        want = [cuda.download(do, (B.tokens, 1024), np.float32)] + [cuda.download(p, B.pools[0].shape, np.uint8) for p in (C.dk, C.dv)]
        for g, w in zip(got, want):
            assert np.array_equal(g, w)
        B.free(), C.free()


# ---- attention --------------------------------------------------------------------


def _attn(K, B, q, max_seq=None, cols=0):
    W = B.heads * B.dim
    dq, do = B.up(q), B.up(np.full((B.tokens, W + cols), 7, np.float32))
    ms = max_seq or max(B.lens + [1])
    n = K.attn_tree_ws_bytes(B.cache, B.heads, B.batch, B.tokens, B.max_q, ms)
    ws = B.alloc(n)
    K.attn_tree(B.cache, dq, q.shape[1], do, W + cols, B.heads, B.dstarts, B.dlens, B.up(B.masks()), B.batch, B.tokens, B.max_q,
                ms, 1.0 / np.sqrt(B.dim), ws, ws_bytes=ws.nbytes)
    return B.cuda.download(do, (B.tokens, W + cols), np.float32)


def _close(got, want, tol=ATTN_TOL):
    fine = np.abs(want[np.isfinite(want)])
    size = max(fine.max() if fine.size else 0.0, 1.0)
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(got - want) <= tol * size) & ~(np.isnan(got) & np.isnan(want)) & ~(got == want)
    assert not bad.any(), (np.argwhere(bad)[:5], bad.sum())


def _check_attn(K, B, max_seq=None, cols=0, std=1.0):
    W = B.heads * B.dim
    q = (_f32(B.rng, B.tokens, W + cols) * std).astype(np.float32)
    B.device()
    got = _attn(K, B, q, max_seq, cols=cols)
    want = B.attention_tree(q[:, :W].reshape(B.tokens, B.heads, B.dim), 1.0 / np.sqrt(B.dim), max_seq).reshape(B.tokens, W)
    on = np.zeros(B.tokens, bool)
    for b in range(B.batch):
        on[B.starts[b]:B.starts[b] + min(B.new[b], B.max_q)] = True
    _close(got[on, :W], want[on])
    assert (got[~on] == 7).all() and (got[:, W:] == 7).all()
    B.free()


# A bound on the lengths that is far above them, in a table that is as wide: more than some
# dozens of query rows are then attention's of many rows, in spans of the context.
WIDE = dict(cols=4000)


def _bound(wide):
    return 4000 * 16 if wide else None


FORMS = [(f, d) for f in (lp.KV_F16, lp.KV_Q4) for d in (64, 128)]


@pytest.mark.parametrize("fmt,dim", FORMS)
@pytest.mark.parametrize("sizes,past,heads,kv,page", [
    ([1], [0], 1, 1, 16),                            # a root and nothing else
    ([1], [700], 8, 1, 16),                          # one token: as a step without drafts
    ([2, 3], [0, 31], 4, 4, 16),                     # few rows, nothing before them
    ([7], [1500], 16, 8, 64),                        # a token's two heads a KV head
    ([4], [2999], 16, 2, 32),                        # 32 rows, a long context in parts
    ([5, 2, 3], [500, 63, 64], 3, 1, 16),            # odd heads to a KV head
    ([26], [1500], 32, 4, 64),                       # 208 rows: two tiles
    ([64, 20, 1], [129, 1, 300], 8, 1, 128),
    ([65], [63], 2, 1, 16),                          # a second mask word, context a row short of a chunk
    ([200], [190], 2, 1, 64),
    ([0, 12, 0], [40, 20, 0], 8, 2, 256),            # sequences without a token
])
def test_attention(cuda, K, fmt, dim, sizes, past, heads, kv, page):
    rng = np.random.default_rng(sum(sizes) + dim)
    trees = [random_tree(rng, n) if n else [] for n in sizes]
    _check_attn(K, Trees(cuda, trees, past, heads, kv, dim, page, fmt, seed=sum(sizes), pad=2))


@pytest.mark.parametrize("fmt,dim", FORMS)
@pytest.mark.parametrize("heads,kv,wide", [(2, 1, False), (16, 1, False), (64, 4, False), (16, 1, True)])
def test_attention_where_the_context_ends(cuda, K, fmt, dim, heads, kv, wide):
    """Contexts that end at every place of a chunk's last rows, of parts and of pages."""
    rng = np.random.default_rng(heads)
    past = [0, 1, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511]
    _check_attn(K, Trees(cuda, [random_tree(rng, int(rng.integers(1, 16))) for _ in past], past, heads, kv, dim, 16, fmt, seed=3,
                         **(WIDE if wide else {})), _bound(wide))


@pytest.mark.parametrize("fmt,dim", FORMS)
@pytest.mark.parametrize("n,heads", [(11, 2), (30, 1), (30, 8), (130, 2)])
@pytest.mark.parametrize("past", [0, 37])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_any_masks(cuda, K, fmt, dim, n, heads, past, wide):
    """Masks that are no ancestors: bits at random, none, all, behind the tokens and
    past max_q; a row without any and no context is zeros."""
    rng = np.random.default_rng(n + past)
    B = Trees(cuda, [[-1] * n, [-1] * 3], [past, 5], heads, 1, dim, 16, fmt, seed=n, max_q=n + 3, **(WIDE if wide else {}))
    B.bits = [int.from_bytes(rng.bytes(24), "little") for _ in range(B.tokens)]
    B.bits[0], B.bits[1], B.bits[2], B.bits[n - 1] = 0, (1 << 192) - 1, 1 << (n - 1), 0
    want = [m & ((1 << n) - 1) for m in B.bits[:n]] + [m & 7 for m in B.bits[n:]]
    masks = words_of([m & ((1 << (64 * B.words)) - 1) for m in B.bits], B.words)
    B.bits = want
    B.masks = lambda: masks
    _check_attn(K, B, _bound(wide))


@pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])
@pytest.mark.parametrize("max_q", [3, 16, 70])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_tokens_past_max_q(cuda, K, fmt, max_q, wide):
    """They are left as they were, and their rows are seen by none."""
    rng = np.random.default_rng(9)
    B = Trees(cuda, [[-1] * 90, random_tree(rng, 5)], [100, 40], 12, 2, 64, 16, fmt, seed=4, max_q=max_q, **(WIDE if wide else {}))
    full = [int.from_bytes(rng.bytes(16), "little") for _ in range(B.tokens)]
    masks = words_of([m & ((1 << (64 * B.words)) - 1) for m in full], B.words)
    B.bits = [m & ((1 << 90) - 1) for m in full[:90]] + [m & 31 for m in full[90:]]
    B.masks = lambda: masks
    _check_attn(K, B, _bound(wide))


@pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])
@pytest.mark.parametrize("n,max_seq", [(3, 40), (3, 7), (3, 1), (40, 50), (40, 20), (200, 128)])
def test_attention_lengths_past_max_seq(cuda, K, fmt, n, max_seq):
    """A larger length is taken as max_seq; where that is less than the tokens, the first
    ones' rows are not there."""
    rng = np.random.default_rng(n)
    _check_attn(K, Trees(cuda, [random_tree(rng, n), [-1, 0]], [90, 1], 4, 2, 64, 16, fmt, seed=n), max_seq=max_seq)


@pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])
@pytest.mark.parametrize("n,heads", [(5, 2), (60, 8)])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_pages_that_are_not_there(cuda, K, fmt, n, heads, wide):
    rng = np.random.default_rng(n)
    B = Trees(cuda, [random_tree(rng, n), random_tree(rng, n)], [120, 33], heads, 1, 128, 16, fmt, seed=5, **(WIDE if wide else {}))
    B.table[0, 1], B.table[0, 7], B.table[1, 2], B.table[1, 0] = -1, B.pages, 2 ** 31 - 1, -2 ** 31
    _check_attn(K, B, _bound(wide))


@pytest.mark.parametrize("n,heads,dim", [(6, 2, 64), (6, 2, 128), (14, 2, 128), (70, 2, 64), (70, 4, 128), (70, 8, 64)])
@pytest.mark.parametrize("kind", ["hidden", "seen"])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_rows_that_are_no_numbers(cuda, K, n, heads, dim, kind, wide):
    """fp16 rows of NaN and infinities: what does not see them is as without them, and
    what does has what the formula gives."""
    rng = np.random.default_rng(n)
    B = Trees(cuda, [random_tree(rng, n), [-1, 0, 0]], [70, 30], heads, 1, dim, 16, lp.KV_F16, seed=6, **(WIDE if wide else {}))
    bad = n - 2
    if kind == "hidden":
        for t in range(n):
            B.bits[t] &= ~(1 << bad)
    v = rng.standard_normal((1, dim))
    v[0, 3], v[0, 5], v[0, 9] = np.inf, -np.inf, np.nan
    B.put(70 + bad, k=np.full((1, dim), np.nan) if kind == "hidden" else None, v=v)
    _check_attn(K, B, _bound(wide))


@pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])
@pytest.mark.parametrize("n", [3, 40])
def test_attention_strided(cuda, K, fmt, n):
    rng = np.random.default_rng(n)
    _check_attn(K, Trees(cuda, [random_tree(rng, n), [-1, 0]], [50, 9], 4, 2, 64, 32, fmt, seed=7, pad=3), cols=12)


@pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])
def test_attention_many_sequences(cuda, K, fmt):
    rng = np.random.default_rng(1)
    _check_attn(K, Trees(cuda, [random_tree(rng, int(n)) if n else [] for n in rng.integers(0, 9, 300)],
                         [int(p) for p in rng.integers(0, 60, 300)], 4, 4, 64, 16, fmt, seed=8))


@pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])
def test_attention_many_sequences_in_blocks(cuda, K, fmt):
    """More sequences than lanes, of several blocks of query rows each, whose parts are joined."""
    rng = np.random.default_rng(2)
    n = 150
    _check_attn(K, Trees(cuda, [random_tree(rng, int(k)) if k else [] for k in rng.integers(0, 14, n)],
                         [int(p) for p in rng.integers(0, 900, n)], 4, 1, 64, 16, fmt, seed=9))


@pytest.mark.parametrize("fmt,dim", FORMS)
@pytest.mark.parametrize("n", [3, 64, 80])
def test_attention_of_many_rows_shared_out(cuda, K, fmt, dim, n):
    """128 query rows and more a workgroup, whose parts go by the lengths in memory: some
    sequences have none, some one, some several; in lanes, and past as many sequences."""
    rng = np.random.default_rng(dim)
    long, bound = (1000, 4000) if n > 3 else (6000, 96000)
    past = [0, long] + [int(p) for p in rng.integers(0, long // 2, n - 2)]
    trees = [random_tree(rng, 14), random_tree(rng, 9)] + [random_tree(rng, int(k)) if k else [] for k in rng.integers(0, 14, n - 2)]
    _check_attn(K, Trees(cuda, trees, past, 16, 1, dim, 16, fmt, seed=n, cols=bound // 16), bound)


@pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])
@pytest.mark.parametrize("n,kv,group", [(40, 8, 16), (64, 9, 4), (66, 8, 4), (5, 5, 16)])
def test_attention_a_workgroup_a_block(cuda, K, fmt, n, kv, group):
    """Blocks of 128 query rows that no other workgroup helps with: by their lengths, in one
    round and in several, and of more sequences than lanes."""
    rng = np.random.default_rng(n)
    nodes = [9, 0, 1] + [int(k) for k in rng.integers(0, 10, n - 3)]
    if n == 5:
        nodes = [150, 0, 90, 150, 17]
    past = [290, 40, 2] + [int(p) for p in rng.integers(0, 290, n - 3)]
    _check_attn(K, Trees(cuda, [random_tree(rng, k) if k else [] for k in nodes], past, kv * group, kv, 64, 16, fmt, seed=n))


@pytest.mark.parametrize("fmt,dim", FORMS)
@pytest.mark.parametrize("n,heads", [(3, 8), (9, 2), (40, 8), (130, 8)])
def test_attention_long_contexts(cuda, K, fmt, dim, n, heads):
    """Contexts that many workgroups share, ragged ones, and joins of their parts."""
    rng = np.random.default_rng(n)
    _check_attn(K, Trees(cuda, [random_tree(rng, n), random_tree(rng, max(1, n // 2)), [-1]], [8000, 777, 4100], heads, 1, dim, 64, fmt, seed=9))


def test_attention_of_a_chain_is_the_paged_one(cuda, K):
    """Chains see what causal attention shows them: the same sums, if not always cut into
    parts in the same places (a few roundings of 2^-22)."""
    for fmt in (lp.KV_F16, lp.KV_Q4):
        for n, heads, tol in ((3, 4, 0.0), (12, 2, 2e-6), (50, 8, 2e-6), (300, 8, 2e-6)):
            B = Trees(cuda, [[-1] + list(range(n - 1)), [-1, 0]], [333, 64], heads, 1, 128, 32, fmt, seed=n)
            q = _f32(B.rng, B.tokens, heads * 128)
            B.device()
            got = _attn(K, B, q)
            do, dq = B.alloc(got.nbytes), B.up(q)
            ws = B.alloc(K.attn_paged_ws_bytes(B.cache, heads, 2, B.tokens, B.max_q, max(B.lens)))
            K.attn_paged(B.cache, dq, heads * 128, do, heads * 128, heads, B.dstarts, B.dlens, 2, B.tokens, B.max_q, max(B.lens),
                         1.0 / np.sqrt(128), ws, ws_bytes=ws.nbytes)
            _close(got, cuda.download(do, got.shape, np.float32), tol)
            B.free()


# ---- keep -------------------------------------------------------------------------


def _random_path(rng, n, most):
    k = int(rng.integers(1, min(n, most) + 1))
    return [0] + sorted(rng.choice(np.arange(1, n), k - 1, replace=False).tolist()) if n > 1 else [0]


def _check_keep(cuda, K, Bs, paths, max_depth, kept=None, lens_out=True, want_paths=None):
    """Layers Bs (batches alike but for their pools' contents)."""
    B = Bs[0]
    for L in Bs:
        L.table = B.table
        L.device()
        L.cache.table = B.dtable
    table = np.full((B.batch, max_depth + 1), -1, np.int32)
    for b, p in enumerate(paths):
        table[b, :len(p)] = p[:max_depth + 1]
    kept = np.array([len(p) for p in paths] if kept is None else kept, np.int32)
    do = B.up(np.full(B.batch, 7, np.int32))
    K.kv_keep([L.cache for L in Bs], B.up(table), max_depth, B.up(kept), B.dstarts, B.dlens, do if lens_out else 0, B.batch)
    take = [max(0, min(int(kept[b]), max_depth + 1, B.new[b])) for b in range(B.batch)]
    paths = [list(table[b, :take[b]]) for b in range(B.batch)] if want_paths is None else want_paths
    for L in Bs:
        want = L.keep(L.pools, paths)
        for d, w in zip((L.dk, L.dv), want):
            assert np.array_equal(cuda.download(d, w.shape, np.uint8), w)
    lens = [B.past[b] + take[b] for b in range(B.batch)] if lens_out else [7] * B.batch
    assert np.array_equal(cuda.download(do, (B.batch,), np.int32), lens)
    for L in Bs:
        L.free()


@pytest.mark.parametrize("fmt,dim", FORMS)
@pytest.mark.parametrize("sizes,past,kv,page,layers,depth", [
    ([1], [0], 1, 16, 1, 0),
    ([26], [300], 4, 64, 3, 6),
    ([9, 40, 1, 0, 17], [15, 30, 4, 9, 0], 3, 16, 2, 12),   # over page borders; a sequence without tokens
    ([200], [5], 1, 32, 1, 150),                            # more than 64 nodes stay
    ([30, 12], [2, 50], 24, 16, 1, 9),                      # more heads than a wave's share
    ([12, 7], [20, 3], 2, 16, 70, 5),                       # more layers than a launch takes
])
def test_keep(cuda, K, fmt, dim, sizes, past, kv, page, layers, depth):
    rng = np.random.default_rng(sum(sizes))
    trees = [random_tree(rng, n) if n else [] for n in sizes]
    Bs = [Trees(cuda, trees, past, kv, kv, dim, page, fmt, seed=l) for l in range(layers)]
    _check_keep(cuda, K, Bs, [_random_path(rng, n, depth + 1) if n else [] for n in sizes], depth)


@pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])
def test_keep_rows_that_are_read_and_written(cuda, K, fmt):
    """Paths where one node's new row is another's old one, all the way along."""
    n = 40
    B = Trees(cuda, [[-1] * n] * 3, [9, 16, 30], 2, 2, 64, 16, fmt, seed=1)
    _check_keep(cuda, K, [B], [[0] + list(range(2, n)), list(range(n)), [0] + list(range(3, n, 2))], n - 1)


@pytest.mark.parametrize("fmt", [lp.KV_F16, lp.KV_Q4])
def test_keep_what_is_not_there(cuda, K, fmt):
    """Entries that are no nodes, counts past the tokens and below none, absent pages."""
    B = Trees(cuda, [[-1] * 20] * 5, [10, 14, 3, 50, 7], 2, 2, 128, 16, fmt, seed=2)
    B.table[1, 0] = -1
    B.table[3, 4] = B.pages + 5
    _check_keep(cuda, K, [B], [[0, 5, 20, 2 ** 31 - 1], [0, 3, 9], [0, 2, 4], [0, 1, 12, 15], [-1, -2 ** 31, 4]], 5,
                kept=[4, 3, -2, 4, 1000], want_paths=[[0, 5], [0, 3, 9], [], [0, 1, 12, 15], [0, 1, 4]])


def test_keep_without_lengths(cuda, K):
    B = Trees(cuda, [[-1] * 6], [10], 1, 1, 64, 16, lp.KV_F16, seed=3)
    _check_keep(cuda, K, [B], [[0, 3, 5]], 3, lens_out=False)


# ---- streams and graphs -------------------------------------------------------------


@pytest.mark.parametrize("capture", ["library", "runtime"])
def test_captured_steps(cuda, K, capture):
    """Layout, append, attention and keep in a graph, replayed with other trees and
    lengths between the program's own calls on that stream."""
    rng = np.random.default_rng(7)
    page, heads, kv, dim, Q, T = 16, 4, 2, 64, 24, 40
    base = Trees(cuda, [random_tree(rng, 24), random_tree(rng, 16)], [900, 400], heads, kv, dim, page, lp.KV_F16, seed=1, max_q=Q).device()
    W = (heads + 2 * kv) * dim
    dx, dpar, dstarts, dlens = base.alloc(T * W * 4), base.alloc(T * 4), base.alloc(12), base.alloc(8)
    ddep, dmask, dq, do = base.alloc(T * 4), base.alloc(T * 8), base.alloc(T * heads * dim * 4), base.alloc(T * heads * dim * 4)
    dpath, dkept, dlo, dfreq = base.alloc(2 * 6 * 4), base.alloc(8), base.alloc(8), base.up(base.freq)
    ws = base.alloc(K.attn_tree_ws_bytes(base.cache, heads, 2, T, Q, 940))
    s = cuda.stream()

    def step(stream):
        K.tree_layout(dpar, dstarts, 2, T, Q, ddep, dmask, stream)
        K.kv_append_tree(base.cache, dx, W, dx + heads * dim * 4, W, dx + (heads + kv) * dim * 4, W, 0, 0, EPS, dfreq, 1.0, dq,
                         heads * dim, 0, 0, heads, dstarts, dlens, ddep, 2, T, stream)
        K.attn_tree(base.cache, dq, heads * dim, do, heads * dim, heads, dstarts, dlens, dmask, 2, T, Q, 940,
                    1.0 / np.sqrt(dim), ws, stream, ws_bytes=ws.nbytes)
        K.kv_keep([base.cache], dpath, 5, dkept, dstarts, dlens, dlo, 2, stream)

    if capture == "library":
        cuda.capture_begin(s)
        step(s)
        g = cuda.capture_end(s)
    else:
        g = HipGraph(s, step)
    pools = base.pools
    for i in range(5):
        sizes = [int(rng.integers(1, 25)), int(rng.integers(1, 17))]
        past = [int(rng.integers(0, 900)), int(rng.integers(0, 400))]
        B = Trees(cuda, [random_tree(rng, n) for n in sizes], past, heads, kv, dim, page, lp.KV_F16, seed=1, max_q=Q, cols=base.cols)
        B.table, B.pools, B.pages = base.table, pools, base.pages
        x = _f32(rng, T, W)
        paths = [_random_path(rng, n, 6) for n in sizes]
        table = np.array([p + [-1] * (6 - len(p)) for p in paths], np.int32)
        parents = np.concatenate((B.parents, np.zeros(T - B.tokens, np.int32)))
        for d, v in ((dx, x), (dpar, parents), (dstarts, B.starts), (dlens, np.asarray(B.lens, np.int32)), (dpath, table),
                     (dkept, np.array([len(p) for p in paths], np.int32))):
            cuda.htod_async(d, v)
        cuda.sync()
        if i != 2:
            g.launch(s)
        else:
            step(s)  # the program's own, between replays
        n = B.tokens
        a, b = heads * dim, (heads + kv) * dim
        wq, _, _, after = B.append_tree(x[:n, :a], x[:n, a:b], x[:n, b:], None, None, EPS)
        got = cuda.download(do, (T, heads * dim), np.float32, s)
        B.pools = after
        want = B.attention_tree(wq, 1.0 / np.sqrt(dim))
        _close(got[:n].reshape(n, heads, dim), want, 1e-3)  # a step of fp16 rows, 2^-11, where 64 bits sit on a border
        moved = B.keep(after, paths)
        for d, w in zip((base.dk, base.dv), moved):
            h = cuda.download(d, w.shape, np.uint8, s)
            steps = h.view(np.int16).astype(np.int32) - w.view(np.int16)
            assert np.abs(steps).max() <= 1 and (steps != 0).mean() < 1e-3
        assert np.array_equal(cuda.download(dlo, (2,), np.int32, s), [p + len(x_) for p, x_ in zip(past, paths)])
        pools = [cuda.download(p, pools[0].shape, np.uint8, s) for p in (base.dk, base.dv)]
    g.close()
    cuda.destroy_stream(s)
    base.free()


def test_attention_on_two_streams(cuda, K):
    """Calls that overlap, each with its workspace."""
    rng = np.random.default_rng(2)
    Bs = [Trees(cuda, [random_tree(rng, n), [-1, 0]], [5000, 900], 8, 2, 128, 64, lp.KV_Q4, seed=n).device() for n in (4, 20)]
    qs = [_f32(B.rng, B.tokens, 1024) for B in Bs]
    streams = [cuda.stream() for _ in Bs]
    jobs = []
    for B, q in zip(Bs, qs):
        dq, do, dm = B.up(q), B.alloc(q.nbytes), B.up(B.masks())
        ws = B.alloc(K.attn_tree_ws_bytes(B.cache, 8, 2, B.tokens, B.max_q, 5030))
        jobs.append((dq, do, dm, ws))
    cuda.sync()
    for _ in range(20):
        for B, s, (dq, do, dm, ws) in zip(Bs, streams, jobs):
            K.attn_tree(B.cache, dq, 1024, do, 1024, 8, B.dstarts, B.dlens, dm, 2, B.tokens, B.max_q, 5030, 1.0 / np.sqrt(128), ws,
                        s, ws_bytes=ws.nbytes)
    for B, q, s, (dq, do, dm, ws) in zip(Bs, qs, streams, jobs):
        got = cuda.download(do, (B.tokens, 8, 128), np.float32, s)
        _close(got, B.attention_tree(q.reshape(B.tokens, 8, 128), 1.0 / np.sqrt(128)))
    for s in streams:
        cuda.destroy_stream(s)
    for B in Bs:
        B.free()
