"""lp_verify_tree on the GPU against its definition in 64 bits (tests/_tree.py), and a
whole step with drafted tokens as a program runs it.

Paths and tokens are whole numbers and have to be equal.  Both sides' sums are 64-bit, the
device's exponentials good to 2^-40: a border between two tokens is off by 1e-12 of the whole
at most, and of 2^24 numbers u the chance that one lies that near any of 2^19 borders is below
1e-6 a draw."""
import numpy as np
import pytest

import llmpager_amd as lp
from _paged import HipGraph
from _tree import Trees, random_tree, row_probs, pick, verify
from test_gpu_tree import Mem

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(cuda):
    return lp.Kernels(cuda)


class Case:
    """Trees of drafts over rows of logits, in which some drafts are what is drawn."""

    def __init__(self, rng, sizes, vocab, max_depth, sampled=False, temps=None, chain=False, pad=0, front=0, luck=0.75, limit=1 << 30):
        self.vocab, self.max_depth, self.sampled = vocab, max_depth, sampled
        self.trees = [([-1] + list(range(n - 1)) if chain else random_tree(rng, n, limit)) if n else [] for n in sizes]
        self.starts = (front + np.concatenate(([0], np.cumsum(sizes)))).astype(np.int32)
        self.T = int(self.starts[-1]) + pad
        self.x = (rng.standard_normal((self.T, vocab)) * 2).astype(np.float32)
        self.x = (self.x.view(np.uint32) & 0xffff0000).view(np.float32)  # a coarse grid: equal values
        self.x[::3, vocab // 3] += 7
        self.temps = np.array([rng.choice([0.6, 1.0, 1.3]) for _ in sizes] if temps is None else temps, np.float32)
        self.u = rng.random(self.T, dtype=np.float32)
        self.parents = np.full(self.T, 0, np.int32)
        self.drafts = rng.integers(0, vocab, self.T).astype(np.int32)
        self.q = None
        if sampled:
            y = self.x + rng.standard_normal(self.x.shape).astype(np.float32)
            e = np.exp(y - y.max(1, keepdims=True))
            self.q = (e / e.sum(1, keepdims=True)).astype(np.float32)
        for b, up in enumerate(self.trees):
            at = int(self.starts[b])
            self.parents[at:at + len(up)] = up
            for i, p in enumerate(up):
                if i == 0:
                    continue
                if sampled:
                    self.drafts[at + i] = pick(self.q[at + p].astype(np.float64), rng.random())
                elif rng.random() < luck:
                    pr = row_probs(self.x[at + p], self.temps[b])
                    self.drafts[at + i] = pick(pr, float(self.u[at + p]) if self.temps[b] > 0 else 0.0)

    def want(self):
        return verify(self.x, self.drafts, self.trees, self.starts, self.temps, self.u, self.q, self.max_depth)

    def device(self, cuda, K, cols=0, shift=0, max_q=None):
        """Uploads; `cols` floats behind a row, rows `shift` floats off 16 bytes."""
        m = self.m = Mem(cuda)
        self.stride = self.vocab + cols

        def rows(a):
            flat = np.full(shift + self.T * self.stride, np.nan, np.float32)
            flat[shift:].reshape(self.T, self.stride)[:, :self.vocab] = a
            return m.up(flat) + 4 * shift

        self.dx, self.dq = rows(self.x), rows(self.q) if self.sampled else 0
        self.dd, self.dp, self.ds = m.up(self.drafts), m.up(self.parents), m.up(self.starts)
        self.dt, self.du = m.up(self.temps), m.up(self.u)
        B = len(self.trees)
        self.max_q = max_q or max([len(t) for t in self.trees] + [1])
        self.out = [m.up(np.full(n, 7, np.int32)) for n in (B * (self.max_depth + 1), B, B)]
        self.ws = m.alloc(K.verify_tree_ws_bytes(self.vocab, B, self.T, self.max_q, self.max_depth, self.sampled))
        return self

    def run(self, K, stream=None, temps=True):
        K.verify_tree(self.dx, self.stride, self.vocab, self.dd, self.dp, self.ds, len(self.trees), self.T, self.max_q,
                      self.max_depth, self.dt if temps else 0, self.dq, self.stride, self.du, *self.out, self.ws, stream,
                      ws_bytes=self.ws.nbytes)

    def got(self, cuda, stream=None):
        B = len(self.trees)
        return tuple(cuda.download(d, s, np.int32, stream) for d, s in zip(self.out, ((B, self.max_depth + 1), (B,), (B,))))


def _same(got, want):
    for g, w, n in zip(got, want, ("path", "kept", "next")):
        assert np.array_equal(g, w), (n, np.argwhere(g != w)[:4], g[g != w][:4], w[g != w][:4])


def _check(cuda, K, c, **kw):
    c.device(cuda, K, **kw)
    c.run(K)
    want = c.want()
    _same(c.got(cuda), want)
    c.m.free()
    return want


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 255, 257, 1000, 1023, 1024, 1025, 4097, 32003])
def test_vocabularies(cuda, K, vocab, sampled):
    rng = np.random.default_rng(vocab)
    w = _check(cuda, K, Case(rng, [9, 1, 6, 12], vocab, 5, sampled))
    assert vocab < 1000 or w[1].max() > 1


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("vocab", [151936, 300001, 1 << 19])
def test_large_vocabularies(cuda, K, vocab, sampled):
    rng = np.random.default_rng(vocab)
    _check(cuda, K, Case(rng, [5, 3], vocab, 4, sampled))


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("sizes,max_depth,kw", [
    ([1], 0, {}), ([1, 1, 1], 3, {}), ([8], 0, {}), ([8, 5], 1, {}),
    ([0, 7, 0, 0, 2, 0], 4, dict(pad=3, front=2)),
    ([7] * 20, 6, dict(chain=True)),
    ([40, 64], 30, dict(chain=True, luck=1.0)),
    ([65, 130, 3], 9, {}),
    ([30, 20, 10], 2, dict(limit=2)),
    ([50, 50], 10, dict(limit=1)),                 # many children of one node
])
def test_trees(cuda, K, sizes, max_depth, kw, sampled):
    rng = np.random.default_rng(sum(sizes) + max_depth)
    _check(cuda, K, Case(rng, sizes, 700, max_depth, sampled, **kw))


@pytest.mark.parametrize("sampled", [False, True])
def test_many_nodes(cuda, K, sampled):
    rng = np.random.default_rng(1)
    w = _check(cuda, K, Case(rng, [1024, 700], 90, 40, sampled))
    assert w[1].max() > (1 if sampled else 4)


@pytest.mark.parametrize("sampled", [False, True])
def test_many_sequences(cuda, K, sampled):
    """More sequences than lanes, than a set of arrival counters, and tokens than that."""
    rng = np.random.default_rng(2)
    sizes = rng.integers(0, 5, 1300).tolist()
    _check(cuda, K, Case(rng, sizes, 300, 3, sampled, pad=2))


def _path_alone(K, sizes, vocab, max_depth):
    """Whether a call reads the rows of the path one behind the other: its workspace
    has no records of the others."""
    n = K.verify_tree_ws_bytes(vocab, len(sizes), sum(sizes) + 2, max(sizes), max_depth, False)
    return n < sum(sizes) * (vocab // 1024) * 16


@pytest.mark.parametrize("sizes,vocab,max_depth", [([100, 3, 0, 80, 1], 150000, 3), ([300], 200001, 7), ([64] * 40, 30001, 5),
                                                   ([0, 200, 150, 90, 0, 200], 70001, 6), ([120] * 64, 3001, 4),
                                                   ([1000, 1, 700], 60001, 6), ([7] * 1300, 3000, 2)])
def test_large_trees(cuda, K, sizes, vocab, max_depth):
    """Sizes at which the rows of the path alone are read."""
    assert _path_alone(K, sizes, vocab, max_depth)
    rng = np.random.default_rng(vocab)
    temps = [rng.choice([0.0, 0.7, 1.0]) for _ in sizes]
    w = _check(cuda, K, Case(rng, sizes, vocab, max_depth, temps=temps, pad=1, front=1))
    assert w[1].max() > 2


@pytest.mark.parametrize("kind", ["temperatures", "drafts", "numbers", "rows", "max_q"])
def test_large_trees_at_the_ends(cuda, K, kind):
    """What the tests below look at, where the rows of the path alone are read."""
    rng = np.random.default_rng(len(kind))
    sizes, vocab = [200] * 6, 30001
    assert _path_alone(K, sizes, vocab, 5)
    c = Case(rng, sizes, vocab, 5, luck=0.9, front=1, pad=1, temps=[0, -1, np.nan, 1e-6, 0.01, 50] if kind == "temperatures" else [0, 0.7, 0.7, 1, 1, 1])
    if kind == "drafts":
        c.drafts[rng.random(c.T) < 0.2] = -1
        c.drafts[rng.random(c.T) < 0.1] = vocab
        for t in rng.choice(c.T, 100, replace=False):
            c.parents[t] = rng.choice([-1, 199, 200, -2 ** 31, 2 ** 31 - 1])
        c.trees = [c.parents[c.starts[b]:c.starts[b + 1]].tolist() for b in range(6)]
    if kind == "numbers":
        c.u[:] = rng.choice([0.0, 2.0 ** -24, 1 - 2.0 ** -24], c.T)
        c.x[:, :2300] = -np.inf
        c.x[:, 29000:] = -np.inf
    if kind == "rows":
        c.x[::4, 1029] = np.inf
        c.x[2::4, vocab - 1] = np.nan
    if kind != "max_q":
        _check(cuda, K, c, cols=3, shift=1)
        return
    full, c.trees = c.trees, [t[:150] for t in c.trees]
    want = c.want()
    c.trees = full
    c.device(cuda, K, max_q=150)
    c.run(K)
    _same(c.got(cuda), want)
    c.m.free()


@pytest.mark.parametrize("sampled", [False, True])
def test_temperatures(cuda, K, sampled):
    """0, negative, NaN, tiny, large and infinite ones."""
    rng = np.random.default_rng(3)
    c = Case(rng, [8] * 9, 3000, 5, sampled, temps=[0, -1, np.nan, 1e-6, 1e-20, 0.01, 50, 1e6, 1])
    c.temps[2] = np.nan
    _check(cuda, K, c)


@pytest.mark.parametrize("sampled", [False, True])
def test_without_temperatures(cuda, K, sampled):
    rng = np.random.default_rng(4)
    c = Case(rng, [8, 6, 3], 2000, 5, sampled, temps=[1, 1, 1]).device(cuda, K)
    c.run(K, temps=False)
    _same(c.got(cuda), c.want())
    c.m.free()


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_rows_that_are_strided_and_off_16_bytes(cuda, K, sampled, shift):
    rng = np.random.default_rng(5)
    _check(cuda, K, Case(rng, [9, 4], 1501, 5, sampled), cols=shift + 2, shift=shift)


@pytest.mark.parametrize("sampled", [False, True])
def test_numbers_at_the_ends(cuda, K, sampled):
    """u of 0, of the smallest step and of the largest below 1; logits of -inf before, between
    and behind those that can be drawn."""
    rng = np.random.default_rng(6)
    c = Case(rng, [6] * 6, 2100, 4, sampled)
    c.u[:] = rng.choice([0.0, 2.0 ** -24, 1 - 2.0 ** -24], c.T)
    c.x[:, :300] = -np.inf
    c.x[:, 900:1930:2] = -np.inf
    c.x[:, 2000:] = -np.inf
    _check(cuda, K, c)


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("sizes,vocab", [([9] * 8, 1300), ([90] * 10, 50000)])
def test_rows_from_which_nothing_can_be_drawn(cuda, K, sampled, sizes, vocab):
    rng = np.random.default_rng(7)
    c = Case(rng, sizes, vocab, 4, sampled, luck=1.0, front=1, temps=[0.0 if b % 4 == 3 else 0.8 for b in range(len(sizes))])
    for t in range(0, c.T, 5):
        c.x[t] = [np.full(vocab, -np.inf), np.where(np.arange(vocab) == vocab - 1, np.nan, c.x[t]),
                  np.where(np.arange(vocab) == 1029, np.inf, c.x[t])][t // 5 % 3]
    w = _check(cuda, K, c)
    assert (w[2] == -1).any() and (w[2] >= 0).any()


@pytest.mark.parametrize("sampled", [False, True])
def test_rows_sure_of_one_token(cuda, K, sampled):
    """One logit far above all others, at the row's ends and between blocks."""
    rng = np.random.default_rng(8)
    c = Case(rng, [7] * 6, 5000, 5, sampled)
    for t in range(c.T):
        c.x[t, [0, 1023, 1024, 4999, 2500][t % 5]] = [60.0, 400.0, 1e30][t % 3]
    for b, up in enumerate(c.trees):
        for i in range(1, len(up)):
            c.drafts[c.starts[b] + i] = np.argmax(c.x[c.starts[b] + up[i]]) if rng.random() < 0.7 else 17
    _check(cuda, K, c)


@pytest.mark.parametrize("sampled", [False, True])
def test_drafts_that_are_equal_or_no_tokens(cuda, K, sampled):
    rng = np.random.default_rng(9)
    c = Case(rng, [20] * 8, 40, 6, sampled, temps=[0, 0.5, 1, 1, 1, 1, 2, 2])
    c.drafts[rng.random(c.T) < 0.2] = -1
    c.drafts[rng.random(c.T) < 0.1] = 40
    c.drafts[rng.random(c.T) < 0.1] = 2 ** 31 - 1
    _check(cuda, K, c)


@pytest.mark.parametrize("sampled", [False, True])
def test_parents_that_are_none(cuda, K, sampled):
    """Nodes that follow no lower one are never come to."""
    rng = np.random.default_rng(10)
    c = Case(rng, [12] * 4, 500, 6, sampled)
    for t in rng.choice(c.T, 12, replace=False):
        c.parents[t] = rng.choice([-1, 11, 12, -2 ** 31, 2 ** 31 - 1])
    c.trees = [c.parents[c.starts[b]:c.starts[b + 1]].tolist() for b in range(4)]
    _check(cuda, K, c)


@pytest.mark.parametrize("sampled", [False, True])
def test_tokens_past_max_q(cuda, K, sampled):
    rng = np.random.default_rng(11)
    c = Case(rng, [20, 3, 9], 500, 6, sampled)
    full, c.trees = c.trees, [t[:8] for t in c.trees]
    want = c.want()
    c.trees = full
    c.device(cuda, K, max_q=8)
    c.run(K)
    _same(c.got(cuda), want)
    c.m.free()


def test_distributions_that_end(cuda, K):
    """Draft probabilities that leave nothing of the target's (q above p everywhere): p
    itself counts again; and rows of zeros, which leave all of it."""
    rng = np.random.default_rng(12)
    c = Case(rng, [6] * 12, 50, 4, True)
    c.q[:36] = 2.0
    c.q[36:] = 0.0
    c.u[:] = rng.random(c.T, dtype=np.float32) * 0.9 + 0.1
    _check(cuda, K, c)


def test_starts_that_fall_change_nothing(cuda, K):
    rng = np.random.default_rng(13)
    for vocab, n in ((200, 4), (33000, 400)):  # all rows at once, and those of the path
        c = Case(rng, [n, n, n], vocab, 3)
        c.starts[2] = c.starts[1] - 2
        c.device(cuda, K)
        c.run(K)
        cuda.sync()
        c.m.free()
        c = Case(rng, [n, n, n], vocab, 3)  # and the calls behind it are as ever
        _check(cuda, K, c)


def test_starts_that_fall_with_sampled_drafts(cuda, K):
    """No row has a sequence then, and none is left a walk to go on with, whatever the
    workspace held before."""
    rng = np.random.default_rng(14)
    c = Case(rng, [4, 4, 4], 200, 3, True)
    c.starts[2] = c.starts[1] - 2
    c.device(cuda, K)
    cuda.htod_async(c.ws, np.full(c.ws.nbytes, 0x5a, np.uint8))
    c.run(K)
    path, kept, after = c.got(cuda)
    assert (path == -1).all() and (kept == 0).all() and (after == -1).all()
    c.m.free()
    _check(cuda, K, Case(rng, [4, 4, 4], 200, 3, True))  # and the calls behind it are as ever


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("capture", ["library", "runtime"])
@pytest.mark.parametrize("sizes,vocab", [([12] * 4, 9000), ([200] * 3, 40000)])
def test_captured(cuda, K, sampled, capture, sizes, vocab):
    """Replayed with other logits, numbers and trees, the program's own calls between."""
    rng = np.random.default_rng(14)
    c = Case(rng, sizes, vocab, 4, sampled).device(cuda, K)
    s = cuda.stream()
    if capture == "library":
        cuda.capture_begin(s)
        c.run(K, s)
        g = cuda.capture_end(s)
    else:
        g = HipGraph(s, lambda stream: c.run(K, stream))
    for i in range(4):
        n = Case(rng, [max(1, k - 3 * i) for k in sizes], vocab, 4, sampled, pad=sum(min(3 * i, k - 1) for k in sizes))
        assert n.T == c.T
        for d, v in ((c.dx, n.x), (c.dd, n.drafts), (c.dp, n.parents), (c.ds, n.starts), (c.dt, n.temps), (c.du, n.u)):
            cuda.htod_async(d, v)
        if sampled:
            cuda.htod_async(c.dq, n.q)
        cuda.sync()
        if i == 2:
            c.run(K, s)
            _same(c.got(cuda, s), n.want())
        g.launch(s)
        _same(c.got(cuda, s), n.want())
    g.close()
    cuda.destroy_stream(s)
    c.m.free()


def test_on_two_streams(cuda, K):
    rng = np.random.default_rng(15)
    cs = [Case(rng, [10] * 5, 20000, 4, i % 2 == 1).device(cuda, K) for i in range(4)]
    streams = [cuda.stream() for _ in cs]
    cuda.sync()
    for _ in range(15):
        for c, s in zip(cs, streams):
            c.run(K, s)
    for c, s in zip(cs, streams):
        _same(c.got(cuda, s), c.want())
        cuda.destroy_stream(s)
        c.m.free()


# ---- a step as a program runs it -----------------------------------------------------


def test_steps_of_a_small_model(cuda, K):
    """Greedy decoding of a one-layer model with trees of drafts, some right, gives the
    tokens and the cache rows that decoding one token at a time gives in 64 bits."""
    rng = np.random.default_rng(16)
    heads, kv, dim, page, V, steps = 4, 2, 64, 16, 120, 6
    H, W = heads * dim, (heads + 2 * kv) * dim
    emb = rng.standard_normal((V, W)).astype(np.float32)
    head = (rng.standard_normal((H, V)) / np.sqrt(H) * 4).astype(np.float32)
    prompts = [rng.integers(0, V, n).tolist() for n in (5, 17, 1)]
    nb, n_max, room = len(prompts), 9, 64
    B = Trees(cuda, [[]] * nb, [room] * nb, heads, kv, dim, page, lp.KV_F16, seed=1)
    freq = B.freq.astype(np.float64)

    def turn(x, pos):  # [..., dim]
        c, s = np.cos(pos * freq), np.sin(pos * freq)
        a, z = x[..., :dim // 2], x[..., dim // 2:]
        return np.concatenate((a * c - z * s, a * s + z * c), -1)

    def decode(tokens):
        """(the next token, keys, values of all) in 64 bits, rows rounded as held."""
        e = emb[tokens].astype(np.float64)
        ks = np.stack([turn(e[i, H:H + kv * dim].reshape(kv, dim), i) for i in range(len(tokens))]).astype(np.float16).astype(np.float64)
        vs = e[:, H + kv * dim:].reshape(-1, kv, dim).astype(np.float16).astype(np.float64)
        q = turn(e[-1, :H].reshape(heads, dim), len(tokens) - 1).reshape(kv, heads // kv, dim)
        s = np.einsum("kgd,rkd->kgr", q, ks) / np.sqrt(dim)
        p = np.exp(s - s.max(-1, keepdims=True))
        o = np.einsum("kgr,rkd->kgd", p / p.sum(-1, keepdims=True), vs).reshape(H)
        x = o @ head.astype(np.float64)
        best = np.sort(x)
        assert best[-1] - best[-2] > 1e-3  # else the test's own seed decides nothing
        return int(np.argmax(x)), ks, vs

    truth = [list(p) for p in prompts]
    for t in truth:
        for _ in range(steps * 5 + 8):
            t.append(decode(t)[0])
    table = np.stack([np.arange(b * 4, b * 4 + 4) for b in range(nb)]).astype(np.int32)
    B.pages, B.cols, B.table = 4 * nb + 3, 4, table
    B.pools = [np.zeros((B.pages, kv, B.page_bytes), np.uint8) for _ in range(2)]
    # the prompts but for their last tokens are there already
    lens = [len(p) - 1 for p in prompts]
    for b, p in enumerate(prompts):
        if len(p) > 1:
            _, ks, vs = decode(p)
            for i in range(len(p) - 1):
                B.put(i, ks[i].astype(np.float16), vs[i].astype(np.float16), b)
    B.device()
    m = Mem(cuda)
    done = [list(p) for p in prompts]
    for step in range(steps):
        trees, drafts = [], []
        for b in range(nb):
            up = random_tree(rng, int(rng.integers(2, n_max + 1)), 5)
            d = [done[b][-1]]
            for i in range(1, len(up)):
                chain, j = [], up[i]
                while j > 0:
                    chain.insert(0, d[j])
                    j = up[j]
                at = len(done[b]) + len(chain)
                right = truth[b][at] if truth[b][len(done[b]):at] == chain else None
                d.append(right if right is not None and rng.random() < 0.6 else int(rng.integers(0, V)))
            trees.append(up), drafts.append(d)
        starts = np.concatenate(([0], np.cumsum([len(t) for t in trees]))).astype(np.int32)
        T, Q = int(starts[-1]), max(map(len, trees))
        now = np.array([n + len(t) for n, t in zip(lens, trees)], np.int32)
        flat = np.concatenate(drafts).astype(np.int32)
        dx, dp, ds, dl = m.up(emb[flat]), m.up(np.concatenate(trees).astype(np.int32)), m.up(starts), m.up(now)
        ddep, dmask, dq, do = m.alloc(4 * T), m.alloc(8 * T), m.alloc(T * H * 4), m.alloc(T * H * 4)
        K.tree_layout(dp, ds, nb, T, Q, ddep, dmask)
        K.kv_append_tree(B.cache, dx, W, dx + H * 4, W, dx + (H + kv * dim) * 4, W, 0, 0, 1e-6, B.up(B.freq), 1.0, dq, H, 0, 0, heads,
                         ds, dl, ddep, nb, T)
        ws = m.alloc(K.attn_tree_ws_bytes(B.cache, heads, nb, T, Q, room))
        K.attn_tree(B.cache, dq, H, do, H, heads, ds, dl, dmask, nb, T, Q, room, 1.0 / np.sqrt(dim), ws, ws_bytes=ws.nbytes)
        logits = (cuda.download(do, (T, H), np.float32).astype(np.float64) @ head).astype(np.float32)
        out = [m.alloc(4 * n) for n in (nb * 6, nb, nb, nb)]
        ws = m.alloc(K.verify_tree_ws_bytes(V, nb, T, Q, 5, False))
        K.verify_tree(m.up(logits), V, V, m.up(flat), dp, ds, nb, T, Q, 5, m.up(np.zeros(nb, np.float32)), 0, 0,
                      m.up(np.zeros(T, np.float32)), *out[:3], ws, ws_bytes=ws.nbytes)
        K.kv_keep([B.cache], out[0], 5, out[1], ds, dl, out[3], nb)
        path, kept, nxt, after = (cuda.download(d, s, np.int32) for d, s in zip(out, ((nb, 6), (nb,), (nb,), (nb,))))
        for b in range(nb):
            done[b] += [drafts[b][i] for i in path[b, 1:kept[b]]] + [int(nxt[b])]
            lens[b] = int(after[b])
            assert lens[b] == len(done[b]) - 1
            assert done[b] == truth[b][:len(done[b])]
    assert sum(map(len, done)) > sum(map(len, prompts)) + steps * nb  # some drafts stayed
    k, v = (cuda.download(d, B.pools[0].shape, np.uint8).view(np.float16).reshape(B.pages, kv, page, dim) for d in (B.dk, B.dv))
    for b in range(nb):
        _, ks, vs = decode(done[b][:-1])
        for got, want in ((k, ks), (v, vs)):
            rows = np.concatenate([got[p] for p in table[b]], 1).transpose(1, 0, 2)[:lens[b]]
            assert np.allclose(rows, want, rtol=2.0 ** -10, atol=2.0 ** -24)
    m.free(), B.free()
