"""lp_verify_tree on the GPU at the ends of what its description allows, against its definition
in 64 bits (tests/_tree.py); paths and tokens are whole numbers and have to be equal."""
import numpy as np
import pytest

import llmpager_amd as lp
from _tree import verify
from test_gpu_tree import Mem
from test_gpu_verify import Case, _path_alone, _same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(cuda):
    return lp.Kernels(cuda)


# ---- calls without tokens -----------------------------------------------------------


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("batch,max_depth", [(1, 0), (3, 5), (70, 70), (1300, 2)])
@pytest.mark.parametrize("tokens,max_q,starts", [(0, 5, 0), (0, 5, 2), (9, 0, 0), (9, 0, 1), (0, 0, 0)])
def test_without_tokens(cuda, K, sampled, batch, max_depth, tokens, max_q, starts):
    """No sequence has a token, whatever the starts say (they rise by `starts`): nothing kept
    and no next token, over what a step before has left there, without a workspace."""
    m = Mem(cuda)
    x = m.up(np.zeros(9 * 50, np.float32))
    i = m.up(np.zeros(9, np.int32))
    ds = m.up(np.arange(batch + 1, dtype=np.int32) * starts)
    shapes = ((batch, max_depth + 1), (batch,), (batch,))
    out = [m.up(np.full(s, 7, np.int32)) for s in shapes]
    assert K.verify_tree_ws_bytes(50, batch, tokens, max_q, max_depth, sampled) == 0
    fill = [np.full(s, 7, np.int32) for s in shapes]
    for stream in (None, cuda.stream()):
        if stream is not None:
            for d, f in zip(out, fill):
                cuda.htod_async(d, f, stream)
        K.verify_tree(x, 50, 50, i, i, ds, batch, tokens, max_q, max_depth, 0, x if sampled else 0, 50, x, *out, 0, stream, ws_bytes=0)
        path, kept, after = (cuda.download(d, s, np.int32, stream) for d, s in zip(out, shapes))
        assert (path == -1).all() and (kept == 0).all() and (after == -1).all()
        if stream is not None:
            cuda.destroy_stream(stream)
    m.free()


# ---- tokens that are all but impossible ----------------------------------------------


def _cut(c):
    """The rows with what counts as impossible, 660 or more below the largest over the
    temperature, as -inf."""
    x = c.x.astype(np.float64)
    for b in range(len(c.trees)):
        s = slice(int(c.starts[b]), int(c.starts[b + 1]))
        x[s][(x[s] - x[s].max(1, keepdims=True)) / float(c.temps[b]) <= -660.0] = -np.inf
    return x


def _check_cut(cuda, K, c):
    c.device(cuda, K)
    c.run(K)
    want = verify(_cut(c), c.drafts, c.trees, c.starts, c.temps, c.u, c.q, c.max_depth)
    _same(c.got(cuda), want)
    c.m.free()
    return want


GAPS = [630.0, 659.0, 659.75, 660.0, 660.25, 663.0, 665.0, 666.0, 667.0, 667.5, 667.75, 668.0, 669.0, 670.0, 675.0, 690.0, 699.0, 701.0, 740.0]


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("temp", [1.0, 0.5, 0.0625])
@pytest.mark.parametrize("vocab", [5, 257, 3000])
def test_draws_of_0_beside_tokens_far_below(cuda, K, sampled, temp, vocab):
    """u = 0 draws the first token that can be drawn: those just above the border are, alone or
    many together, those below it are not, however many there are."""
    rng = np.random.default_rng(vocab)
    c = Case(rng, [4] * len(GAPS), vocab, 3, sampled, temps=[temp] * len(GAPS))
    c.u[:] = 0.0
    for b, gap in enumerate(GAPS):
        x = c.x[c.starts[b]:c.starts[b + 1]]
        x[:] = -gap * temp
        x[:, vocab - 2] = 0.0
        x[1::2, vocab - 1] = 0.0
        x[2, :vocab // 2] = -np.inf
    if sampled:
        c.q[:] = 0.0
        c.q[:, vocab - 1] = 1.0
    c.drafts[:] = vocab - 1
    w = _check_cut(cuda, K, c)
    assert (w[2][:3] != vocab - 2).any() and (w[2][3:] >= vocab // 2).all()


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("vocab", [6, 2500])
def test_what_is_left_far_below(cuda, K, gap, vocab):
    """A child is turned down, and beside a token or none only tokens far below are left: p itself
    counts again where none of them can be drawn."""
    rng = np.random.default_rng(vocab)
    c = Case(rng, [2, 3, 2, 3], vocab, 3, True, temps=[1.0] * 4)
    c.u[:] = 0.0
    for b in range(4):
        s = int(c.starts[b])
        c.trees[b] = [-1] + [0] * (len(c.trees[b]) - 1)
        c.parents[s:s + len(c.trees[b])] = c.trees[b]
        c.x[s] = -gap
        c.x[s, vocab - 3] = 0.0
        if b >= 2:
            c.x[s, vocab - 2] = 0.0
        c.q[s] = 0.0
        c.q[s, vocab - 3] = 1.0
        c.drafts[s + 1:s + len(c.trees[b])] = vocab - 3
        c.u[s + 1:s + len(c.trees[b])] = 1 - 2.0 ** -24
        c.q[s, vocab - 3] = 1.5
    _check_cut(cuda, K, c)


@pytest.mark.parametrize("gap", GAPS)
def test_draws_of_0_on_large_trees(cuda, K, gap):
    """The same, and by the smallest number above 0, where the rows of the path alone are read."""
    sizes, vocab = [200] * 6, 30001
    assert _path_alone(K, sizes, vocab, 5)
    rng = np.random.default_rng(5)
    c = Case(rng, sizes, vocab, 5, temps=[1.0] * 6)
    c.x[:] = -gap
    c.x[:, 12345] = 0.0
    c.x[::2, 777] = 0.0
    c.u[:] = rng.choice(np.array([0.0, 2.0 ** -149, 0.75], np.float32), c.T)
    assert (c.u > 0).any() and (c.u[c.u > 0] < 1e-40).any()
    c.drafts[:] = rng.choice([0, 777, 12345], c.T)
    w = _check_cut(cuda, K, c)
    assert (gap < 660) == (w[2] == 0).any()


# ---- starts that do not rise, temperatures without end ------------------------------------


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("vocab,n,batch", [(200, 4, 3), (33000, 400, 3), (3001, 120, 70)])
def test_starts_that_fall_leave_no_sequences(cuda, K, vocab, n, batch, sampled):
    """Whether all rows are read or those of the path alone."""
    rng = np.random.default_rng(13)
    c = Case(rng, [n] * batch, vocab, 3, sampled)
    assert sampled or _path_alone(K, [n] * batch, vocab, 3) == (n > 4)
    c.starts[batch - 1] = c.starts[batch - 2] - 2
    c.device(cuda, K)
    c.run(K)
    path, kept, after = c.got(cuda)
    assert (path == -1).all() and (kept == 0).all() and (after == -1).all()
    c.m.free()
    c = Case(rng, [n] * batch, vocab, 3, sampled).device(cuda, K)  # and the calls behind it are as ever
    c.run(K)
    _same(c.got(cuda), c.want())
    c.m.free()


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("sizes,vocab", [([8, 5], 3000), ([200] * 3, 40000)])
def test_infinite_temperatures(cuda, K, sampled, sizes, vocab):
    """Every token that can be drawn at all is as likely as any other."""
    rng = np.random.default_rng(15)
    c = Case(rng, sizes, vocab, 5, sampled, temps=[1.0] * len(sizes))
    c.x[:, 100:120] = -np.inf
    c.temps[:] = np.inf
    c.device(cuda, K)
    c.run(K)
    flat = np.where(c.x == -np.inf, -np.inf, 0.0)
    _same(c.got(cuda), verify(flat, c.drafts, c.trees, c.starts, np.ones(len(sizes)), c.u, c.q, c.max_depth))
    c.m.free()
