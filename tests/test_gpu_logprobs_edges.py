"""lp_logprobs of rows that are all but certain: what is left is in the other tokens'
terms alone, far below the 1 of the largest."""
import numpy as np
import pytest

import llmpager_amd as lp
from test_gpu_logprobs import _run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(cuda):
    return lp.Kernels(cuda)


# A term's exponential is good to 2^-22 (1 + |d|) of it for its distance d, the sums
# to 64 bits but for 16 of one lane in fp32 (2^-20 of them), the result to 2^-24.
@pytest.mark.parametrize("rows,vocab,top", [(1, 700, 3), (3, 151936, 5), (2, 32003, 0), (600, 5000, 1)])
@pytest.mark.parametrize("gap", [30.0, 37.0, 40.0, 60.0, 75.0])
@pytest.mark.parametrize("at", ["first", "middle", "last"])
def test_all_but_certain(cuda, K, rows, vocab, top, gap, at):
    rng = np.random.default_rng(int(gap) + vocab)
    k = {"first": 0, "middle": vocab // 2, "last": vocab - 1}[at]
    x = (-gap + rng.standard_normal((rows, vocab))).astype(np.float32)
    x[:, k] = 0.25
    logp, ent, ids, tp = _run(cuda, K, x, np.full(rows, k), top)
    d = x.astype(np.float64) - 0.25
    d[:, k] = -np.inf
    r = np.exp(d).sum(1)
    want = np.log1p(r) + (np.exp(d) * np.where(np.isinf(d), 0, -d)).sum(1) / (1 + r)
    tol = 2.0 ** -22 * (gap + 6) + 2.0 ** -20
    assert (np.abs(logp / -np.log1p(r) - 1) < tol).all(), (logp, r)
    assert (np.abs(ent / want - 1) < tol).all(), (ent, want)
    if top:
        assert (ids[:, 0] == k).all() and np.array_equal(tp[:, 0], logp)


@pytest.mark.parametrize("vocab", [900, 151936])
@pytest.mark.parametrize("n", [2, 5, 300])
def test_equal_best_and_next_to_nothing_else(cuda, K, vocab, n):
    """n equal logits far above the others: ln n and, of it, what fp32 holds."""
    rng = np.random.default_rng(n)
    x = (-50 + rng.standard_normal((2, vocab))).astype(np.float32)
    at = rng.permutation(vocab)[:n]
    x[:, at] = 3.0
    logp, ent, _, _ = _run(cuda, K, x, np.full(2, at[0]), 0)
    assert (np.abs(logp / -np.log(n) - 1) < 2.0 ** -23).all() and (np.abs(ent / np.log(n) - 1) < 2.0 ** -23).all()
