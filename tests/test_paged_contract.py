"""What lp_kv_cache, lp_kv_append_paged, lp_attn_paged and lp_logprobs state in
include/llmpager_hip.h, on the CPU."""
import numpy as np

from _paged import q4


def test_scales_that_a_q4_page_may_hold():
    """Every scale of 7 significant bits within 2^-17 .. 896: 72 of it and its
    multiples -8 .. 7 are fp16 numbers, so n s - 72 s is exact; some scale of 11 bits is
    off by s / 29 and none by more than s / 28, and from 910 on 72 of it is no number."""
    s = np.array([m * 2.0 ** e for e in range(-23, 10) for m in range(64, 128) if 2.0 ** -17 <= m * 2.0 ** e <= 896.0])
    for n in [72.0] + list(range(-8, 8)):
        assert np.array_equal((n * s).astype(np.float16).astype(np.float64), n * s)
    h = np.arange(1, 1 << 15, dtype=np.uint16).view(np.float16).astype(np.float64)
    h = h[(h >= 2.0 ** -10) & (h < 909.0)]
    off = np.abs((72.0 * h).astype(np.float16).astype(np.float64) - 72.0 * h) / h
    assert 1 / 29 < off.max() < 1 / 28
    with np.errstate(over="ignore"):
        assert np.isinf(np.float16(72.0 * 910.0)) and np.isfinite(np.float16(72.0 * 896.0))


def test_scales_as_the_append_makes_them():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((4000, 64)) * 10.0 ** rng.uniform(-8, 6, (4000, 1))
    x[0], x[1, 3] = 0.0, np.inf
    _, s = q4(x)
    m, _ = np.frexp(s)
    assert s.min() == 2.0 ** -17 and s.max() == 896.0 and np.array_equal(m * 128, np.rint(m * 128))
    assert np.array_equal(s.astype(np.float16).astype(np.float64), s)
