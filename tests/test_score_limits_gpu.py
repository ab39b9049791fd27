"""The largest sizes that the 8-bit norm, the 8-bit matrix product and the token
log probabilities take (what lies past them is refused on the host), and rows
whose scale leaves fp32; references and tolerances of test_score_ops_gpu."""

import numpy as np
import pytest

from tests.test_score_ops_gpu import (RESIDUAL, STORE, SWIGLU, check_logprobs, check_norm,
                                      matmul_inputs, matmul_ref, norm_ref, run_matmul, run_norm)
from tests.util import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,epilogue", [(1, STORE), (3, RESIDUAL), (20, SWIGLU)])
def test_matmul_a8_most_rows(hip, rng, N, epilogue):
    M, K = (1 << 20) - 1, 64
    say(f"matmul_a8 M={M} N={N} epilogue={epilogue}")
    x, sx, q, sw, y = matmul_inputs(rng, M, N, K, epilogue)
    got = run_matmul(hip, x, sx, q, sw, y, epilogue)
    want, tol = matmul_ref(x, sx, q, sw, y, epilogue)
    assert (np.abs(got - want) <= tol * 1.0001 + 1e-37).all()


@pytest.mark.parametrize("M", [1, 3])
def test_matmul_a8_most_outputs(hip, rng, M):
    N, K = (1 << 23) - 1, 64
    say(f"matmul_a8 M={M} N={N}")
    x, sx, q, sw, y = matmul_inputs(rng, M, 4093, K, STORE)
    some, tol = matmul_ref(x, sx, q, sw, y, STORE)
    rows = np.arange(N) % 4093
    got = run_matmul(hip, x, sx, q[rows], sw[rows], np.zeros((M, N), np.float32), STORE)
    assert (np.abs(got - some[:, rows]) <= tol[:, rows] * 1.0001 + 1e-37).all()


@pytest.mark.parametrize("n", [1, 5, 66])
def test_norm_q8_most_rows(hip, rng, n):
    rows = 1 << 21
    say(f"norm_q8 rows={rows} n={n}")
    x = rng.standard_normal((rows, n)).astype(np.float32)
    w = rng.uniform(-0.5, 0.5, n).astype(np.float32)
    check_norm(run_norm(hip, x, None, w), norm_ref(x, None, w, 1e-6))


@pytest.mark.parametrize("n,top", [(3, 2), (1, 0), (5, 5)])
def test_token_logprobs_most_rows(hip, rng, n, top):
    rows = 1 << 21
    say(f"logprobs rows={rows} n={n} top={top}")
    x = rng.standard_normal((rows, n)).astype(np.float32)
    check_logprobs(hip, x, np.zeros((rows, 0), np.int32), top)


@pytest.mark.parametrize("n,fits", [(300, True), (2560, True), (16129, True), (16641, False),
                                    (40000, False)])
def test_norm_q8_scale_past_the_range(hip, rng, n, fits):
    """One value under a gain of fp32's largest: y is sqrt(n) and the scale
    sqrt(n) / 127 of 1 + that. At n = 127^2 this is 1 + the largest, which rounds
    to the largest and fits; beyond it there is no scale: NaN, bytes 0. In the row
    beside it the same gain meets zeros only."""
    say(f"norm_q8 scale past the range n={n}")
    x, w = np.zeros((2, n), np.float32), np.zeros(n, np.float32)
    x[0, n // 2] = x[1, 0] = 2.0
    w[n // 2] = np.finfo(np.float32).max
    q, sc, _ = run_norm(hip, x, None, w, eps=0.0)
    qr, scr, _ = norm_ref(x, None, w, 0.0)
    with np.errstate(over="ignore"):
        assert fits == np.isfinite(np.float32(scr[0]))
    if not fits:
        assert np.isnan(sc[0]) and not q[0].any()
    fine = slice(0 if fits else 1, 2)
    check_norm((q[fine], sc[fine], None), (qr[fine], scr[fine], None))


@pytest.mark.parametrize("n", [300, 2560, 40000])
def test_norm_q8_sum_past_the_range(hip, rng, n):
    """A sum that is infinite makes its row one that is not finite."""
    say(f"norm_q8 sum past the range n={n}")
    x, d = rng.standard_normal((2, 3, n)).astype(np.float32)
    x[1, n - 1] = d[1, n - 1] = 3e38
    w = np.zeros(n, np.float32)
    q, sc, s = run_norm(hip, x, d, w)
    with np.errstate(all="ignore"):
        qr, scr, sr = norm_ref(x, d, w, 1e-6)
    assert np.isnan(sc[1]) and not q[1].any() and np.isposinf(s[1, n - 1])
    fine = [0, 2]
    check_norm((q[fine], sc[fine], s), (qr[fine], scr[fine], sr))
