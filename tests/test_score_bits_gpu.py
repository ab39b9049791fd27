"""The 8-bit matrix product's bits: the number of rows picks the form (streamed,
tiles of three sizes, K in slices), and a row's result is the same in each, with
every rounding of the epilogue where the definition has it. The token log
probabilities' bits, whose form the number of alternatives picks."""

import numpy as np
import pytest

from tests.test_score_ops_gpu import (RESIDUAL, STORE, SWIGLU, matmul_inputs, run_logprobs,
                                      run_matmul, tiles_of)
from tests.util import say

pytestmark = pytest.mark.gpu


def stepwise(x, sx, q, sw, y, epilogue):
    """The result with one fp32 rounding a step: the sum, its product with the
    row's scale, with the channel's, and for RESIDUAL the addition."""
    p = (x.astype(np.float64) @ q.astype(np.float64).T).astype(np.float32)
    p = p * sx[:, None] * sw
    assert p.dtype == np.float32
    return y + p if epilogue == RESIDUAL else p


@pytest.mark.parametrize("epilogue", [STORE, RESIDUAL, SWIGLU])
@pytest.mark.parametrize("N,K,rows", [
    # streamed in each shape, tiles of 128 x 128, 128 x 256 and 256 x 256, and the
    # last with its left-over columns as either of the others
    (8003, 1088, (1, 7, 17, 40, 63, 70, 110, 160, 300, 700, 1100, 1300, 2100)),
    (8000, 1088, (1, 17, 160, 700, 2100)),
    # K in slices, their sums joined
    (2560, 9728, (1, 16, 64, 200, 300, 512, 1000)), (2561, 9728, (5, 300, 600)),
    # two weight tiles a workgroup, for thousands of them
    (66002, 192, (1, 5, 17, 33))])
def test_matmul_a8_bits_in_every_form(hip, rng, N, K, rows, epilogue):
    x, sx, q, sw, y = matmul_inputs(rng, rows[-1], N, K, epilogue)
    tiles = tiles_of(hip, q, 2 if epilogue == SWIGLU else 1)
    want = None if epilogue == SWIGLU else stepwise(x, sx, q, sw, y, epilogue)
    for M in reversed(rows):
        say(f"matmul_a8 bits M={M} N={N} K={K} epilogue={epilogue}")
        got = run_matmul(hip, x[:M], sx[:M], q, sw, y[:M], epilogue, tiles=tiles, pad=1)
        want = got if want is None else want
        assert np.array_equal(got, want[:M]), M


# The gate's whole range: flat ends, where the exponential or its reciprocal
# leaves the normal numbers (-87.3, -88.7), where silu does (-91.9, -104), beyond.
GATES = [3.4e38, 1e30, 1e4, 200.0, 104.0, 89.0, 85.0, 60.0, 20.0, 5.0, 1.0, 0.25, 1e-3, 1e-20, 1e-37,
         0.0, -1e-37, -1e-20, -1e-3, -0.25, -1.0, -1.2784645, -5.0, -20.0, -60.0, -79.5, -80.0,
         -80.5, -85.0, -87.0, -87.33, -87.5, -88.0, -88.7, -88.8, -89.0, -91.0, -91.9, -92.0, -95.0,
         -100.0, -103.0, -104.0, -110.0, -120.0, -150.0, -175.0, -200.0, -300.0, -1e4, -1e30, -3.4e38]
UPS = [1.0, -3.0, 1e-30, -1e20, 3e38]


@pytest.mark.parametrize("M,N,K", [(1, 300, 128), (64, 8200, 128), (150, 8200, 192),  # streamed
                                   (100, 2500, 9792), (300, 2560, 9728),  # K in slices
                                   (700, 5003, 128), (1100, 9000, 128), (1500, 5003, 320)])
def test_matmul_a8_swiglu_over_the_gates_range(hip, M, N, K):
    """Every sum is 1 and every row's scale 1, so gate and up are the channels'
    scales. silu of a gate down to -80 is off by 6 roundings (3 of the
    exponential, the sum, the reciprocal, the product), below by 13 with its
    product by up (twice 4 of four exponentials, 5 products), which is the
    seventh above; where that leaves the normal range, half the spacing there."""
    say(f"matmul_a8 gates M={M} N={N} K={K}")
    x, q = np.zeros((M, K), np.int8), np.zeros((2 * N, K), np.int8)
    x[:, K - 1] = q[:, K - 1] = 1
    n = np.arange(N)
    gate = np.float32(GATES)[n % len(GATES)]
    # no up that would take a positive gate's result past the range
    up = np.float32(UPS)[np.where(gate > 1, 2, n // len(GATES) % len(UPS))]
    one = np.ones(M, np.float32)
    got = run_matmul(hip, x, one, q, np.concatenate([gate, up]), np.zeros((M, N), np.float32), SWIGLU)
    g, u = gate.astype(np.float64), up.astype(np.float64)
    t = np.exp(-np.abs(g))
    want = g * np.where(g < 0, t, 1) / (1 + t) * u
    tol = np.where(g < -80, 13, 7) * 2.0 ** -24 * (1 + 1e-5) * np.abs(want) + 2.0 ** -150
    off = np.abs(got - want)
    bad = np.argwhere(~(off <= tol))
    assert not len(bad), [(int(i), float(gate[j]), float(up[j]), float(got[i, j]), want[j])
                          for i, j in bad[:8]]


@pytest.mark.parametrize("M", [1, 40, 300, 700])
def test_matmul_a8_swiglu_gate_past_the_range(hip, M):
    """A gate that is -inf in fp32 leaves 0, as any gate below -300 does; +inf
    and NaN stay what they are."""
    N, K = 50, 64
    say(f"matmul_a8 infinite gates M={M}")
    x, q = np.ones((M, K), np.int8), np.ones((2 * N, K), np.int8)
    q[1:N:3] = -1
    sx, sw = np.full(M, 1e30, np.float32), np.full(2 * N, 1e20, np.float32)
    sw[N:], sw[2:N:3] = 1e-31, np.nan
    got = run_matmul(hip, x, sx, q, sw, np.zeros((M, N), np.float32), SWIGLU)
    assert np.isposinf(got[:, 0::3]).all()
    assert (got[:, 1::3] == 0).all()
    assert np.isnan(got[:, 2::3]).all()


@pytest.mark.parametrize("rows,n", [(1, 300), (3, 151936), (20, 9000), (256, 16384), (300, 70001),
                                    (800, 5003), (800, 40000), (3000, 700)])
def test_token_logprobs_bits_whatever_is_asked_for(hip, rng, rows, n):
    """The sums' order goes by rows and n alone: any number of alternatives
    leaves the same log probabilities and entropies, and fewer alternatives are
    the first of more."""
    x = (rng.standard_normal((rows, n)) * rng.uniform(0.5, 6, (rows, 1))).astype(np.float32)
    x[::5, rng.integers(0, n, n // 3)] = -np.inf
    ids = rng.integers(0, n, (rows, 2))
    say(f"logprobs bits rows={rows} n={n} top=64")
    lp, H, ti, tl = run_logprobs(hip, x, ids, 64)
    for top in (0, 1, 5, 8, 9, 24, 25, 40):
        say(f"logprobs bits rows={rows} n={n} top={top}")
        got = run_logprobs(hip, x, ids, top)
        for a, b in zip(got, (lp, H, ti[:, :top], tl[:, :top])):
            assert np.array_equal(a, b, equal_nan=a.dtype == np.float32), top
