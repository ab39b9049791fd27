"""The 8-bit matrix product's bits: the number of rows picks the form (streamed,
tiles of three sizes, K in slices), and a row's result is the same in each, with
every rounding of the epilogue where the definition has it."""

import numpy as np
import pytest

from tests.test_score_ops_gpu import RESIDUAL, STORE, SWIGLU, matmul_inputs, run_matmul, tiles_of
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
