"""Every form that the 8-bit matrix product and the token log probabilities
take by the size of a call, and offsets past 32 bits, against the definitions
in 64 bits (references and tolerances of test_score_ops_gpu)."""

import numpy as np
import pytest

from tests.test_score_ops_gpu import (RESIDUAL, STORE, SWIGLU, buf, check_logprobs, check_norm,
                                      logprobs_ref, matmul_inputs, matmul_ref, norm_ref,
                                      run_matmul, run_norm, tiles_of)
from tests.util import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("epilogue", [STORE, RESIDUAL, SWIGLU])
@pytest.mark.parametrize("M,N,K", [
    # streamed: rows and weight tiles a workgroup, its waves, the depth of their rings
    (1, 8200, 704), (5, 66000, 192), (17, 66000, 192), (17, 8200, 320), (31, 3001, 1088),
    (33, 8200, 704), (50, 8200, 704), (33, 2500, 2624), (50, 2500, 1216), (65, 2500, 2624),
    (130, 2500, 1216), (2600, 131, 320),
    # tiles of 128 x 128, whole and with K in 2, 4 and 8 slices, odd blocks of K
    (150, 8200, 192), (513, 4100, 1984), (50, 9000, 9792), (50, 5003, 9792), (100, 2500, 9792),
    (100, 1040, 9792), (100, 5003, 2624),
    # tiles of 128 x 256
    (521, 9741, 448), (600, 9100, 1088), (521, 9741, 1024),
    # tiles of 256 x 256, alone and with columns left over
    (2600, 5003, 192), (1500, 5003, 320), (700, 33000, 192), (4100, 8300, 192),
    (1573, 12985, 448), (1904, 5720, 448)])
def test_matmul_a8_forms(hip, rng, M, N, K, epilogue):
    say(f"matmul_a8 M={M} N={N} K={K} epilogue={epilogue} forms")
    x, sx, q, sw, y = matmul_inputs(rng, M, N, K, epilogue)
    got = run_matmul(hip, x, sx, q, sw, y, epilogue, pad=3)
    want, tol = matmul_ref(x, sx, q, sw, y, epilogue)
    assert (np.abs(got - want) <= tol * 1.0001 + 1e-37).all()


@pytest.mark.parametrize("K", [64, 128, 192, 256, 320, 448, 512, 576, 1024, 1088])
@pytest.mark.parametrize("M,epilogue", [(600, STORE), (1500, SWIGLU)])
def test_matmul_a8_tiles_of_few_blocks(hip, rng, M, K, epilogue):
    """Fewer blocks of K than the rings of either tile hold, as many, and more."""
    say(f"matmul_a8 M={M} K={K} rings")
    x, sx, q, sw, y = matmul_inputs(rng, M, 5003, K, epilogue)
    got = run_matmul(hip, x, sx, q, sw, y, epilogue)
    want, tol = matmul_ref(x, sx, q, sw, y, epilogue)
    assert (np.abs(got - want) <= tol * 1.0001 + 1e-37).all()


@pytest.mark.parametrize("rows,n", [(1100, 1100), (1024, 2560), (1030, 3001), (1500, 4095),
                                    (2100, 700), (2100, 200), (1023, 2560)])
def test_norm_q8_many_rows(hip, rng, rows, n):
    say(f"norm_q8 rows={rows} n={n}")
    x = rng.standard_normal((rows, n)).astype(np.float32)
    d = rng.standard_normal((rows, n)).astype(np.float32)
    w = (rng.standard_normal(n) * 0.1).astype(np.float32)
    check_norm(run_norm(hip, x, d, w, pad=3), norm_ref(x, d, w, 1e-6))
    check_norm(run_norm(hip, x, None, w), norm_ref(x, None, w, 1e-6))


def put(hip, p, a):
    hip.check(hip.lib().qlm_memcpy_h2d(p, a.ctypes.data, a.nbytes, None))
    hip.sync()


def get(hip, p, shape, dtype):
    out = np.empty(shape, dtype)
    hip.check(hip.lib().qlm_memcpy_d2h(out.ctypes.data, p, out.nbytes, None))
    hip.sync()
    return out


@pytest.mark.parametrize("M", [520, 700])
def test_matmul_a8_offsets_past_32_bits(hip, rng, M):
    """The last row of x lies 4 GB behind the first, that of y 8 GB."""
    N, K, ldx, ldy = 16 if M < 600 else 9000, 128, (1 << 23) - 16, 1 << 22
    say(f"matmul_a8 M={M} N={N} far rows")
    x, sx, q, sw, y = matmul_inputs(rng, 2, N, K, STORE)
    scales = np.ones(M, np.float32)
    scales[[0, M - 1]] = sx
    dx, dy = hip.DeviceBuffer((M - 1) * ldx + K), hip.DeviceBuffer(4 * ((M - 1) * ldy + N))
    for i, r in enumerate((0, M - 1)):
        put(hip, dx.ptr + r * ldx, x[i])
    nb = hip.lib().qlm_matmul_a8_workspace_bytes(M, N, K, STORE)
    work = hip.DeviceBuffer(nb)
    hip.call("qlm_matmul_a8", dx, ldx, buf(hip, scales), tiles_of(hip, q, 1), buf(hip, sw), dy,
             ldy, M, N, K, STORE, work if nb else None, nb, None)
    got = np.stack([get(hip, dy.ptr + 4 * r * ldy, N, np.float32) for r in (0, M - 1)])
    want, tol = matmul_ref(x, sx, q, sw, y, STORE)
    assert (np.abs(got - want) <= tol * 1.0001 + 1e-37).all()


def test_norm_q8_offsets_past_32_bits(hip, rng):
    rows, n, ld = 3, 300, 1 << 30
    say("norm_q8 far rows")
    x = rng.standard_normal((rows, n)).astype(np.float32)
    w = rng.uniform(-0.5, 0.5, n).astype(np.float32)
    dx, dq = hip.DeviceBuffer(4 * (2 * ld + n)), hip.DeviceBuffer(2 * ld + n)
    dsc = hip.DeviceBuffer(4 * rows)
    for r in range(rows):
        put(hip, dx.ptr + 4 * r * ld, x[r])
    hip.call("qlm_add_rms_norm_q8", dx, ld, None, 0, buf(hip, w), 1e-6, None, 0, dq, ld, dsc, rows,
             n, None)
    got = np.stack([get(hip, dq.ptr + r * ld, n, np.int8) for r in range(rows)])
    check_norm((got, dsc.to_numpy(rows, np.float32), None), norm_ref(x, None, w, 1e-6))


@pytest.mark.parametrize("rows,n,top", [
    (800, 5003, 5), (800, 5003, 20), (800, 5003, 0), (800, 5003, 64), (800, 5003, 25),
    (770, 20001, 24), (767, 20001, 24),  # whole rows, and slices of them
    (256, 16384, 30), (256, 16385, 30), (257, 16384, 30), (1, 4097, 64), (2000, 300, 8),
    (3000, 17, 17), (300, 70001, 64)])
def test_token_logprobs_forms(hip, rng, rows, n, top):
    say(f"logprobs rows={rows} n={n} top={top} forms")
    x = (rng.standard_normal((rows, n)) * rng.uniform(0.5, 6, (rows, 1))).astype(np.float32)
    x[::7, rng.integers(0, n, n // 3)] = -np.inf
    x[3::50] = np.float32(-3.4028235e38)  # all tokens alike, at the type's lowest value
    check_logprobs(hip, x, rng.integers(0, n, (rows, 2)), top)


@pytest.mark.parametrize("n", [300, 20001])
def test_token_logprobs_offsets_past_32_bits(hip, rng, n):
    rows, ldl, top = 3, (1 << 30) + 1, 5
    say(f"logprobs n={n} far rows")
    x = rng.standard_normal((rows, n)).astype(np.float32)
    dl = hip.DeviceBuffer(4 * (2 * ldl + n))
    for r in range(rows):
        put(hip, dl.ptr + 4 * r * ldl, x[r])
    ids = rng.integers(0, n, (rows, 1)).astype(np.int32)
    lp, ti, tl = (hip.DeviceBuffer(4 * rows * m) for m in (1, top, top))
    nb = hip.lib().qlm_token_logprobs_workspace_bytes(rows, n, top)
    hip.call("qlm_token_logprobs", dl, ldl, n, rows, buf(hip, ids), 1, lp, None, top, ti, tl,
             hip.DeviceBuffer(nb), nb, None)
    rlp, _, rti, rtl, (t1, _, t3) = logprobs_ref(x, ids, top)
    assert np.array_equal(ti.to_numpy((rows, top), np.int32), rti)
    assert (np.abs(lp.to_numpy((rows, 1), np.float32) - rlp) <= t1).all()
    assert (np.abs(tl.to_numpy((rows, top), np.float32) - rtl) <= t3).all()


@pytest.mark.parametrize("M", [1, 40, 700])
def test_matmul_a8_results_past_the_range(hip, rng, M):
    """Scales whose product with a sum leaves fp32: infinities as the formula
    has them, and silu(+inf) up = +-inf."""
    N, K = 300, 128
    x = rng.integers(1, 128, (M, K), dtype=np.int8)
    q = rng.integers(1, 128, (2 * N, K), dtype=np.int8)
    q[N + 1::2] *= -1  # up sums of either sign
    sx, sw = np.full(M, 1e20, np.float32), np.full(2 * N, 1e20, np.float32)
    sw[N:] = 1e-24
    say(f"matmul_a8 past the range M={M}")
    y = np.zeros((M, N), np.float32)
    got = run_matmul(hip, x, sx, q, sw, y, SWIGLU)
    assert np.array_equal(got, np.where(np.arange(N) % 2, -np.inf, np.inf) * np.ones((M, 1)))
    got = run_matmul(hip, x, sx, q[:N], sw[:N], y, STORE)
    assert np.isposinf(got).all()


@pytest.mark.parametrize("rows,n,top", [(3, 20001, 20), (2, 300001, 64), (1, 1 << 21, 20),
                                        (2, 40000, 1), (780, 20001, 24), (20, 9000, 64)])
@pytest.mark.parametrize("kind", ["whole", "few", "mixed"])
def test_token_logprobs_ties_over_many_chunks(hip, rng, rows, n, top, kind):
    """Whole numbers, most chunks' maxima the same; few values over a constant,
    or over a mask, fewer than asked for in some rows; all three in turn."""
    say(f"logprobs rows={rows} n={n} top={top} ties {kind}")
    x = rng.integers(-3, 4, (rows, n)).astype(np.float32)
    for r in range(rows):
        if kind == "few" or (kind == "mixed" and r % 2 == 0):
            x[r] = -np.inf if r % 3 == 0 else 1.0
            some = rng.integers(0, n, top // 2 + (r % 2) * top)
            x[r, some] = rng.standard_normal(some.size) + 3
        if kind == "mixed":
            x[r, :300] = -np.inf
    check_logprobs(hip, x, rng.integers(0, n, (rows, 1)), top)


@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 4, 2 ** 31 - 5])
def test_norm_q8_longest_rows(hip, n):
    """One row of up to 2^31 - 1 values, zero but for a few far apart; the gain
    is the row itself, so t = r (1 + r). Each value is a whole number, so sums
    and quotients are those of the definition."""
    say(f"norm_q8 n={n}")
    at = np.array([0, 5, 300, 70001, (1 << 30) + 7, n - 6, n - 3, n - 2, n - 1])
    r = np.float64([3, -2, 5, 1, -6, 4, 2, -4, 6])
    dx, dq, dsc = hip.DeviceBuffer(4 * n), hip.DeviceBuffer(n + 1), hip.DeviceBuffer(4)
    dx.zero()
    hip.call("qlm_fill_u8", dq, 99, n + 1, None)
    for i, v in zip(at, r.astype(np.float32)):
        put(hip, dx.ptr + 4 * int(i), np.array([v]))
    hip.call("qlm_add_rms_norm_q8", dx, n, None, 0, dx, 1e-6, None, 0, dq, n, dsc, 1, n, None)
    q = dq.to_numpy(n + 1, np.int8)
    t = r * (1 + r)
    top = np.abs(t).max()
    scale = top / 127 / np.sqrt((r * r).sum() / n + np.float64(np.float32(1e-6)))
    assert q[n] == 99
    assert np.array_equal(q[at], np.rint(127 * t / top).astype(np.int8))
    q[at] = 0
    assert not q[:n].any()
    assert abs(dsc.to_numpy(1, np.float32)[0] - scale) <= 2.0 ** -24 * scale * (1 + 1e-6)
