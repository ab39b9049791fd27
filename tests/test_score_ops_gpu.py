"""The 8-bit norm, the 8-bit matrix product and the token log probabilities
against their definitions in 64 bits. Tolerances count fp32 roundings (U, half
a step) and are derived where they stand."""

import ctypes as C

import numpy as np
import pytest

from tests.util import say

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # the largest relative error of one fp32 rounding
STORE, RESIDUAL, SWIGLU = 0, 1, 2


def buf(hip, a):
    return hip.DeviceBuffer.from_numpy(a)


# ---- norm ------------------------------------------------------------------------


def norm_ref(x, delta, w, eps):
    """(q, scale, sum): the sum in fp32 as it is stored, the rest in 64 bits."""
    r32 = x if delta is None else (x + delta).astype(np.float32)
    r = r32.astype(np.float64)
    t = r * (1.0 + w.astype(np.float64))
    top = np.abs(t).max(axis=1)
    rms = np.sqrt((r * r).mean(axis=1) + np.float64(np.float32(eps)))
    scale = np.where(top > 0, top / 127 / rms, 1.0)
    q = np.rint(t * 127.0 / np.where(top > 0, top, 1.0)[:, None])
    return q.astype(np.int8), scale, r32


def run_norm(hip, x, delta, w, eps=1e-6, pad=0, in_place=None, keep_sum=True):
    """in_place: None (a buffer of its own), "x" or "delta"."""
    rows, n = x.shape
    ld = n + pad

    def wide(a, fill):
        out = np.full((rows, ld), fill, a.dtype)
        out[:, :n] = a
        return out

    dx, dw = buf(hip, wide(x, 7.0)), buf(hip, w)
    dd = buf(hip, wide(delta, 7.0)) if delta is not None else None
    ds = None
    if delta is not None and keep_sum:
        ds = {"x": dx, "delta": dd}.get(in_place) or buf(hip, np.full((rows, ld), 7.0, np.float32))
    dq = buf(hip, np.full((rows + 1, ld), 99, np.int8))
    dsc = buf(hip, np.full(rows + 1, 5.0, np.float32))
    hip.call("qlm_add_rms_norm_q8", dx, ld, dd, ld, dw, eps, ds, ld, dq, ld, dsc, rows, n, None)
    q, sc = dq.to_numpy((rows + 1, ld), np.int8), dsc.to_numpy(rows + 1, np.float32)
    s = ds.to_numpy((rows, ld), np.float32) if ds else None
    # what lies past the rows and past a row's columns is left as it was
    assert (q[rows] == 99).all() and sc[rows] == 5.0 and (q[:, n:] == 99).all()
    if s is not None:
        assert (s[:, n:] == 7.0).all()
        s = s[:, :n]
    return q[:rows, :n], sc[:rows], s


def check_norm(got, want):
    q, sc, s = got
    qr, scr, sr = want
    assert np.array_equal(q, qr)
    # the scale is computed in 64 bits and rounded to fp32 once
    assert (np.abs(sc - scr) <= U * scr * (1 + 1e-6)).all()
    if s is not None:
        assert np.array_equal(s, sr)


@pytest.mark.parametrize("n", [1, 2, 3, 5, 63, 64, 65, 255, 256, 257, 1001, 1024, 1027, 2560,
                               4096, 4100, 9728, 16384, 16385, 16390, 40000])
@pytest.mark.parametrize("rows,pad", [(1, 0), (7, 5)])
def test_norm_q8(hip, rng, n, rows, pad):
    say(f"norm_q8 rows={rows} n={n} pad={pad}")
    x = rng.standard_normal((rows, n)).astype(np.float32)
    x[:, ::251] *= 20
    d = rng.standard_normal((rows, n)).astype(np.float32)
    w = (rng.standard_normal(n) * 0.1).astype(np.float32)
    check_norm(run_norm(hip, x, d, w, pad=pad), norm_ref(x, d, w, 1e-6))
    check_norm(run_norm(hip, x, None, w, pad=pad), norm_ref(x, None, w, 1e-6))


@pytest.mark.parametrize("in_place", ["x", "delta"])
@pytest.mark.parametrize("n", [100, 2560, 20000])
def test_norm_q8_in_place(hip, rng, n, in_place):
    say(f"norm_q8 in place of {in_place} n={n}")
    x, d = rng.standard_normal((2, 9, n)).astype(np.float32)
    w = rng.standard_normal(n).astype(np.float32)
    want = norm_ref(x, d, w, 1e-6)
    check_norm(run_norm(hip, x, d, w, pad=3, in_place=in_place), want)
    check_norm(run_norm(hip, x, d, w, keep_sum=False), want)


@pytest.mark.parametrize("n", [77, 2560, 17000])
def test_norm_q8_values_at_the_edges(hip, rng, n):
    """Rows of zeros, of one value, of huge and of tiny ones, a single
    non-zero value, and values exactly between two bytes (ties to even)."""
    say(f"norm_q8 edges n={n}")
    x = rng.standard_normal((8, n)).astype(np.float32)
    x[0] = 0.0
    x[1] = -3.0
    x[2] *= np.float32(1e37)  # squares overflow fp32
    x[3] *= np.float32(1e-30)  # squares vanish in fp32: eps rules
    x[4] = 0.0
    x[4, n // 2] = -0.25
    x[5] = (np.arange(n) % 509 - 254) * 0.5  # max 127: every other value a tie
    x[6, 0] = 1e30
    x[7] = np.float32(1e-42)  # denormal
    w = np.zeros(n, np.float32)
    q, sc, _ = got = run_norm(hip, x, None, w)
    want = norm_ref(x, None, w, 1e-6)
    assert np.array_equal(q, want[0])
    # a scale below the normal fp32 range is off by half its spacing, 2^-150
    assert (np.abs(sc - want[1]) <= U * want[1] * (1 + 1e-6) + 2.0 ** -150).all()
    assert sc[0] == 1.0 and not q[0].any()
    assert (q[1] == -127).all()


@pytest.mark.parametrize("n", [64, 2560, 20000])
def test_norm_q8_rows_that_are_not_finite(hip, rng, n):
    """A row with NaN or an infinity gets scale NaN and bytes 0; the rows
    beside it are as ever."""
    say(f"norm_q8 not finite n={n}")
    x = rng.standard_normal((6, n)).astype(np.float32)
    w = rng.standard_normal(n).astype(np.float32)
    want = norm_ref(x, None, w, 1e-6)
    x[1, n - 1], x[3, 0], x[4, n // 2] = np.nan, np.inf, -np.inf
    q, sc, _ = run_norm(hip, x, None, w)
    for r in (1, 3, 4):
        assert np.isnan(sc[r]) and not q[r].any()
    fine = [0, 2, 5]
    check_norm((q[fine], sc[fine], None), (want[0][fine], want[1][fine], None))
    w[n // 3] = np.inf  # a gain reaches every row
    q, sc, _ = run_norm(hip, x, None, w)
    assert np.isnan(sc).all() and not q.any()


# ---- matrix product ---------------------------------------------------------------


def tiles_of(hip, q, halves):
    rows, K = q.shape[0] // halves, q.shape[1]
    qb, sb = C.c_size_t(), C.c_size_t()
    hip.check(hip.lib().qlm_mx_layout_bytes(rows, K, K, halves, C.byref(qb), C.byref(sb)))
    dq, out = buf(hip, q), hip.DeviceBuffer(qb.value)
    hip.call("qlm_mx_swizzle", dq, None, K, rows, K, halves, out, None, None)
    hip.sync()
    return out


def products(x, sx, q, sw):
    """sx sw (x . q): the integer sums exactly, the scaling in 64 bits."""
    acc = x.astype(np.float64) @ q.astype(np.float64).T
    return acc * sx.astype(np.float64)[:, None] * sw.astype(np.float64)


def matmul_ref(x, sx, q, sw, y, epilogue):
    """The result and the error that fp32 roundings may leave: a product has
    three (the sum's, and one a scale), 3 U p."""
    p = products(x, sx, q, sw)
    if epilogue == STORE:
        return p, 3 * U * np.abs(p)
    if epilogue == RESIDUAL:
        return y + p, 3 * U * np.abs(p) + U * np.abs(y + p)
    N = q.shape[0] // 2
    g, u = p[:, :N], p[:, N:]
    out = g / (1 + np.exp(-g)) * u
    # silu: the gate's 3 roundings, carried through exp (times |g|), expf (2
    # steps = 4 U), the sum and the quotient; then the up product's 3 and one
    return out, (3 + 3 * np.abs(g) + 4 + 1 + 1 + 3 + 1) * U * np.abs(out)


def run_matmul(hip, x, sx, q, sw, y, epilogue, ldx=None, pad=0, tiles=None):
    M, K = x.shape
    N = q.shape[0] // (2 if epilogue == SWIGLU else 1)
    ldx = ldx or K
    wide = np.full((M, ldx), 100, np.int8)
    wide[:, :K] = x
    yw = np.full((M + 1, N + pad), 7.0, np.float32)
    yw[:M, :N] = y
    tiles = tiles or tiles_of(hip, q, 2 if epilogue == SWIGLU else 1)
    nb = hip.lib().qlm_matmul_a8_workspace_bytes(M, N, K, epilogue)
    work = buf(hip, np.full(max(nb, 1), 0xA5, np.uint8))
    dx, dsx, dsw, dy = buf(hip, wide), buf(hip, sx), buf(hip, sw), buf(hip, yw)
    hip.call("qlm_matmul_a8", dx, ldx, dsx, tiles, dsw, dy, N + pad, M, N, K, epilogue,
             work if nb else None, nb, None)
    out = dy.to_numpy((M + 1, N + pad), np.float32)
    assert (out[M] == 7.0).all() and (out[:, N:] == 7.0).all()
    return out[:M, :N]


def matmul_inputs(rng, M, N, K, epilogue):
    halves = 2 if epilogue == SWIGLU else 1
    x = rng.integers(-127, 128, (M, K), dtype=np.int8)
    q = rng.integers(-127, 128, (halves * N, K), dtype=np.int8)
    # products of about unit size
    sx = (rng.uniform(0.5, 2, M) / 5400).astype(np.float32)
    sw = (rng.uniform(0.5, 2, halves * N) / np.sqrt(K)).astype(np.float32)
    return x, sx, q, sw, rng.standard_normal((M, N)).astype(np.float32)


@pytest.mark.parametrize("epilogue", [STORE, RESIDUAL, SWIGLU])
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 32, 33, 48, 64, 65, 127, 128, 129, 200, 257, 520])
@pytest.mark.parametrize("N,K", [(1, 64), (16, 128), (37, 192), (131, 704), (300, 2560),
                                 (1040, 320)])
def test_matmul_a8(hip, rng, M, N, K, epilogue):
    say(f"matmul_a8 M={M} N={N} K={K} epilogue={epilogue}")
    x, sx, q, sw, y = matmul_inputs(rng, M, N, K, epilogue)
    got = run_matmul(hip, x, sx, q, sw, y, epilogue)
    want, tol = matmul_ref(x, sx, q, sw, y, epilogue)
    assert (np.abs(got - want) <= tol * 1.0001 + 1e-37).all()


@pytest.mark.parametrize("epilogue", [STORE, RESIDUAL, SWIGLU])
@pytest.mark.parametrize("M,N,K", [(1, 2560, 9728), (16, 2560, 9728), (5, 5003, 1088),
                                   (77, 5003, 1088), (300, 2500, 2560), (700, 1300, 9728),
                                   (1100, 4003, 512)])
def test_matmul_a8_model_sizes(hip, rng, M, N, K, epilogue):
    """Wider than a launch of the smallest form, rows strided on both sides."""
    say(f"matmul_a8 M={M} N={N} K={K} epilogue={epilogue} strided")
    x, sx, q, sw, y = matmul_inputs(rng, M, N, K, epilogue)
    got = run_matmul(hip, x, sx, q, sw, y, epilogue, ldx=K + 48, pad=13)
    want, tol = matmul_ref(x, sx, q, sw, y, epilogue)
    assert (np.abs(got - want) <= tol * 1.0001 + 1e-37).all()


@pytest.mark.parametrize("M", [1, 20, 100, 300])
def test_matmul_a8_largest_sums(hip, M):
    """Every operand -128 at the longest K: the sums end just below 2^31."""
    K, N = 131008, 48
    say(f"matmul_a8 largest sums M={M}")
    x, q = np.full((M, K), -128, np.int8), np.full((N, K), -128, np.int8)
    q[1] = 127
    one = np.ones(max(M, N), np.float32)
    got = run_matmul(hip, x, one[:M], q, one[:N], np.zeros((M, N), np.float32), STORE)
    want = np.full((M, N), np.float32(K * 16384))
    want[:, 1] = np.float32(-128 * 127 * K)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("M", [3, 40, 90, 300])
def test_matmul_a8_scales_that_are_not_finite(hip, rng, M):
    """A row whose scale is NaN comes out NaN, and only that row."""
    x, sx, q, sw, y = matmul_inputs(rng, M, 50, 256, STORE)
    x[M - 1] = 0
    sx[M - 1] = np.nan
    say(f"matmul_a8 NaN scale M={M}")
    got = run_matmul(hip, x, sx, q, sw, y, STORE)
    assert np.isnan(got[M - 1]).all() and np.isfinite(got[:M - 1]).all()


def test_matmul_a8_rows_do_not_depend_on_their_number(hip, rng):
    """A row's result is the same bits in every form (M picks the form)."""
    x, sx, q, sw, y = matmul_inputs(rng, 400, 333, 1024, SWIGLU)
    tiles = tiles_of(hip, q, 2)
    say("matmul_a8 rows alone and together")
    whole = run_matmul(hip, x, sx, q, sw, y, SWIGLU, tiles=tiles)
    for M in (1, 7, 16, 31, 64, 100, 256):
        part = run_matmul(hip, x[:M], sx[:M], q, sw, y[:M], SWIGLU, tiles=tiles)
        assert np.array_equal(part, whole[:M]), M


# ---- log probabilities --------------------------------------------------------------


def logprobs_ref(logits, ids, top):
    """(id_logprobs, entropy, top_ids, top_logprobs, tolerances) in 64 bits.

    Error of log z, in U: a term's exponent is off by at most 2 |d| (the
    difference and its product with log2 e) and exp2 by 2; a lane adds at most
    4 chunks / 4 terms in turn; joining lanes, waves and slices takes at most
    8 + 8 (chunks / 16 + 4) more; the logarithm is off by 4 of its size."""
    rows, n = logits.shape
    l = logits.astype(np.float64)
    with np.errstate(all="ignore"):
        M = l.max(axis=1, keepdims=True)
        d = l - M
        e = np.exp(d)
        z = e.sum(axis=1)
        lsm = d - np.log(z)[:, None]
        lsm[lsm < -3.4028236e38] = -np.inf  # below the fp32 range: rounds to -inf
        ed = np.where(e > 0, e * d, e)
        H = np.log(z) - ed.sum(axis=1) / z
        mean_d = np.abs(ed).sum(axis=1) / z
        chunks = -(-n // 256)
        eps_z = U * (2 * mean_d + 2 + chunks + 4 + 8 + 8 * (chunks / 16 + 4) + 4 * np.log(z))
        # entropy: the log's error, and that of u / z with |u| / z = mean_d
        tol_h = eps_z + mean_d * 2 * eps_z + U * (np.log(z) + 4 * mean_d)
        key = np.where(np.isnan(l), -np.inf, l)
        order = np.argsort(-key, axis=1, kind="stable")[:, :top].astype(np.int32)
        lp = np.full(ids.shape, np.nan)
        dd = np.full(ids.shape, np.nan)
        for r in range(rows):
            for j in range(ids.shape[1]):
                if 0 <= ids[r, j] < n:
                    lp[r, j], dd[r, j] = lsm[r, ids[r, j]], d[r, ids[r, j]]
        tl, td = np.take_along_axis(lsm, order, 1), np.take_along_axis(d, order, 1)
    return lp, H, order, tl, (eps_z[:, None] + U * (np.abs(dd) + np.abs(lp)), tol_h,
                              eps_z[:, None] + U * (np.abs(td) + np.abs(tl)))


def run_logprobs(hip, logits, ids, top, pad=0, entropy=True):
    rows, n = logits.shape
    wide = np.full((rows, n + pad), np.nan, np.float32)  # never to be read
    wide[:, :n] = logits
    k = ids.shape[1]
    dl, di = buf(hip, wide), buf(hip, np.ascontiguousarray(ids, np.int32)) if k else None
    guard = np.full((rows + 1) * max(k, top, 1), 7.0, np.float32)
    dlp, dh, dtl = buf(hip, guard), buf(hip, guard), buf(hip, guard)
    dti = buf(hip, np.full((rows + 1) * max(top, 1), -7, np.int32))
    nb = hip.lib().qlm_token_logprobs_workspace_bytes(rows, n, top)
    work = buf(hip, np.full(nb, 0xA5, np.uint8))
    hip.call("qlm_token_logprobs", dl, n + pad, n, rows, di, k, dlp if k else None,
             dh if entropy else None, top, dti if top else None, dtl if top else None, work, nb,
             None)
    out = []
    for d, m, t, fill in ((dlp, k, np.float32, 7.0), (dh, 1 if entropy else 0, np.float32, 7.0),
                          (dti, top, np.int32, -7), (dtl, top, np.float32, 7.0)):
        a = d.to_numpy((rows + 1) * max(m, 1), t)
        assert (a[rows * m:] == fill).all()
        out.append(a[:rows * m].reshape(rows, m))
    return out


def close(got, want, tol):
    got = got.astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    fine = np.isfinite(want)
    off = np.abs(got[fine] - want[fine])
    assert (off <= np.broadcast_to(tol, want.shape)[fine]).all(), off.max()


def check_logprobs(hip, logits, ids, top, pad=0):
    lp, H, ti, tl = run_logprobs(hip, logits, ids, top, pad)
    rlp, rH, rti, rtl, (t1, t2, t3) = logprobs_ref(logits, ids, top)
    assert np.array_equal(ti, rti)
    close(lp, rlp, t1)
    close(H[:, 0], rH, t2)
    close(tl, rtl, t3)


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 255, 256, 257, 1000, 4096, 5003, 16400, 18433,
                               32003, 151936])
@pytest.mark.parametrize("rows,pad,top,n_ids", [(1, 0, 20, 1), (5, 3, 64, 4), (33, 1, 1, 0),
                                                (9, 0, 0, 8), (2, 0, 5, 300)])
def test_token_logprobs(hip, rng, n, rows, pad, top, n_ids):
    top = min(top, n)
    say(f"logprobs n={n} rows={rows} pad={pad} top={top} ids={n_ids}")
    x = (rng.standard_normal((rows, n)) * rng.uniform(0.5, 6, (rows, 1))).astype(np.float32)
    check_logprobs(hip, x, rng.integers(0, n, (rows, n_ids)), top, pad)


@pytest.mark.parametrize("n", [300, 5003, 70000])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_token_logprobs_order(hip, rng, n, top):
    """Ascending, descending, equal, two-valued and coarse logits, the largest
    in one chunk, and zeros of both signs: ties go to the lower id."""
    say(f"logprobs order n={n} top={top}")
    i = np.arange(n)
    x = np.stack([
        i * 1e-3, -i * 1e-3, np.zeros(n), np.where(i % 7 == 3, 2.0, 1.0),
        np.round(rng.standard_normal(n) * 2), np.where((i >= 256) & (i < 290), 50.0 + i % 5, -1.0),
        np.where(i % 2 == 0, 0.0, -0.0), np.where(i == n - 1, 30.0, -40.0),
        rng.standard_normal(n) * 1e-6, rng.standard_normal(n) * 1e4]).astype(np.float32)
    check_logprobs(hip, x, rng.integers(0, n, (len(x), 3)), top)


@pytest.mark.parametrize("n", [5, 300, 5003, 70000])
@pytest.mark.parametrize("top", [0, 1, 5, 64])
def test_token_logprobs_masks(hip, rng, n, top):
    """Rows with few tokens left, one, none; masked by the type's lowest
    value; with NaN, with +inf, with NaN among nothing but masked ones."""
    top = min(top, n)
    say(f"logprobs masks n={n} top={top}")
    x = (rng.standard_normal((12, n)) * 3).astype(np.float32)
    low = np.finfo(np.float32).min
    x[0, rng.random(n) < 0.9] = -np.inf
    x[1] = -np.inf
    x[1, [n - 1, n // 2, 0]] = [1.0, 1.0, -2.0]
    x[2] = -np.inf
    x[2, n - 1] = -3e38  # one token: probability 1
    x[3] = -np.inf
    x[4, rng.random(n) < 0.9] = low
    x[5] = low  # equal logits, whatever their value
    x[6, n // 3] = np.nan
    x[7, n // 2] = np.inf
    x[8] = -np.inf
    x[8, n - 1] = np.nan
    x[9] = np.nan
    x[10, : n - 1] = -np.inf
    x[11, 0], x[11, 1:] = 3e38, low
    ids = rng.integers(0, n, (12, 4))
    ids[:, 3] = n - 1
    check_logprobs(hip, x, ids, top, pad=2)


def test_token_logprobs_ids_outside_the_row(hip, rng):
    """An id that is no token gets NaN; the ids beside it are as ever."""
    x = rng.standard_normal((3, 400)).astype(np.float32)
    ids = np.array([[-1, 0, 399, 400], [2**31 - 1, 5, 5, -2**31], [399, 1, 401, 2]])
    say("logprobs ids outside")
    check_logprobs(hip, x, ids, 2, pad=5)


def test_token_logprobs_parts_alone(hip, rng):
    """Each output on its own is the same bits as all together."""
    x = (rng.standard_normal((4, 9000)) * 3).astype(np.float32)
    ids = rng.integers(0, 9000, (4, 2))
    say("logprobs parts")
    lp, H, ti, tl = run_logprobs(hip, x, ids, 7)
    assert np.array_equal(run_logprobs(hip, x, ids, 0, entropy=False)[0], lp)
    assert np.array_equal(run_logprobs(hip, x, ids[:, :0], 0)[1], H)
    _, _, ti2, tl2 = run_logprobs(hip, x, ids[:, :0], 7, entropy=False)
    assert np.array_equal(ti, ti2) and np.array_equal(tl, tl2)


# ---- together ------------------------------------------------------------------------


class Scorer:
    """The last layer's MLP and the head of a model scoring T rows: the calls
    in order on one stream, every buffer kept for the stage checks."""

    def __init__(self, hip, rng, T, H, F, V, top):
        self.hip, self.T, self.H, self.F, self.V, self.top = hip, T, H, F, V, top

        def weight(n, k):
            w = (rng.standard_normal((n, k)) * k ** -0.5).astype(np.float32)
            dq, ds = hip.DeviceBuffer(n * k), hip.DeviceBuffer(n * 4)
            hip.call("qlm_quantize_q8_f32", buf(hip, w), n, k, k, dq, ds, None)
            return dq.to_numpy((n, k), np.int8), ds.to_numpy(n, np.float32)

        self.w = {"gate_up": weight(2 * F, H), "down": weight(H, F), "head": weight(V, H)}
        self.x0 = rng.standard_normal((T, H)).astype(np.float32)
        self.d0 = rng.standard_normal((T, H)).astype(np.float32)
        self.n1, self.n2 = (rng.standard_normal((2, H)) * 0.1).astype(np.float32)
        self.ids = rng.integers(0, V, (T, 1)).astype(np.int32)
        up = {k: (tiles_of(hip, q, 2 if k == "gate_up" else 1), buf(hip, s))
              for k, (q, s) in self.w.items()}
        L = hip.lib()
        wb = max(L.qlm_matmul_a8_workspace_bytes(T, F, H, SWIGLU),
                 L.qlm_matmul_a8_workspace_bytes(T, H, F, RESIDUAL),
                 L.qlm_matmul_a8_workspace_bytes(T, V, H, STORE),
                 L.qlm_token_logprobs_workspace_bytes(T, V, top))
        z = lambda n: buf(hip, np.zeros(n, np.uint8))  # noqa: E731
        self.b = dict(x=buf(hip, self.x0), d=buf(hip, self.d0), n1=buf(hip, self.n1),
                      n2=buf(hip, self.n2), ids=buf(hip, self.ids), res=z(T * H * 4),
                      q1=z(T * H), s1=z(T * 4), act=z(T * F * 4), q2=z(T * F), s2=z(T * 4),
                      q3=z(T * H), s3=z(T * 4), logits=z(T * V * 4), lp=z(T * 4), ent=z(T * 4),
                      ti=z(T * top * 4), tl=z(T * top * 4), work=z(max(wb, 1)))
        self.up, self.wb = up, wb
        hip.sync()

    def enqueue(self, st):
        b, T, H, F, V, call = self.b, self.T, self.H, self.F, self.V, self.hip.call
        call("qlm_add_rms_norm_q8", b["x"], H, b["d"], H, b["n1"], 1e-6, b["res"], H, b["q1"], H,
             b["s1"], T, H, st)
        call("qlm_matmul_a8", b["q1"], H, b["s1"], *self.up["gate_up"], b["act"], F, T, F, H,
             SWIGLU, b["work"], self.wb, st)
        call("qlm_quantize_q8_f32", b["act"], T, F, F, b["q2"], b["s2"], st)
        call("qlm_matmul_a8", b["q2"], F, b["s2"], *self.up["down"], b["res"], H, T, H, F,
             RESIDUAL, b["work"], self.wb, st)
        call("qlm_add_rms_norm_q8", b["res"], H, None, 0, b["n2"], 1e-6, None, 0, b["q3"], H,
             b["s3"], T, H, st)
        call("qlm_matmul_a8", b["q3"], H, b["s3"], *self.up["head"], b["logits"], V, T, V, H,
             STORE, b["work"], self.wb, st)
        call("qlm_token_logprobs", b["logits"], V, V, T, b["ids"], 1, b["lp"], b["ent"], self.top,
             b["ti"], b["tl"], b["work"], self.wb, st)

    def get(self, name, *shape, t=np.float32):
        return self.b[name].to_numpy(shape, t)

    def results(self):
        T, k = self.T, self.top
        return [self.get("logits", T, self.V), self.get("lp", T, 1), self.get("ent", T),
                self.get("ti", T, k, t=np.int32), self.get("tl", T, k)]

    def check(self):
        """Every stage against its definition on what the stage before left."""
        T, H, F, V = self.T, self.H, self.F, self.V
        q, s, r = norm_ref(self.x0, self.d0, self.n1, 1e-6)
        q1, s1 = self.get("q1", T, H, t=np.int8), self.get("s1", T)
        check_norm((q1, s1, None), (q, s, None))
        act = self.get("act", T, F)
        want, tol = matmul_ref(q1, s1, *self.w["gate_up"], None, SWIGLU)
        assert (np.abs(act - want) <= tol * 1.0001 + 1e-37).all()
        q2, s2 = self.get("q2", T, F, t=np.int8), self.get("s2", T)
        res = self.get("res", T, H)
        want, tol = matmul_ref(q2, s2, *self.w["down"], r.astype(np.float64), RESIDUAL)
        assert (np.abs(res - want) <= tol * 1.0001).all()
        q3, s3 = self.get("q3", T, H, t=np.int8), self.get("s3", T)
        check_norm((q3, s3, None), norm_ref(res, None, self.n2, 1e-6))
        logits, lp, ent, ti, tl = self.results()
        want, tol = matmul_ref(q3, s3, *self.w["head"], None, STORE)
        assert (np.abs(logits - want) <= tol * 1.0001 + 1e-37).all()
        rlp, rH, rti, rtl, (t1, t2, t3) = logprobs_ref(logits, self.ids, self.top)
        assert np.array_equal(ti, rti)
        close(lp, rlp, t1)
        close(ent, rH, t2)
        close(tl, rtl, t3)


@pytest.mark.parametrize("T", [1, 19, 150])
def test_scoring_a_prompt(hip, rng, T):
    say(f"scoring T={T}")
    s = Scorer(hip, rng, T, 512, 1088, 3001, 5)
    s.enqueue(None)
    hip.sync()
    s.check()


@pytest.mark.parametrize("T", [1, 33, 130])
def test_scoring_in_a_captured_graph(hip, rng, T):
    """Captured once and replayed, with eager calls between the replays: each
    replay leaves the eager call's bits, also on inputs changed in place."""
    hip.check(hip.lib().qlm_set_device(0))
    L, s, st = hip.lib(), Scorer(hip, rng, T, 320, 704, 2003, 3), hip.Stream()
    say(f"scoring graph T={T}")
    s.enqueue(None)
    hip.sync()
    want = s.results()
    g = C.c_void_p()
    hip.check(L.qlm_graph_begin(st.ptr))
    s.enqueue(st.ptr)
    hip.check(L.qlm_graph_end(st.ptr, C.byref(g)))
    try:
        for rep in range(3):
            for k in ("res", "logits", "lp", "ent", "tl"):
                s.b[k].zero()
            hip.sync()
            hip.check(L.qlm_graph_launch(g, st.ptr))
            st.sync()
            for a, b in zip(s.results(), want):
                assert np.array_equal(a, b), rep
            s.b["work"].zero()
            s.x0 = rng.standard_normal(s.x0.shape).astype(np.float32)
            s.b["x"].upload(s.x0)
            s.enqueue(None)
            hip.sync()
            want = s.results()
        s.check()
    finally:
        hip.check(L.qlm_graph_destroy(g))


def test_scoring_on_two_streams(hip, rng):
    """Two scorers with buffers of their own, their calls alternating between
    two streams without a wait, give what each gives alone."""
    a, b = Scorer(hip, rng, 70, 512, 640, 4001, 4), Scorer(hip, rng, 3, 512, 640, 4001, 4)
    say("scoring on two streams")
    want = []
    for s in (a, b):
        s.enqueue(None)
        hip.sync()
        want.append(s.results())
    s1, s2 = hip.Stream(), hip.Stream()
    for _ in range(4):
        a.enqueue(s1.ptr)
        b.enqueue(s2.ptr)
    s1.sync()
    s2.sync()
    for s, w in zip((a, b), want):
        for x, y in zip(s.results(), w):
            assert np.array_equal(x, y)
