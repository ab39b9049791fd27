"""The paged append, the paged attention, the tree commit and the DeltaNet mixer
over trees against their definitions in 64 bits. Tolerances count fp32 roundings
(U, half a step) and bf16 ones (half a step: 2^-8), and are derived where they
stand."""

import ctypes as C

import numpy as np
import pytest

from tests.tree_util import (TREE, Pages, Rows, attention_ref, attention_tol, deltanet_ref, lines,
                             random_tree, rope_ref)
from tests.util import bf16_bits, bf16_to_f32, say

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FILL = 7.5


def buf(hip, a):
    return hip.DeviceBuffer.from_numpy(a)


def tables(n_pos, half):
    """cos and sin of every position, fp32 [n_pos, half]."""
    a = np.arange(n_pos)[:, None] * 1e4 ** (-np.arange(half) / max(half, 1))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


# ---- append ----------------------------------------------------------------------


def run_append(hip, rng, rows, pages, n_q, gated, rot, axes=0, norm=True, pad=0, n_pos=400,
               shift=0):
    """q_out, the pools after the call, and the inputs. shift: floats that the
    arrays begin past a 16-byte border."""
    hd, n_kv = pages.hd, pages.n_kv
    ld, ldq = n_q * hd * (2 if gated else 1) + 2 * n_kv * hd + pad, n_q * hd + pad
    x = rng.standard_normal((rows.rows, ld)).astype(np.float32)
    qn, kn = (rng.standard_normal(hd).astype(np.float32) * 0.3 for _ in range(2))
    cos, sin = tables(n_pos, rot // 2)
    pos = rng.integers(0, n_pos, (max(axes, 1), rows.rows)).astype(np.int32)
    axis = rng.integers(0, max(axes, 1), max(rot // 2, 1)).astype(np.int32)

    def at(a):
        flat = np.concatenate([np.zeros(shift, a.dtype), a.ravel()])
        d = buf(hip, flat)
        return d, d.ptr + 4 * shift

    dx, px = at(x)
    dq, pq = at(np.full((rows.rows, ldq), FILL, np.float32))
    dn = [at(a) for a in (qn, kn, cos, sin)]
    dp = [buf(hip, a) for a in (pos, axis)]
    hip.call("qlm_paged_append", px, ld, dn[0][1] if norm else None, dn[1][1] if norm else None,
             dn[2][1], dn[3][1], n_pos, rot, dp[0].ptr if axes else None, rows.rows,
             dp[1].ptr if axes > 1 else None, axes, rows.c, pages.c, pq, ldq, n_q, int(gated), None)
    got = dq.to_numpy(shift + rows.rows * ldq, np.float32)[shift:].reshape(rows.rows, ldq)
    return got, pages.download(), dict(x=x, qn=qn if norm else None, kn=kn if norm else None,
                                       cos=cos, sin=sin, pos=pos if axes else None,
                                       axis=axis if axes > 1 else None)


def check_append(rows, pages, got, pools, inp, n_q, gated, rot):
    """Every output within its roundings, everything else as it was. A head's
    sum of squares is off by 4 + 6 roundings at most, so its root's reciprocal by
    5 and the mean's, the addition's, the root's and the quotient's 4; the two
    products and the gain's sum 3; a rotated pair's products and sum 3 more: 16
    with one to spare, of the terms' absolute sum."""
    hd, n_kv, half = pages.hd, pages.n_kv, rot // 2
    x = inp["x"].astype(np.float64)
    head = hd * (2 if gated else 1)

    def head_ref(v, gain, where):
        if gain is not None:
            v = v / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-6) * (1 + gain.astype(np.float64))
        if not half:
            return v, np.abs(v)
        top = np.abs(v).copy()
        top[..., :half] += np.abs(v[..., half:2 * half])
        top[..., half:2 * half] += np.abs(v[..., :half])
        return rope_ref(v, where, half, inp["cos"], inp["sin"]), top

    want_k, want_v = pages.k.copy(), pages.v.copy()
    seen = np.zeros(rows.rows, bool)
    for b, first, n, ctx, ls in rows.seqs():
        for i in range(n):
            r = first + i
            seen[r] = True
            live = ls[i] is not None
            if inp["pos"] is not None:
                ax = inp["axis"] if inp["axis"] is not None else np.zeros(max(half, 1), int)
                where = inp["pos"][ax[:half], r]
            else:
                where = np.full(half, ctx + (len(ls[i]) - 1 if live else 0))
            q = x[r, :n_q * head].reshape(n_q, head)[:, :hd]
            k = x[r, n_q * head:n_q * head + n_kv * hd].reshape(n_kv, hd)
            v = x[r, n_q * head + n_kv * hd:][:n_kv * hd].reshape(n_kv, hd)
            o = got[r, :n_q * hd].reshape(n_q, hd)
            if not live:
                assert (o == 0).all()
                continue
            want, top = head_ref(q, inp["qn"], where)
            assert (np.abs(o - want) <= 16 * U * top).all(), r
            if ctx + i >= pages.ld * pages.page:
                continue
            p, at = pages.at(b, ctx + i)
            if not 0 <= p < pages.n_pages:
                continue
            want, top = head_ref(k, inp["kn"], where)
            tol = 16 * U * top + (2.0 ** -8 * np.abs(want) * (1 + 1e-4) if pages.bf16 else 0)
            assert (np.abs(pools[0][0, p, :, at] - want) <= tol).all(), r
            stored = bf16_to_f32(bf16_bits(v.astype(np.float32))) if pages.bf16 else v
            assert np.array_equal(pools[1][0, p, :, at], stored.astype(np.float32))
            want_k[0, p, :, at] = pools[0][0, p, :, at]
            want_v[0, p, :, at] = pools[1][0, p, :, at]
    assert (got[~seen] == FILL).all() and (got[:, n_q * hd:] == FILL).all()
    assert np.array_equal(pools[0], want_k, equal_nan=True)
    assert np.array_equal(pools[1], want_v, equal_nan=True)


@pytest.mark.parametrize("hd,bf16", [(128, True), (128, False), (256, True), (256, False)])
@pytest.mark.parametrize("n_q,n_kv,gated,rot,axes,norm", [
    (4, 1, True, 32, 0, True), (2, 2, False, 34, 3, True), (8, 2, True, 2, 1, False),
    (3, 3, False, 0, 0, True), (7, 1, True, 128, 2, True)])
def test_append(hip, rng, hd, bf16, n_q, n_kv, gated, rot, axes, norm):
    say(f"append hd={hd} bf16={bf16} n_q={n_q} n_kv={n_kv} rot={rot} axes={axes}")
    n, ctx = [3, 0, 1, 7, 18], [0, 5, 16, 31, 9]
    rows = Rows(hip, n, ctx, before=2, behind=3)
    pages = Pages(hip, rng, [a + c for a, c in zip(n, ctx)], n_kv, hd, 16, bf16, filled=ctx)
    got, pools, inp = run_append(hip, rng, rows, pages, n_q, gated, rot, axes, norm,
                                 pad=5 if gated else 0, shift=1 if gated else 0)
    check_append(rows, pages, got, pools, inp, n_q, gated, rot)


@pytest.mark.parametrize("axes", [4, 5, 9])
def test_append_many_axes(hip, rng, axes):
    say(f"append axes={axes}")
    rows = Rows(hip, [5, 2], [3, 40])
    pages = Pages(hip, rng, [8, 42], 1, 128, 16, True, filled=[3, 40])
    got, pools, inp = run_append(hip, rng, rows, pages, 2, False, 64, axes)
    check_append(rows, pages, got, pools, inp, 2, False, 64)


@pytest.mark.parametrize("page", [16, 64, 256])
def test_append_trees(hip, rng, page):
    """Positions are the context and the depth; rows outside the tree (padding,
    below padding, below a later row, past the 64th) leave no trace."""
    say(f"append trees page={page}")
    n, ctx = [64, 1, 20, 70], [250, 0, 15, 3]
    parents = [random_tree(rng, 64, padding=3), [-1], random_tree(rng, 20), random_tree(rng, 70)]
    parents[2][5] = 5
    parents[2][9] = 12
    parents[2][11] = -7
    parents[2][13] = 9
    rows = Rows(hip, n, ctx, parents, before=1, behind=2)
    pages = Pages(hip, rng, [a + c for a, c in zip(n, ctx)], 2, 128, page, True, filled=ctx)
    got, pools, inp = run_append(hip, rng, rows, pages, 4, True, 32)
    check_append(rows, pages, got, pools, inp, 4, True, 32)


def test_append_slots_that_are_not_there(hip, rng):
    """Page numbers out of range and slots past the table are not written."""
    say("append bad pages")
    n, ctx = [20, 20, 40], [10, 10, 0]
    rows = Rows(hip, n, ctx)
    pages = Pages(hip, rng, [30, 30, 30], 2, 128, 16, True, filled=ctx)
    pages.table[0, 1] = pages.n_pages
    pages.table[1, 0] = -5
    pages.table[2, 1] = 2 ** 31 - 1
    pages.upload(hip)
    got, pools, inp = run_append(hip, rng, rows, pages, 2, False, 64)
    check_append(rows, pages, got, pools, inp, 2, False, 64)


def test_append_positions_without_an_angle(hip, rng):
    """A position outside the table, or an axis that is not there: NaN in its
    pairs alone."""
    say("append bad positions")
    rows = Rows(hip, [4], [0])
    pages = Pages(hip, rng, [4], 1, 128, 16, False, filled=[0])
    cos, sin = tables(10, 16)
    x = rng.standard_normal((4, 128 + 256)).astype(np.float32)
    pos = np.array([[0, 10, 3, 3], [1, 1, -1, 3]], np.int32)
    axis = np.arange(16, dtype=np.int32) % 2
    axis[15] = 2
    d = [buf(hip, a) for a in (x, cos, sin, pos, axis, np.zeros((4, 128), np.float32))]
    hip.call("qlm_paged_append", d[0], 384, None, None, d[1], d[2], 10, 32, d[3], 4, d[4], 2,
             rows.c, pages.c, d[5], 128, 1, 0, None)
    q = d[5].to_numpy((4, 128), np.float32)
    bad = np.zeros((4, 128), bool)
    bad[:, [15, 31]] = True
    bad[1, :32:2] = True  # axis 0
    bad[2, 1:32:2] = True
    assert np.array_equal(np.isnan(q), bad)
    assert np.array_equal(np.isnan(pages.download()[0][0, pages.table[0, 0], 0, :4]), bad)


# ---- attention -------------------------------------------------------------------


def run_attention(hip, rng, rows, pages, n_q, gated=False, pad=0, q=None, qscale=1.0):
    hd = pages.hd
    if q is None:
        q = (rng.standard_normal((rows.rows, n_q * hd + pad)) * qscale).astype(np.float32)
    g = rng.standard_normal((rows.rows, n_q * 2 * hd)).astype(np.float32) if gated else None
    ld = q.shape[1]
    dq, do = buf(hip, q), buf(hip, np.full((rows.rows, ld), FILL, np.float32))
    dg = buf(hip, g) if gated else None
    n = hip.lib().qlm_paged_attention_workspace_bytes(rows.rows, len(rows.n), n_q, pages.n_kv, hd,
                                                      pages.ld * pages.page)
    work = buf(hip, np.full(max(n, 16), 0xff, np.uint8))  # NaN and -1 throughout
    hip.call("qlm_paged_attention", dq, ld, rows.c, pages.c, dg.ptr + 4 * hd if gated else None,
             n_q * 2 * hd if gated else 0, 2 * hd, do, ld, n_q, work, n, None)
    gate = None
    if gated:
        gate = g.reshape(rows.rows, n_q, 2, hd)[:, :, 1].reshape(rows.rows, n_q * hd)
    return do.to_numpy((rows.rows, ld), np.float32), q, gate


def check_attention(rows, pages, got, q, gate, n_q):
    hd = pages.hd
    ref = attention_ref(rows, pages, q, n_q, gate)
    worst = 0.0
    for r, (o, pv, qk, keys) in ref.items():
        x = got[r, :n_q * hd].reshape(n_q, hd)
        if keys == 0:
            assert (x == 0).all(), r
            continue
        err, tol = np.abs(x - o), attention_tol(pv, qk, keys, not pages.bf16)
        assert (err <= tol).all(), (r, float((err / tol).max()))
        worst = max(worst, float((err / tol).max()))
    seen = np.zeros(rows.rows, bool)
    seen[list(ref)] = True
    assert (got[~seen] == FILL).all() and (got[:, n_q * hd:] == FILL).all()
    say(f"  worst error / bound {worst:.3f}")


SHAPES = [(1, 1), (4, 2), (16, 4), (8, 1)]  # G = 1, 2, 4, 8


@pytest.mark.parametrize("hd,bf16", [(128, True), (128, False), (256, True), (256, False)])
@pytest.mark.parametrize("n_q,n_kv", SHAPES)
def test_attention_single_tokens(hip, rng, hd, bf16, n_q, n_kv):
    say(f"attention decode hd={hd} bf16={bf16} {n_q}/{n_kv}")
    ctx = [0, 1, 15, 16, 17, 31, 63, 127, 128, 300, 1000]
    rows = Rows(hip, [1] * len(ctx), ctx, behind=1)
    pages = Pages(hip, rng, [c + 1 for c in ctx], n_kv, hd, 16, bf16)
    check_attention(rows, pages, *run_attention(hip, rng, rows, pages, n_q, gated=True), n_q)


@pytest.mark.parametrize("page", [16, 32, 128, 256])
@pytest.mark.parametrize("ctx", [700, 2500])
def test_attention_one_long_context(hip, rng, page, ctx):
    """Few rows: the keys are split over workgroups and joined."""
    say(f"attention page={page} ctx={ctx}")
    rows = Rows(hip, [1], [ctx])
    pages = Pages(hip, rng, [ctx + 1], 2, 128, page, True)
    check_attention(rows, pages, *run_attention(hip, rng, rows, pages, 8, qscale=3.0), 8)


@pytest.mark.parametrize("hd,bf16", [(128, True), (128, False), (256, True), (256, False)])
@pytest.mark.parametrize("n_q,n_kv,nodes", [(1, 1, 11), (2, 2, 64), (4, 1, 3), (8, 2, 16), (8, 2, 40),
                                            (16, 2, 64)])
def test_attention_trees(hip, rng, hd, bf16, n_q, n_kv, nodes):
    say(f"attention trees hd={hd} bf16={bf16} {n_q}/{n_kv} nodes={nodes}")
    n, ctx = [nodes, 0, 1, nodes], [0, 7, 40, 333]
    parents = [random_tree(rng, nodes), [], [-1], random_tree(rng, nodes, padding=nodes // 8)]
    rows = Rows(hip, n, ctx, parents, before=1, behind=2)
    pages = Pages(hip, rng, [a + c for a, c in zip(n, ctx)], n_kv, hd, 32, bf16)
    check_attention(rows, pages, *run_attention(hip, rng, rows, pages, n_q, gated=True, pad=3), n_q)


@pytest.mark.parametrize("hd,bf16", [(128, True), (128, False), (256, True), (256, False)])
@pytest.mark.parametrize("n_q,n_kv,n,ctx", [
    (2, 2, [65, 200], [0, 100]), (4, 1, [33, 1, 0, 70], [0, 500, 9, 31]), (8, 1, [150], [257])])
def test_attention_prompts(hip, rng, hd, bf16, n_q, n_kv, n, ctx):
    say(f"attention prompts hd={hd} bf16={bf16} {n_q}/{n_kv} n={n} ctx={ctx}")
    rows = Rows(hip, n, ctx, behind=1)
    pages = Pages(hip, rng, [a + c for a, c in zip(n, ctx)], n_kv, hd, 64, bf16)
    check_attention(rows, pages, *run_attention(hip, rng, rows, pages, n_q), n_q)


def test_attention_more_rows_than_a_tree_has(hip, rng):
    """Rows past the 64th, under rows outside the tree, or under later rows."""
    say("attention odd trees")
    parents = [random_tree(rng, 80), random_tree(rng, 30)]
    parents[1][3], parents[1][4], parents[1][10], parents[1][12] = -2, 4, 20, 3
    parents[1][0] = -3 if parents[1][1] else -2
    parents[1][1] = -1
    rows = Rows(hip, [80, 30], [50, 5], parents)
    pages = Pages(hip, rng, [130, 35], 1, 128, 16, True)
    check_attention(rows, pages, *run_attention(hip, rng, rows, pages, 4, gated=True), 4)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("n,n_q", [([1, 1], 4), ([12, 12], 4), ([40, 70], 4)])
def test_attention_slots_that_are_not_there(hip, rng, bf16, n, n_q):
    """Page numbers out of range hide their keys; contexts past the table end
    with it; a row without any key gives 0."""
    say(f"attention bad pages n={n} bf16={bf16}")
    rows = Rows(hip, n, [60, 500])
    pages = Pages(hip, rng, [60 + n[0], 96], 2, 128, 16, bf16)  # (whole pages: all are seen)
    pages.table[0, 1], pages.table[0, 3] = pages.n_pages, -1
    pages.table[1, :3] = [-9, 2 ** 31 - 1, -2 ** 31]
    pages.upload(hip)
    check_attention(rows, pages, *run_attention(hip, rng, rows, pages, n_q), n_q)
    pages.table[1, :] = -1
    pages.upload(hip)
    got = run_attention(hip, rng, rows, pages, n_q)
    check_attention(rows, pages, *got, n_q)
    assert (got[0][n[0]:n[0] + n[1], :n_q * 128] == 0).all()


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("nodes,n_q", [(4, 2), (14, 2), (30, 4)])
def test_attention_other_branches_values(hip, rng, bf16, what, nodes, n_q):
    """NaN and infinities in keys and values that a row does not see leave its
    result alone; a row that sees one in its values has it."""
    say(f"attention {what} in a branch nodes={nodes} bf16={bf16}")
    parents = [[-1] + [0 if i % 2 else i - 1 for i in range(1, nodes)]]
    ctx = 90
    rows = Rows(hip, [nodes], [ctx], parents)
    pages = Pages(hip, rng, [ctx + nodes], 2, 128, 16, bf16)
    sick = 3  # row 3 is seen by itself and by row 4
    p, at = pages.at(0, ctx + sick) if nodes > sick else pages.at(0, ctx)
    clean_k, clean_v = pages.k.copy(), pages.v.copy()
    pages.k[0, p, :, at, 5], pages.v[0, p, :, at, 7] = what, what
    pages.upload(hip)
    got, q, gate = run_attention(hip, rng, rows, pages, n_q)
    ref = attention_ref(rows, pages, q, n_q, k=clean_k, v=clean_v)
    for r, (o, pv, qk, keys) in ref.items():
        x = got[r].reshape(n_q, 128)
        if r in (3, 4):
            # the key's score is infinite or NaN, and so is the value: nothing
            # finite may come out unless the score is -inf, which hides both
            for h in range(n_q):
                low = np.isinf(what) and np.sign(q[r, h * 128 + 5]) * what < 0
                if not low:
                    assert not np.isfinite(x[h, 7])
                else:
                    assert np.isfinite(x[h]).all()
            continue
        assert (np.abs(x - o) <= attention_tol(pv, qk, keys, not bf16)).all(), r


def test_attention_causal_rows_ignore_later_values(hip, rng):
    say("attention NaN behind a row")
    rows = Rows(hip, [100], [20])
    pages = Pages(hip, rng, [120], 1, 128, 16, True)
    clean = pages.v.copy()
    p, at = pages.at(0, 20 + 60)
    pages.v[0, p, 0, at] = np.nan
    pages.upload(hip)
    got, q, _ = run_attention(hip, rng, rows, pages, 2)
    ref = attention_ref(rows, pages, q, 2, v=clean)
    for r in range(60):
        o, pv, qk, keys = ref[r]
        assert (np.abs(got[r].reshape(2, 128) - o) <= attention_tol(pv, qk, keys, False)).all(), r
    assert np.isnan(got[60:]).all()


@pytest.mark.parametrize("scale", [1e-30, 100.0, 3e37])
def test_attention_query_sizes(hip, rng, scale):
    """Scores from none to far past exp's range: one key takes all."""
    say(f"attention queries of {scale}")
    rows = Rows(hip, [1, 1], [50, 300])
    pages = Pages(hip, rng, [51, 301], 1, 128, 16, False)
    pages.k *= 1e-3 if scale > 1e30 else 1.0
    pages.upload(hip)
    got, q, gate = run_attention(hip, rng, rows, pages, 2, qscale=scale)
    if scale < 1e30:
        check_attention(rows, pages, got, q, gate, 2)
        return
    for r, (o, pv, qk, keys) in attention_ref(rows, pages, q, 2).items():
        assert np.abs(got[r].reshape(2, 128) - o).max() <= 2.0 ** -16 * np.abs(o).max()


@pytest.mark.parametrize("B", [65, 200])
def test_attention_many_sequences(hip, rng, B):
    """More sequences than a wave has lanes, some without rows."""
    say(f"attention B={B}")
    n = [int(x) for x in rng.integers(0, 3, B)]
    ctx = [int(x) for x in rng.integers(0, 120, B)]
    rows = Rows(hip, n, ctx, behind=1)
    pages = Pages(hip, rng, [a + c for a, c in zip(n, ctx)], 1, 128, 16, True)
    check_attention(rows, pages, *run_attention(hip, rng, rows, pages, 4), 4)


def test_attention_far_pages(hip, rng):
    """Pages past 2^32 bytes and 2^31 elements of a pool."""
    say("attention far pages")
    hd, page, n_kv, ctx = 128, 256, 8, 600
    n_pages = (5 << 30) // (n_kv * page * hd * 2)
    slots = [n_pages - 1, 1, n_pages - 2]
    rows = Rows(hip, [2], [ctx])
    dk, dv = hip.DeviceBuffer(5 << 30), hip.DeviceBuffer(5 << 30)
    size = n_kv * page * hd * 2
    k, v = (bf16_bits(rng.standard_normal((3, n_kv, page, hd)).astype(np.float32))
            for _ in range(2))
    for i, p in enumerate(slots):
        for d, a in ((dk, k), (dv, v)):
            one = np.ascontiguousarray(a[i])
            hip.check(hip.lib().qlm_memcpy_h2d(d.ptr + p * size, one.ctypes.data, size, None))
            hip.sync()
    table = buf(hip, np.array([slots], np.int32))
    small = Pages.__new__(Pages)
    small.page, small.n_kv, small.hd, small.bf16, small.ld, small.n_pages = page, n_kv, hd, True, 3, 3
    small.table = np.array([[0, 1, 2]])
    small.k, small.v = bf16_to_f32(k)[None], bf16_to_f32(v)[None]
    small.c = hip.KvPages(dk.ptr, dv.ptr, 1, n_pages, page, n_kv, hd, table.ptr, 3)
    check_attention(rows, small, *run_attention(hip, rng, rows, small, 16), 16)


def test_attention_of_one_batch_is_repeatable(hip, rng):
    say("attention twice")
    rows = Rows(hip, [1] * 8, [1500] * 8)
    pages = Pages(hip, rng, [1501] * 8, 2, 128, 64, True)
    a, q, _ = run_attention(hip, rng, rows, pages, 8)
    b, _, _ = run_attention(hip, rng, rows, pages, 8, q=q)
    assert np.array_equal(a, b)


@pytest.mark.parametrize("bf16", [True, False])
def test_attention_many_rows_and_heads(hip, rng, bf16):
    """More tasks than the joining launch has waves, of three kv heads. The
    oracle takes a copy that has all but a few rows' queries left out."""
    say(f"attention many rows bf16={bf16}")
    n, ctx, n_q = [300, 1, 500], [40, 200, 0], 12
    rows = Rows(hip, n, ctx)
    pages = Pages(hip, rng, [a + c for a, c in zip(n, ctx)], 3, 128, 32, bf16)
    got, q, _ = run_attention(hip, rng, rows, pages, n_q)
    for r, i in [(0, 0), (150, 150), (299, 299), (301, 0), (540, 239), (800, 499)]:
        b = 0 if r < 300 else 2
        one = Rows(hip, [1], [ctx[b] + i])
        own = Pages.__new__(Pages)
        own.__dict__.update(pages.__dict__, table=pages.table[b:b + 1])
        o, pv, qk, keys = attention_ref(one, own, q[r:r + 1], n_q)[0]
        err, tol = np.abs(got[r].reshape(n_q, 128) - o), attention_tol(pv, qk, keys, not bf16)
        assert (err <= tol).all(), (r, float((err / tol).max()))


def test_attention_two_calls_at_once(hip, rng):
    """Two streams, a workspace each, one cache; and one workspace for two calls
    of different sizes on one stream."""
    say("attention on two streams")
    L, st = hip.lib(), [hip.Stream(), hip.Stream()]
    batches = [Rows(hip, [1, 1], [2000, 900]), Rows(hip, [70, 9], [1500, 20])]
    pages = Pages(hip, rng, [2001, 900], 2, 128, 64, True)
    q = [rng.standard_normal((r.rows, 1024)).astype(np.float32) for r in batches]
    want = [run_attention(hip, rng, r, pages, 8, q=x)[0] for r, x in zip(batches, q)]
    size = [L.qlm_paged_attention_workspace_bytes(r.rows, 2, 8, 2, 128, pages.ld * 64)
            for r in batches]
    dq = [buf(hip, x) for x in q]
    for shared in (False, True):
        work = [buf(hip, np.full(max(size), 0xff, np.uint8)) for _ in batches]
        out = [buf(hip, np.full_like(x, FILL)) for x in q]
        for _ in range(3):
            for i, r in enumerate(batches):
                w = work[0 if shared else i]
                hip.call("qlm_paged_attention", dq[i], 1024, r.c, pages.c, None, 0, 0, out[i],
                         1024, 8, w, max(size), st[0 if shared else i].ptr)
        for s in st:
            s.sync()
        # (slot 900 of the second sequence holds NaN, and the row that sees it gives it)
        for x, o in zip(want, out):
            assert np.array_equal(x, o.to_numpy(x.shape, np.float32), equal_nan=True)


# ---- commit ----------------------------------------------------------------------


def walk(parents, tokens, picks):
    path = [0] if parents and parents[0] == -1 else []
    while path:
        kids = [i for i in range(1, min(len(parents), TREE))
                if parents[i] == path[-1] and i > path[-1] and tokens[i] == picks[path[-1]]]
        if not kids:
            break
        path.append(kids[0])
    return path


def run_commit(hip, rows, pages, tokens, picks, layers=1, ld_path=64):
    B = len(rows.n)
    d = [buf(hip, np.array(a, np.int32)) for a in (tokens, picks)]
    path = buf(hip, np.full((B, ld_path), 9, np.int32))
    out = [buf(hip, np.full(B, 9, np.int32)) for _ in range(3)]
    stride = pages.k[0].size
    hip.call("qlm_tree_commit", d[0], d[1], rows.c, pages.c, layers, stride, path, ld_path, *out,
             None)
    return [path.to_numpy((B, ld_path), np.int32)] + [o.to_numpy(B, np.int32) for o in out]


@pytest.mark.parametrize("hd,bf16,layers,page", [(128, True, 1, 16), (128, False, 3, 64),
                                                 (256, True, 2, 256), (256, False, 1, 32)])
@pytest.mark.parametrize("alphabet", [1, 2, 50])
def test_commit(hip, rng, hd, bf16, layers, page, alphabet):
    """Few distinct tokens: long paths and several children with the pick (the
    first is taken); many: short ones."""
    say(f"commit hd={hd} bf16={bf16} layers={layers} page={page} alphabet={alphabet}")
    n, ctx = [64, 1, 0, 17, 30, 70], [100, 0, 3, 15, 5, 31]
    parents = [random_tree(rng, k, reach=3, padding=k // 10) for k in n]
    parents[4][0] = -2  # no root
    rows = Rows(hip, n, ctx, parents, before=1, behind=2)
    pages = Pages(hip, rng, [a + c for a, c in zip(n, ctx)], 3, hd, page, bf16, layers=layers)
    tokens, picks = (rng.integers(0, alphabet, rows.rows) for _ in range(2))
    path, acc, nxt, ln = run_commit(hip, rows, pages, tokens, picks, layers, ld_path=67)
    want = [pages.k.copy(), pages.v.copy()]
    for b, first, k, c, _ in rows.seqs():
        p = walk(parents[b], tokens[first:first + k], picks[first:first + k])
        assert path[b].tolist() == p + [-1] * (67 - len(p))
        assert acc[b] == len(p) and ln[b] == c + len(p)
        assert nxt[b] == (picks[first + p[-1]] if p else -1)
        for w, pool in zip(want, (pages.k, pages.v)):
            for i, r in enumerate(p):
                (tp, ti), (fp, fi) = pages.at(b, c + i), pages.at(b, c + r)
                w[:, tp, :, ti] = pool[:, fp, :, fi]
    for w, g in zip(want, pages.download()):
        assert np.array_equal(w, g, equal_nan=True)


def test_commit_slots_that_are_not_there(hip, rng):
    """A move from or to a page that is out of range does not happen."""
    say("commit bad pages")
    parents = [[-1, 0, 0, 2, 3, 4] + [5 + i for i in range(20)]]
    rows = Rows(hip, [26], [14], parents)
    pages = Pages(hip, rng, [40], 2, 128, 16, True)
    pages.table[0, 1] = 2 ** 30
    pages.upload(hip)
    tokens = np.arange(26)
    picks = np.array([2, 0, 3, 4, 5] + [6 + i for i in range(21)])
    path, acc, nxt, ln = run_commit(hip, rows, pages, tokens, picks)
    assert path[0, :25].tolist() == [0] + list(range(2, 26)) and acc[0] == 25 and nxt[0] == 26
    for w, g in zip((pages.k, pages.v), pages.download()):
        for i, r in enumerate(path[0, :25]):
            (tp, ti), (fp, fi) = pages.at(0, 14 + i), pages.at(0, 14 + r)
            if tp < pages.n_pages and fp < pages.n_pages and i != r:
                assert np.array_equal(g[:, tp, :, ti], w[:, fp, :, fi])
        # slot 16 + 14 lies in the page that is not there: nothing else changed
        p = pages.table[0, 0]
        assert np.array_equal(g[:, p, :, :15], w[:, p, :, :15])


# ---- DeltaNet --------------------------------------------------------------------


def dn_inputs(rng, rows, H, B, pad=0, strong=False):
    C = 3 * H * 128
    r = lambda *s: rng.standard_normal(s).astype(np.float32)
    dt = np.exp(rng.uniform(np.log(1e-3), np.log(1e-1), H))
    return dict(proj=r(rows.rows, 4 * H * 128 + 2 * H + pad), conv=r(B, 3, C), conv_w=r(4, C) * 0.4,
                A_log=np.log(rng.uniform(1, 16, H)).astype(np.float32) + (4 if strong else 0),
                dt=np.log(np.expm1(dt)).astype(np.float32) + (3 if strong else 0),
                norm=1 + 0.1 * r(128), state=r(B, H, 128, 128) * 0.1)


def run_tree(hip, rows, inp, H, ldo=None):
    d = {k: buf(hip, v) for k, v in inp.items()}
    ldo = ldo or H * 128
    out = buf(hip, np.full((rows.rows, ldo), FILL, np.float32))
    n = hip.lib().qlm_deltanet_tree_workspace_bytes(rows.rows, H, 128)
    work = buf(hip, np.full(n, 0xff, np.uint8))
    hip.call("qlm_deltanet_tree", d["proj"], inp["proj"].shape[1], rows.c, d["conv"], d["conv_w"],
             d["A_log"], d["dt"], d["norm"], d["state"], out, ldo, H, 128, work, n, None)
    assert np.array_equal(d["state"].to_numpy(inp["state"].shape, np.float32), inp["state"],
                          equal_nan=True)
    assert np.array_equal(d["conv"].to_numpy(inp["conv"].shape, np.float32), inp["conv"])
    return out.to_numpy((rows.rows, ldo), np.float32)


# What fp32 arithmetic may leave of a head's largest output, normwise: the
# framework's bound for reassociated DeltaNet forms. A line of 64 nodes is at
# most 64 steps of ~10 roundings whose effect the decays and the unit keys keep
# from growing: 64 * 10 * 2^-24 = 4e-5. But o = sum q_i S_ij is no better than
# its terms: q has the conv's (8), SiLU's (4) and the norm's (12) roundings, S
# as many of its own, the sum 16 more, so it is off by up to 64 2^-24 of sum |q_i|
# |S_ij|, whatever is left of that sum. A strong decay leaves S about k w^T, so
# that o is about (q . k) w, where q . k of a node may be 10^-3 of its terms' sum:
# numpy's own fp32 then has 2e-5, with q . k = -3e-4.
DN_TOL = 4e-5


def check_tree(rows, inp, H, out, skip=()):
    seen = np.zeros(rows.rows, bool)
    for b, first, n, ctx, ls in rows.seqs():
        ls = [l if i < TREE else None for i, l in enumerate(ls)]
        seen[first:first + n] = True
        done = deltanet_ref(rows, b, ls, inp["proj"], inp["conv"][b], inp["conv_w"], inp["A_log"],
                            inp["dt"], inp["state"][b], H, first, ctx)
        for i in range(n):
            x = out[first + i, :H * 128]
            if ls[i] is None:
                assert (x == 0).all(), (b, i)
                continue
            if first + i in skip:
                continue
            o, cond = done[i][1], done[i][3]
            z = inp["proj"][first + i, 3 * H * 128:4 * H * 128].reshape(H, 128).astype(np.float64)
            want = o / np.sqrt((o * o).mean(1, keepdims=True) + 1e-6) * inp["norm"]
            want = want * z / (1 + np.exp(-z))
            tol = np.maximum(DN_TOL, 64 * U * cond) * np.abs(want).max(1)
            assert (np.abs(x.reshape(H, 128) - want).max(1) <= tol).all(), (b, i)
    assert (out[~seen] == FILL).all() and (out[:, H * 128:] == FILL).all()


@pytest.mark.parametrize("H", [1, 2, 5])
@pytest.mark.parametrize("n", [[1], [16], [5, 0, 11], [17, 2], [64, 33], [64, 70, 3, 40]])
@pytest.mark.parametrize("strong", [False, True])
def test_deltanet_tree(hip, rng, H, n, strong):
    say(f"deltanet tree H={H} n={n} strong={strong}")
    ctx = [int(x) for x in rng.integers(0, 9, len(n))]
    rows = Rows(hip, n, ctx, [random_tree(rng, k, padding=k // 9) for k in n], before=1, behind=2)
    inp = dn_inputs(rng, rows, H, len(n), pad=3, strong=strong)
    check_tree(rows, inp, H, run_tree(hip, rows, inp, H, H * 128 + 5))


@pytest.mark.parametrize("B,H", [(16, 2), (3, 16), (9, 16), (40, 4)])
def test_deltanet_tree_batches(hip, rng, B, H):
    """Every way of sharing a head's columns out."""
    say(f"deltanet tree B={B} H={H}")
    n = [int(x) for x in rng.integers(0, 7, B)]
    n[0] = 24
    rows = Rows(hip, n, [b % 5 for b in range(B)], [random_tree(rng, k) for k in n])
    inp = dn_inputs(rng, rows, H, B)
    check_tree(rows, inp, H, run_tree(hip, rows, inp, H))


@pytest.mark.parametrize("B,H", [(1, 33), (5, 16), (9, 16)])
def test_deltanet_tree_odd_values_and_many_rows(hip, rng, B, H):
    """Where a head's columns are four workgroups', two's and one's: rows past
    the 64th, and a node that is not finite."""
    say(f"deltanet odd values B={B} H={H}")
    n = [70] + [3] * (B - 1)
    parents = [[-1] + [max(0, i - 2) for i in range(1, k)] for k in n]
    rows = Rows(hip, n, [b % 3 for b in range(B)], parents, behind=1)
    inp = dn_inputs(rng, rows, H, B)
    check_tree(rows, inp, H, run_tree(hip, rows, inp, H))
    clean = {k: v.copy() for k, v in inp.items()}
    inp["proj"][40, H * 128 + 9] = np.nan  # a key channel of head 0
    out = run_tree(hip, rows, inp, H)
    below = {i for i, l in enumerate(lines(parents[0], n[0])) if l and 40 in l}
    check_tree(rows, clean, H, out, skip=below)
    assert np.isnan(out[40, :128]).any() and np.isfinite(out[40, 128:]).all()


def test_deltanet_chain_equals_prefill(hip, rng):
    """A chain is the prefill of its rows, but for the state."""
    H, T, ctx = 2, 40, 7
    say("deltanet chain")
    rows = Rows(hip, [T], [ctx])
    inp = dn_inputs(rng, rows, H, 1)
    got = run_tree(hip, rows, inp, H)
    d = {k: buf(hip, v) for k, v in inp.items()}
    out = buf(hip, np.zeros((T, H * 128), np.float32))
    hip.call("qlm_deltanet_prefill", d["proj"], inp["proj"].shape[1], T, d["conv"], d["conv_w"],
             d["A_log"], d["dt"], d["norm"], d["state"], ctx, out, H * 128, H, 128, None)
    want = out.to_numpy((T, H * 128), np.float32)
    assert np.abs(got - want).max() <= 2 * DN_TOL * np.abs(want).max()


@pytest.mark.parametrize("what", [np.nan, np.inf])
def test_deltanet_other_branches_values(hip, rng, what):
    """A node that is not finite reaches those below it and nobody else."""
    H, n = 2, 20
    say(f"deltanet {what} in a branch")
    parents = [[-1] + [max(0, i - 2) for i in range(1, n)]]
    parents[0][5] = 3
    rows = Rows(hip, [n], [4], parents)
    inp = dn_inputs(rng, rows, H, 1)
    clean = {k: v.copy() for k, v in inp.items()}
    inp["proj"][4, 130] = what  # a query channel of head 1
    inp["proj"][4, 2 * H * 128 + 7] = what  # a value channel of head 0
    out = run_tree(hip, rows, inp, H)
    below = {i for i, l in enumerate(lines(parents[0], n)) if 4 in l}
    check_tree(rows, clean, H, out, skip=below)
    assert not np.isfinite(out[4, :256]).all()


@pytest.mark.parametrize("H,B", [(1, 1), (2, 3), (16, 5), (16, 9)])
@pytest.mark.parametrize("n", [1, 15, 40, 64])
def test_deltanet_commit(hip, rng, H, B, n):
    say(f"deltanet commit H={H} B={B} n={n}")
    ctx = [int(x) for x in rng.integers(0, 9, B)]
    parents = [random_tree(rng, n, reach=2) for _ in range(B)]
    rows = Rows(hip, [n] * B, ctx, parents, before=1)
    inp = dn_inputs(rng, rows, H, B)
    paths, path = [], np.full((B, 66), -1, np.int32)
    for b in range(B):
        ls = lines(parents[b], n)
        one = ls[int(rng.integers(0, n))] if b else ls[-1]
        if b == 2:
            one = []
        path[b, :len(one)] = one
        paths.append(list(one))
    acc = np.array([len(p) for p in paths], np.int32)
    if B > 3:
        acc[3] = 65  # the path's own end counts
    d = {k: buf(hip, v) for k, v in inp.items()}
    hip.call("qlm_deltanet_tree_commit", d["proj"], inp["proj"].shape[1], rows.c, buf(hip, path),
             66, buf(hip, acc), d["conv"], d["conv_w"], d["A_log"], d["dt"], d["state"], H, 128,
             None)
    state = d["state"].to_numpy(inp["state"].shape, np.float32)
    conv = d["conv"].to_numpy(inp["conv"].shape, np.float32)
    for b in range(B):
        if not paths[b]:
            assert np.array_equal(state[b], inp["state"][b])
            assert np.array_equal(conv[b], inp["conv"][b])
            continue
        done = deltanet_ref(rows, b, lines(parents[b], n), inp["proj"], inp["conv"][b],
                            inp["conv_w"], inp["A_log"], inp["dt"], inp["state"][b], H,
                            rows.start[b], ctx[b])
        S, _, line, _ = done[paths[b][-1]]
        assert np.abs(state[b] - S).max() <= DN_TOL * np.abs(S).max()
        for j in range(3):
            assert np.array_equal(conv[b, (ctx[b] + len(paths[b]) + j) % 3], line[j])


# ---- together --------------------------------------------------------------------


class Serving:
    """One attention layer and one DeltaNet layer of a small hybrid model with
    drafted trees: append, attention, mixer, then the commits."""

    n_q, n_kv, hd, H, rot = 8, 2, 128, 2, 32

    def __init__(self, hip, rng, n, ctx, parents):
        self.hip, self.rows = hip, Rows(hip, n, ctx, parents, behind=1)
        self.room = [a + c for a, c in zip(n, ctx)]
        self.pages = Pages(hip, rng, self.room, self.n_kv, self.hd, 16, True, filled=ctx)
        R, B = self.rows.rows, len(n)
        self.ld = self.n_q * 256 + 2 * self.n_kv * 128
        self.qkv = rng.standard_normal((R, self.ld)).astype(np.float32)
        self.cos, self.sin = tables(max(self.room) + 1, self.rot // 2)
        self.inp = dn_inputs(rng, self.rows, self.H, B)
        self.tokens, self.picks = (rng.integers(0, 2, R).astype(np.int32) for _ in range(2))
        L = hip.lib()
        self.wa = L.qlm_paged_attention_workspace_bytes(R, B, self.n_q, self.n_kv, self.hd,
                                                        self.pages.ld * 16)
        self.wd = L.qlm_deltanet_tree_workspace_bytes(R, self.H, 128)
        z = lambda *s: buf(hip, np.zeros(s, np.float32))
        self.d = {k: buf(hip, v) for k, v in
                  dict(self.inp, qkv=self.qkv, cos=self.cos, sin=self.sin, tokens=self.tokens,
                       picks=self.picks).items()}
        self.d.update(q=z(R, 1024), att=z(R, 1024), mix=z(R, 256), work=z(max(self.wa, self.wd)),
                      path=buf(hip, np.zeros((B, 64), np.int32)),
                      acc=buf(hip, np.zeros(B, np.int32)), next=buf(hip, np.zeros(B, np.int32)))

    def run(self, stream=None):
        d, r, p, call = self.d, self.rows.c, self.pages.c, self.hip.call
        call("qlm_paged_append", d["qkv"], self.ld, None, None, d["cos"], d["sin"],
             self.cos.shape[0], self.rot, None, 0, None, 0, r, p, d["q"], 1024, self.n_q, 1, stream)
        call("qlm_paged_attention", d["q"], 1024, r, p, d["qkv"].ptr + 4 * 128, self.ld, 256,
             d["att"], 1024, self.n_q, d["work"], self.wa, stream)
        ldp = self.inp["proj"].shape[1]
        call("qlm_deltanet_tree", d["proj"], ldp, r, d["conv"], d["conv_w"], d["A_log"], d["dt"],
             d["norm"], d["state"], d["mix"], 256, self.H, 128, d["work"], self.wd, stream)
        call("qlm_tree_commit", d["tokens"], d["picks"], r, p, 1, 0, d["path"], 64, d["acc"],
             d["next"], None, stream)
        call("qlm_deltanet_tree_commit", d["proj"], ldp, r, d["path"], 64, d["acc"], d["conv"],
             d["conv_w"], d["A_log"], d["dt"], d["state"], self.H, 128, stream)

    def outputs(self):
        R, B, d = self.rows.rows, len(self.rows.n), self.d
        return [d["att"].to_numpy((R, 1024), np.float32), d["mix"].to_numpy((R, 256), np.float32),
                d["path"].to_numpy((B, 64), np.int32), d["acc"].to_numpy(B, np.int32),
                d["state"].to_numpy(self.inp["state"].shape, np.float32),
                d["conv"].to_numpy(self.inp["conv"].shape, np.float32)] + self.pages.download()

    def reset(self):
        self.pages.dk.upload(bf16_bits(self.pages.k))
        self.pages.dv.upload(bf16_bits(self.pages.v))
        for k in ("state", "conv"):
            self.d[k].upload(self.inp[k])


def serving(hip, rng):
    n, ctx = [20, 1, 0, 33], [300, 0, 5, 64]
    return Serving(hip, rng, n, ctx, [random_tree(rng, k, reach=3, padding=k // 10) for k in n])


def test_a_verification_from_end_to_end(hip, rng):
    say("verification")
    s = serving(hip, rng)
    s.run()
    att, mix, path, acc, state, conv, k, v = s.outputs()
    # the pools before the commit, with the queries' own path through append
    ref_pages = Pages(hip, rng, s.room, s.n_kv, s.hd, 16, True, filled=[0] * 4)
    ref_pages.table, ref_pages.k, ref_pages.v = s.pages.table, s.pages.k.copy(), s.pages.v.copy()
    q = np.zeros((s.rows.rows, 1024), np.float32)
    for b, first, n, ctx, ls in s.rows.seqs():
        for i in range(n):
            if ls[i] is None:
                continue
            where = np.full(16, ctx + len(ls[i]) - 1)
            x = s.qkv[first + i].astype(np.float64)
            heads = x[:8 * 256].reshape(8, 256)[:, :128]
            q[first + i] = rope_ref(heads, where, 16, s.cos, s.sin).ravel()
            p, at = s.pages.at(b, ctx + i)
            kk = rope_ref(x[2048:2304].reshape(2, 128), where, 16, s.cos, s.sin)
            # a key next to a rounding border may have gone either way: what was
            # stored is one of its two neighbours
            kb = bf16_to_f32(bf16_bits(kk.astype(np.float32)))
            ref_pages.k[0, p, :, at] = kb
            ref_pages.v[0, p, :, at] = bf16_to_f32(bf16_bits(x[2304:2560].astype(np.float32)
                                                             .reshape(2, 128)))
    gate = s.qkv[:, :2048].reshape(-1, 8, 2, 128)[:, :, 1].reshape(-1, 1024)
    for r, (o, pv, qk, keys) in attention_ref(s.rows, ref_pages, q, 8, gate).items():
        # queries off by a rotation's roundings (16 U), and one key element in
        # a few thousand by a bf16 step (2^-7 of it, a 128th of its score's bound)
        tol = attention_tol(pv, qk, keys, False) * (1 + 16 * U) + qk[:, None] * 2.0 ** -13 * pv
        assert (np.abs(att[r].reshape(8, 128) - o) <= tol).all(), r
    check_tree(s.rows, s.inp, s.H, np.where(np.arange(len(mix))[:, None] < s.rows.start[-1], mix,
                                            FILL).astype(np.float32))
    for b, first, n, ctx, ls in s.rows.seqs():
        one = walk(s.rows.parents[b], s.tokens[first:first + n], s.picks[first:first + n])
        assert path[b].tolist() == one + [-1] * (64 - len(one)) and acc[b] == len(one)
        for i, r in enumerate(one):
            (tp, ti), (fp, fi) = s.pages.at(b, ctx + i), s.pages.at(b, ctx + r)
            assert np.array_equal(v[0, tp, :, ti], ref_pages.v[0, fp, :, fi])
        if one:
            done = deltanet_ref(s.rows, b, ls, s.inp["proj"], s.inp["conv"][b], s.inp["conv_w"],
                                s.inp["A_log"], s.inp["dt"], s.inp["state"][b], s.H, first, ctx)
            S = done[one[-1]][0]
            assert np.abs(state[b] - S).max() <= DN_TOL * np.abs(S).max()


def test_a_verification_in_a_captured_graph(hip, rng):
    """Replayed with eager work between, on trees and lengths that change
    between the replays: the arrays are read on the device."""
    say("verification graph")
    s, L = serving(hip, rng), hip.lib()
    st, g = hip.Stream(), C.c_void_p()
    hip.check(L.qlm_graph_begin(st.ptr))
    s.run(st.ptr)
    hip.check(L.qlm_graph_end(st.ptr, C.byref(g)))
    try:
        for step in range(4):
            parents = [random_tree(rng, k, reach=1 + step, padding=step) if k > 8 else p
                       for k, p in zip(s.rows.n, s.rows.parents)]
            flat = np.array([p for q in parents for p in q] + [-2], np.int32)
            s.rows.d[2].upload(flat)
            ctx = [max(0, c - step) for c in (300, 0, 5, 64)]
            s.rows.d[1].upload(np.array(ctx, np.int32))
            s.reset()
            s.run()
            want = s.outputs()
            s.reset()
            hip.check(L.qlm_graph_launch(g, st.ptr))
            st.sync()
            for a, b in zip(want, s.outputs()):
                assert np.array_equal(a, b, equal_nan=True)
    finally:
        hip.check(L.qlm_graph_destroy(g))
