"""Edges of the paged attention and of the DeltaNet mixer over trees: scores and
convolutions at the ends of fp32's range, whatever lies in slots that nobody sees,
contexts that are cut and joined, and every form that a call can take. Against
the definitions in 64 bits, or against the framework's row-by-row mixer where that
is what the operators promise; tolerances are those of test_tree_ops_gpu.py."""

import time

import numpy as np
import pytest

from tests.test_tree_ops_gpu import (DN_TOL, FILL, buf, check_attention, check_tree, dn_inputs,
                                     run_attention, run_tree)
from tests.tree_util import Pages, Rows, deltanet_ref, lines, random_tree
from tests.util import say

pytestmark = pytest.mark.gpu


# ---- DeltaNet: convolutions at the ends of the range ------------------------------


def prefill(hip, inp, T, H, ctx):
    """Outputs, state and ring that the framework's row-by-row mixer leaves."""
    d = {k: buf(hip, v) for k, v in inp.items()}
    out = buf(hip, np.zeros((T, H * 128), np.float32))
    hip.call("qlm_deltanet_prefill", d["proj"], inp["proj"].shape[1], T, d["conv"], d["conv_w"],
             d["A_log"], d["dt"], d["norm"], d["state"], ctx, out, H * 128, H, 128, None)
    return (out.to_numpy((T, H * 128), np.float32),
            d["state"].to_numpy(inp["state"].shape, np.float32),
            d["conv"].to_numpy(inp["conv"].shape, np.float32))


def commit_chain(hip, rows, inp, T, H):
    path = np.full((1, 64), -1, np.int32)
    path[0, :T] = np.arange(T)
    d = {k: buf(hip, v) for k, v in inp.items()}
    hip.call("qlm_deltanet_tree_commit", d["proj"], inp["proj"].shape[1], rows.c, buf(hip, path),
             64, buf(hip, np.array([T], np.int32)), d["conv"], d["conv_w"], d["A_log"], d["dt"],
             d["state"], H, 128, None)
    return (d["state"].to_numpy(inp["state"].shape, np.float32),
            d["conv"].to_numpy(inp["conv"].shape, np.float32))


def sums_of(rng, rows, H, part, values):
    """Inputs whose convolution of channel 5 of head 0 of `part` is values[i] at
    node i."""
    inp = dn_inputs(rng, rows, H, 1)
    ch = "qkv".index(part) * H * 128 + 5
    inp["conv_w"][:, ch] = [0, 0, 0, 1]
    for i, x in values.items():
        inp["proj"][i, ch] = x
    return inp


@pytest.mark.parametrize("H", [1, 140])
@pytest.mark.parametrize("part", ["q", "k", "v"])
@pytest.mark.parametrize("value", [2.5e38, 1e30, -1e25, -1e36, -2.5e38])
def test_deltanet_large_convolutions(hip, rng, H, part, value):
    """SiLU of a sum far from 0 is the sum or 0, as the row-by-row mixer has it."""
    T, ctx = 7, 5
    say(f"deltanet conv {part} = {value} H={H}")
    rows = Rows(hip, [T], [ctx])
    inp = sums_of(rng, rows, H, part, {2: value})
    want, _, _ = prefill(hip, inp, T, H, ctx)
    assert np.isfinite(want).all()
    got = run_tree(hip, rows, inp, H)
    for a, b in zip(got.reshape(T, H, 128), want.reshape(T, H, 128)):
        assert (np.abs(a - b).max(1) <= 2 * DN_TOL * np.abs(b).max(1)).all()


@pytest.mark.parametrize("H", [1, 140])
@pytest.mark.parametrize("part", ["q", "k"])
def test_deltanet_vectors_whose_squares_leave_the_range(hip, rng, H, part):
    """Their l2 norm is infinite: the row-by-row mixer's vector is 0 then, and the
    state goes on."""
    T, ctx = 9, 4
    say(f"deltanet large {part} H={H}")
    rows = Rows(hip, [T], [ctx])
    inp = sums_of(rng, rows, H, part, {2: 1e25, 4: 3e22, 5: 1e18, 7: 2e38})
    inp["state"][0, 0, 5] *= 1e3  # (1e25 times it times 1e18 is past the range too)
    want, state, conv = prefill(hip, inp, T, H, ctx)
    assert np.isfinite(want).all() and np.isfinite(state).all()
    got = run_tree(hip, rows, inp, H)
    for a, b in zip(got.reshape(T, H, 128), want.reshape(T, H, 128)):
        assert (np.abs(a - b).max(1) <= 2 * DN_TOL * np.abs(b).max(1)).all()
    got, ring = commit_chain(hip, rows, inp, T, H)
    err = np.abs(got - state).max((0, 2, 3))
    assert (err <= 2 * DN_TOL * np.abs(state).max((0, 2, 3))).all()
    assert np.array_equal(ring, conv)


@pytest.mark.parametrize("H,B", [(1, 2), (40, 2), (70, 2)])
@pytest.mark.parametrize("nodes", [14, 40])
@pytest.mark.parametrize("what", [np.nan, np.inf])
def test_deltanet_padding_leaves_no_trace(hip, rng, H, B, nodes, what):
    """The same bits come out whatever a padding node's row of proj holds."""
    say(f"deltanet padding of {what} H={H} nodes={nodes}")
    parents = [random_tree(rng, nodes, padding=nodes // 4), random_tree(rng, nodes)]
    parents[1][nodes // 2] = nodes  # no node, and those below it
    rows = Rows(hip, [nodes] * B, [3, 7], parents)
    inp = dn_inputs(rng, rows, H, B)
    unseen = [f + i for _, f, n, _, ls in rows.seqs() for i in range(n) if ls[i] is None]
    out = []
    for x in (0.0, what):
        inp["proj"][unseen] = x
        out.append(run_tree(hip, rows, inp, H))
        check_tree(rows, inp, H, out[-1])
    assert np.array_equal(*out)


# ---- attention: whatever lies in slots that nobody sees ----------------------------


@pytest.mark.parametrize("hd,bf16", [(128, True), (128, False), (256, True), (256, False)])
@pytest.mark.parametrize("n_q,n_kv,nodes,ctx", [
    (1, 1, 7, 0), (2, 2, 9, 1500), (8, 1, 30, 77), (8, 2, 15, 1200), (4, 2, 64, 0), (4, 2, 64, 700)])
@pytest.mark.parametrize("what", [np.nan, -np.inf])
def test_attention_padding_leaves_no_trace(hip, rng, hd, bf16, n_q, n_kv, nodes, ctx, what):
    """Padding nodes' slots are never written. The same bits come out whatever
    they hold, so nothing is computed a second time on their account."""
    say(f"attention padding of {what} hd={hd} bf16={bf16} {n_q}/{n_kv} nodes={nodes} ctx={ctx}")
    n, at = [nodes, 1, nodes], [ctx, 5, ctx // 2]
    parents = [random_tree(rng, nodes, padding=nodes // 4), [-1], random_tree(rng, nodes)]
    parents[2][nodes // 2] = nodes  # no node, and those below it
    rows = Rows(hip, n, at, parents)
    pages = Pages(hip, rng, [a + c for a, c in zip(n, at)], n_kv, hd, 16, bf16)
    unseen = [pages.at(b, c + i) for b, _, k, c, ls in rows.seqs() for i in range(k)
              if ls[i] is None]
    q = rng.standard_normal((rows.rows, n_q * hd)).astype(np.float32)
    out = []
    for x in (0.0, what):
        for p, i in unseen:
            pages.k[0, p, :, i] = pages.v[0, p, :, i] = x
        pages.upload(hip)
        got = run_attention(hip, rng, rows, pages, n_q, q=q)
        check_attention(rows, pages, *got, n_q)
        out.append(got[0])
    assert np.array_equal(*out)


@pytest.mark.parametrize("hd,bf16", [(128, True), (256, False)])
@pytest.mark.parametrize("n", [1, 40])
def test_attention_of_rows_without_a_page_is_no_slower(hip, rng, hd, bf16, n):
    """Sequences that only fill a batch up, their tables without a page and their
    lengths whatever they were: zeros, and sooner than if the pages were there."""
    B, ctx = 16, 8000
    say(f"attention without pages hd={hd} bf16={bf16} n={n}")
    rows = Rows(hip, [n] * B, [ctx] * B)
    pages = Pages(hip, rng, [ctx + n], 2, hd, 64, bf16)
    pages.table = np.repeat(pages.table, B, 0)  # (one context for all)
    pages.upload(hip)
    q = buf(hip, rng.standard_normal((rows.rows, 4 * hd)).astype(np.float32))
    out = buf(hip, np.full((rows.rows, 4 * hd), FILL, np.float32))
    size = hip.lib().qlm_paged_attention_workspace_bytes(rows.rows, B, 4, 2, hd, pages.ld * 64)
    work, took = hip.DeviceBuffer(size), []
    for table in (pages.table, np.full_like(pages.table, -1)):
        pages.dt.upload(table)
        times = []
        for _ in range(6):
            hip.sync()
            t = time.perf_counter()
            hip.call("qlm_paged_attention", q, 4 * hd, rows.c, pages.c, None, 0, 0, out, 4 * hd, 4,
                     work, size, None)
            hip.sync()
            times.append(time.perf_counter() - t)
        took.append(min(times))
    assert (out.to_numpy((rows.rows, 4 * hd), np.float32) == 0).all()
    say(f"  {took[0] * 1e6:.0f} us, without pages {took[1] * 1e6:.0f}")
    assert took[1] <= 1.5 * took[0]


# ---- attention: scores that are next to nothing ------------------------------------


@pytest.mark.parametrize("hd,bf16", [(128, True), (128, False), (256, True), (256, False)])
@pytest.mark.parametrize("n,n_q", [(1, 1), (2, 8), (70, 1)])
def test_attention_scores_that_round_to_minus_zero(hip, rng, hd, bf16, n, n_q):
    """Blocks of keys whose scores are products below the subnormal numbers,
    negative: they weigh exp(0), beside blocks that weigh otherwise."""
    say(f"attention scores of -0 hd={hd} bf16={bf16} n={n} n_q={n_q}")
    ctx = 300
    rows = Rows(hip, [n], [ctx])
    pages = Pages(hip, rng, [ctx + n], 1, hd, 16, bf16)
    half = hd // 2
    for s in range(ctx + n):
        p, at = pages.at(0, s)
        if s // 32 % 4 in (0, 3):
            pages.k[0, p, 0, at, :half] = -2.0 ** -90
            pages.k[0, p, 0, at, half:] = 0
        else:
            pages.k[0, p, 0, at, :half] = 0
    pages.upload(hip)
    q = np.abs(rng.standard_normal((n, n_q * hd))).astype(np.float32)
    q.reshape(n, n_q, 2, half)[:, :, 0] *= 2.0 ** -80
    check_attention(rows, pages, *run_attention(hip, rng, rows, pages, n_q, q=q), n_q)


# ---- attention: contexts that are cut and joined -----------------------------------


CUT = {
    # one longer than the mean by far, one without rows or keys among them
    "uneven": ([40, 1100, 5000, 2500, 0], [1, 1, 1, 1, 1]),
    "even": ([2100, 2100, 2100], [1, 1, 1]),
    "with rows of none": ([1300, 4000, 9, 3000], [1, 0, 1, 1]),
    "one": ([9000], [1]),
}


@pytest.mark.parametrize("hd,bf16", [(128, True), (128, False), (256, True), (256, False)])
@pytest.mark.parametrize("n_q,n_kv,rows_each", [(2, 2, 1), (4, 1, 2), (4, 1, 4), (16, 2, 2)])
@pytest.mark.parametrize("what", CUT)
def test_attention_cut_contexts(hip, rng, hd, bf16, n_q, n_kv, rows_each, what):
    """Units of 8 and of 16 rows."""
    say(f"attention cut {what} hd={hd} bf16={bf16} {n_q}/{n_kv} rows={rows_each}")
    ctx, n = CUT[what]
    n = [k * rows_each for k in n]
    rows = Rows(hip, n, ctx, before=1, behind=1)
    pages = Pages(hip, rng, [a + c for a, c in zip(n, ctx)], n_kv, hd, 64, bf16)
    check_attention(rows, pages, *run_attention(hip, rng, rows, pages, n_q, gated=True), n_q)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("n_q,n_kv,ctx", [(16, 16, [5000, 300, 9000, 40]), (24, 24, [4000, 3900]),
                                          (24, 12, [100, 7000, 2000]), (260, 260, [1500, 700])])
def test_attention_cut_contexts_of_many_heads(hip, rng, bf16, n_q, n_kv, ctx):
    """Few pieces a head: longer than the shortest that a context is cut into, and
    as many as the batch's lengths ask for."""
    say(f"attention cut {n_q}/{n_kv} bf16={bf16}")
    rows = Rows(hip, [1] * len(ctx), ctx)
    pages = Pages(hip, rng, [c + 1 for c in ctx], n_kv, 128, 128, bf16)
    check_attention(rows, pages, *run_attention(hip, rng, rows, pages, n_q), n_q)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("n_q,rows_each", [(1, 1), (8, 2), (4, 20)])
def test_attention_many_sequences_some_of_them_cut(hip, rng, bf16, n_q, rows_each):
    """More sequences than a wave has lanes, whose records begin in the first
    round over them and go on in the later ones."""
    B = 150
    say(f"attention many cut bf16={bf16} n_q={n_q} rows={rows_each}")
    ctx = [int(x) for x in rng.integers(0, 90, B)]
    for b, c in ((3, 1500), (60, 1100), (64, 2600), (65, 1300), (127, 1700), (128, 2000), (149, 1400)):
        ctx[b] = c
    n = [rows_each * int(x > 0.2) for x in rng.random(B)]
    for b in (3, 64, 128, 149):
        n[b] = rows_each
    rows = Rows(hip, n, ctx, behind=1)
    pages = Pages(hip, rng, [a + c for a, c in zip(n, ctx)], 1, 128, 32, bf16)
    check_attention(rows, pages, *run_attention(hip, rng, rows, pages, n_q), n_q)


@pytest.mark.parametrize("hd,bf16", [(128, True), (128, False), (256, True), (256, False)])
@pytest.mark.parametrize("n_q,n_kv", [(2, 2), (4, 1), (8, 1)])
def test_attention_prompts_and_single_tokens_together(hip, rng, hd, bf16, n_q, n_kv):
    """Prompts of several tiles beside tokens whose contexts are cut."""
    say(f"attention mixed hd={hd} bf16={bf16} {n_q}/{n_kv}")
    n, ctx = [150, 1, 1, 0, 90, 1], [0, 3000, 1500, 40, 700, 130]
    rows = Rows(hip, n, ctx, behind=1)
    pages = Pages(hip, rng, [a + c for a, c in zip(n, ctx)], n_kv, hd, 128, bf16)
    check_attention(rows, pages, *run_attention(hip, rng, rows, pages, n_q, gated=True), n_q)


def test_attention_a_long_context(hip, rng):
    say("attention ctx=40000")
    rows = Rows(hip, [1, 3], [40000, 17])
    pages = Pages(hip, rng, [40001, 20], 1, 128, 256, True)
    check_attention(rows, pages, *run_attention(hip, rng, rows, pages, 4), 4)


# ---- DeltaNet: every form ------------------------------------------------------------


# (rows of a call, and so the nodes that a workgroup has room for; heads of all
# its sequences, and so the columns of one)
@pytest.mark.parametrize("H,B", [(2, 1), (20, 2), (80, 1), (70, 2)])
@pytest.mark.parametrize("n", [14, 30, 50])
@pytest.mark.parametrize("strong", [False, True])
def test_deltanet_every_form(hip, rng, H, B, n, strong):
    """Trees of 2 to n nodes, and their longest lines' commit."""
    say(f"deltanet forms H={H} B={B} n={n} strong={strong}")
    sizes = [n] if B == 1 else [n - n // 3, n // 3]
    ctx = [int(x) for x in rng.integers(0, 9, B)]
    parents = [random_tree(rng, k, reach=2) for k in sizes]
    parents[0] = [-1] + [i - 1 if i < sizes[0] - 3 else int(rng.integers(0, i))
                         for i in range(1, sizes[0])]
    rows = Rows(hip, sizes, ctx, parents)
    inp = dn_inputs(rng, rows, H, B, strong=strong)
    check_tree(rows, inp, H, run_tree(hip, rows, inp, H))
    path, paths = np.full((B, 64), -1, np.int32), []
    for b in range(B):
        paths.append(max(lines(parents[b], sizes[b]), key=len))
        path[b, :len(paths[b])] = paths[b]
    d = {k: buf(hip, v) for k, v in inp.items()}
    hip.call("qlm_deltanet_tree_commit", d["proj"], inp["proj"].shape[1], rows.c, buf(hip, path),
             64, buf(hip, np.array([len(p) for p in paths], np.int32)), d["conv"], d["conv_w"],
             d["A_log"], d["dt"], d["state"], H, 128, None)
    state = d["state"].to_numpy(inp["state"].shape, np.float32)
    conv = d["conv"].to_numpy(inp["conv"].shape, np.float32)
    for b in range(B):
        # (the lines of the path's own rows: no other state is needed)
        ref = deltanet_ref(rows, b, [p if p is not None and set(p) <= set(paths[b]) else None
                                     for p in lines(parents[b], sizes[b])], inp["proj"],
                           inp["conv"][b], inp["conv_w"], inp["A_log"], inp["dt"],
                           inp["state"][b], H, rows.start[b], ctx[b])
        S, _, line, _ = ref[paths[b][-1]]
        assert np.abs(state[b] - S).max() <= DN_TOL * np.abs(S).max()
        for j in range(3):
            assert np.array_equal(conv[b, (ctx[b] + len(paths[b]) + j) % 3], line[j])
