"""Ragged rows, trees and paged caches for the tests: inputs on the device, and
the operators' definitions in 64 bits (numpy)."""

import numpy as np

from tests.util import bf16_bits, bf16_to_f32

TREE = 64
EPS = 1e-6


def random_tree(rng, n, reach=9, padding=0):
    """Parents of n nodes: a root, each later node below one of the `reach`
    before it; the last `padding` are no nodes (-2)."""
    p = [-1] + [int(rng.integers(max(0, i - reach), i)) for i in range(1, n)]
    p = p[:n]
    for i in range(n - padding, n):
        p[i] = -2
    return p


def lines(parent, n):
    """Each row's line (root first) as a list of rows, None outside the tree;
    parent None: a chain."""
    if parent is None:
        return [list(range(i + 1)) for i in range(n)]
    out = []
    for i in range(n):
        p = int(parent[i])
        if i >= TREE:
            out.append(None)
        elif p == -1:
            out.append([i])
        elif 0 <= p < i and out[p] is not None:
            out.append(out[p] + [i])
        else:
            out.append(None)
    return out


class Rows:
    """A qlm_row_batch of sequences with n[b] rows after ctx[b] positions;
    parents: a list a sequence, or None for chains. `before` and `behind` rows
    belong to no sequence."""

    def __init__(self, hip, n, ctx, parents=None, before=0, behind=0):
        self.n, self.ctx, self.parents = list(n), list(ctx), parents
        self.start = [before]
        for k in n:
            self.start.append(self.start[-1] + k)
        self.rows = self.start[-1] + behind
        self.d = [hip.DeviceBuffer.from_numpy(np.array(a, np.int32))
                  for a in (self.start, self.ctx)]
        parent = None
        if parents is not None:
            flat = [-2] * before + [p for s in parents for p in s] + [-2] * behind
            parent = hip.DeviceBuffer.from_numpy(np.array(flat, np.int32))
            self.d.append(parent)
        self.c = hip.RowBatch(len(self.n), self.rows, self.d[0].ptr, self.d[1].ptr,
                              parent.ptr if parent else None)

    def seqs(self):
        """(b, first row, rows, context, lines)."""
        for b, (n, ctx) in enumerate(zip(self.n, self.ctx)):
            yield b, self.start[b], n, ctx, lines(self.parents[b] if self.parents else None, n)


class Pages:
    """A qlm_kv_pages with every slot of `room[b]` positions a sequence, pages
    in random order; host copies k, v hold the stored values in fp32. Slots
    that no position has been given hold NaN."""

    def __init__(self, hip, rng, room, n_kv, hd, page, bf16, filled=None, layers=1, spare=2):
        self.page, self.n_kv, self.hd, self.bf16 = page, n_kv, hd, bf16
        counts = [-(-max(r, 1) // page) for r in room]
        self.ld = max(counts) + 1
        self.n_pages = sum(counts) + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(room), self.ld), -1, np.int32)
        at = 0
        for b, c in enumerate(counts):
            self.table[b, :c] = order[at:at + c]
            at += c
        shape = (layers, self.n_pages, n_kv, page, hd)
        self.k = np.full(shape, np.nan, np.float32)
        self.v = np.full(shape, np.nan, np.float32)
        for b, m in enumerate(filled if filled is not None else room):
            for s in range(m):
                p, i = self.at(b, s)
                for pool in (self.k, self.v):
                    x = rng.standard_normal((layers, n_kv, hd)).astype(np.float32)
                    pool[:, p, :, i] = bf16_to_f32(bf16_bits(x)) if bf16 else x
        self.upload(hip)

    def at(self, b, slot):
        return int(self.table[b, slot // self.page]), slot % self.page

    def rows(self, pool, b, slots, layer=0):
        """[len(slots), n_kv, hd] of a host pool."""
        return np.stack([pool[layer, p, :, i] for p, i in (self.at(b, s) for s in slots)])

    def upload(self, hip):
        enc = bf16_bits if self.bf16 else (lambda x: x)
        self.dk, self.dv = (hip.DeviceBuffer.from_numpy(enc(x)) for x in (self.k, self.v))
        self.dt = hip.DeviceBuffer.from_numpy(self.table)
        self.c = hip.KvPages(self.dk.ptr, self.dv.ptr, 1 if self.bf16 else 0, self.n_pages,
                             self.page, self.n_kv, self.hd, self.dt.ptr, self.ld)

    def download(self):
        """The device's pools as fp32."""
        t = np.uint16 if self.bf16 else np.float32
        out = [d.to_numpy(self.k.shape, t) for d in (self.dk, self.dv)]
        return [bf16_to_f32(x) if self.bf16 else x for x in out]


def attention_ref(rows, pages, q, n_q, gate=None, k=None, v=None):
    """{row: (out [n_q, hd], bound [n_q, hd])}: the definition in 64 bits, and
    sum p |v| and max sum |q k| for the tolerance."""
    k = pages.k if k is None else k
    v = pages.v if v is None else v
    hd, G = pages.hd, n_q // pages.n_kv
    room = pages.ld * pages.page
    out = {}
    for b, first, n, ctx, ls in rows.seqs():
        there = {s for s in range(min(ctx + n, room))
                 if 0 <= pages.table[b, s // pages.page] < pages.n_pages}
        for i, line in enumerate(ls):
            slots = [] if line is None else [s for s in list(range(ctx)) + [ctx + j for j in line]
                                             if s in there]
            o, pv, qk = np.zeros((n_q, hd)), np.zeros((n_q, hd)), np.zeros(n_q)
            if slots:
                ks = pages.rows(k, b, slots).astype(np.float64)
                vs = pages.rows(v, b, slots).astype(np.float64)
                for h in range(n_q):
                    x = q[first + i, h * hd:(h + 1) * hd].astype(np.float64)
                    s = ks[:, h // G] @ x / np.sqrt(hd)
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    o[h], pv[h] = p @ vs[:, h // G], p @ np.abs(vs[:, h // G])
                    qk[h] = (np.abs(ks[:, h // G]) @ np.abs(x)).max() / np.sqrt(hd)
            if gate is not None:
                s = 1 / (1 + np.exp(-gate[first + i].reshape(n_q, hd).astype(np.float64)))
                o, pv = o * s, pv * s
            out[first + i] = (o, pv, qk, len(slots))
    return out


def attention_tol(pv, qk, keys, fp32_cache):
    """The largest difference that qlm_paged_attention's fp32 arithmetic allows.
    Products of bf16 terms are exact, and so is a split into three (2^-25 of a
    value). A score: the scale's product and its rounding (2), one accumulation
    for every 32 products of each of the three terms and up to 5 inside of them
    (bf16: 3 * 8 + 5), or one for every product (fp32, 256), beginning at a
    reference no larger than the largest sum |q k|: twice. A score that is off by e
    moves its probability by e relatively, and their sum too. Then the
    exponential and its split (3), and the sums over keys: bf16 one accumulation
    for every 32 keys and term, fp32 one for every key, the probabilities' own
    sum the same, and of chunks and waves that meet at most 40 more."""
    u = 2.0 ** -24
    score = 2 * qk * (260 if fp32_cache else 31) * u
    sums = keys if fp32_cache else 3 * keys / 32 + 5
    rel = 2 * score + (3 + 2 * sums + 40) * u
    return rel[:, None] * pv + 1e-30


def rope_ref(x, pos, half, cos, sin):
    """x [.., hd] in 64 bits, pos [half] a row's table rows."""
    j = np.arange(half)
    c, s = cos[pos, j].astype(np.float64), sin[pos, j].astype(np.float64)
    y = x.copy()
    y[..., :half] = x[..., :half] * c - x[..., half:2 * half] * s
    y[..., half:2 * half] = x[..., half:2 * half] * c + x[..., :half] * s
    return y


def deltanet_ref(rows, b, ls, proj, conv, conv_w, A_log, dt, state, H, first, ctx, d=128):
    """Every node of `ls` (lines) along its own line, one step at a time in 64
    bits: {row: (state, o before the head norm [H, d], the last three inputs, the
    heads' conditions: how much the terms of o's sums cancel)}."""
    C = 3 * H * d
    ring = [conv[(ctx + j) % 3].astype(np.float64) for j in range(3)]
    done = {}
    for i, line in enumerate(ls):
        if line is None:
            continue
        S = done[line[-2]][0] if len(line) > 1 else state.astype(np.float64)
        xs = ring + [proj[first + r, :C].astype(np.float64) for r in line]
        y = sum(xs[len(xs) - 4 + j] * conv_w[j].astype(np.float64) for j in range(4))
        y = y / (1 + np.exp(-y))
        q, k, v = y.reshape(3, H, d)
        q = q / np.sqrt((q * q).sum(1, keepdims=True) + EPS)
        k = k / np.sqrt((k * k).sum(1, keepdims=True) + EPS)
        pr = proj[first + i].astype(np.float64)
        beta = 1 / (1 + np.exp(-pr[4 * H * d:4 * H * d + H]))
        x = pr[4 * H * d + H:4 * H * d + 2 * H] + dt
        a = np.exp(-np.exp(A_log.astype(np.float64)) * np.log1p(np.exp(np.minimum(x, 700.0))))
        S = S * a[:, None, None]
        w = beta[:, None] * (v - np.einsum("hij,hi->hj", S, k))
        S = S + k[:, :, None] * w[:, None, :]
        o = np.einsum("hij,hi->hj", S, q) / np.sqrt(d)
        # how much larger than a head's largest output the terms of one are
        size = np.einsum("hij,hi->hj", np.abs(S), np.abs(q)).max(1) / np.sqrt(d)
        done[i] = (S, o, xs[-3:], size / np.abs(o).max(1))
    return done
