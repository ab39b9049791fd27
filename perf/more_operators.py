"""Operators for serving drafted trees of tokens over a paged key/value cache, as
measurable cases.

  append    QK-norm, rotation by positions of one or several axes and the new
            rows' way into the pages, in one pass (qlm_paged_append)
  attention attention of ragged rows (single tokens, trees, prompts) over the
            pages (qlm_paged_attention)
  commit    the greedy walk through a verified tree and the accepted rows' move
            to their places, all layers at once (qlm_tree_commit)
  deltanet  the Gated DeltaNet mixer over a tree of tokens (qlm_deltanet_tree),
            and its state's and ring's advance along the accepted path
            (qlm_deltanet_tree_commit)

`run` computes the operators' plain form with elementary torch operations, or,
where `own` is true, calls the kernel library.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
EPS = 1e-6
TREE = 64  # nodes of a tree at most
D = 128  # DeltaNet head dim
F32, F64, BF16, I32, I64 = torch.float32, torch.float64, torch.bfloat16, torch.int32, torch.int64

MAX_FLOPS = 4 * 128 * 16 * (2048 * 2048 + 2048 * 2049 // 2)  # of the largest attention
MAX_KV = 64 * 4096  # keys of the largest decode, a batch, at 4 heads of 128 in bf16


def listed():
    return [
        # One decode step of a 4B-class model (16 query / 4 KV heads of 128,
        # quarter rotation, gate beside q): pure latency.
        dict(name="append_1", kind="append", B=1, rows=1, ragged=False, ctx=600, tree=False, tail=0,
             n_q=16, n_kv=4, hd=128, rot=32, axes=1, gated=True, page=64, bf16=True, pad=0),
        # A 2048-token prompt with images: time, height and width positions.
        dict(name="append_2048_axes", kind="append", B=1, rows=2048, ragged=False, ctx=2048,
             tree=False, tail=0, n_q=16, n_kv=4, hd=128, rot=32, axes=3, gated=True, page=64,
             bf16=True, pad=0),
        # A single sequence's next token: latency.
        dict(name="attention_1x600", kind="attention", B=1, rows=1, ragged=False, ctx=600,
             tree=False, tail=0, n_q=16, n_kv=4, hd=128, gated=True, page=64, bf16=True, pad=0),
        # A serving batch of single tokens, contexts from 256 to 8192: the
        # cache's stream.
        dict(name="attention_64x8192_ragged", kind="attention", B=64, rows=1, ragged=True, ctx=8191,
             tree=False, tail=0, n_q=16, n_kv=4, hd=128, gated=True, page=64, bf16=True, pad=0),
        # Verification of 8 trees of 64 drafted tokens, contexts up to 4096.
        dict(name="attention_tree_8x64", kind="attention", B=8, rows=64, ragged=False, ctx=4032,
             tree=True, tail=0, n_q=16, n_kv=4, hd=128, gated=True, page=64, bf16=True, pad=0),
        # The fp32 cache that the engine keeps, wide heads, small pages, trees
        # of odd sizes with padding among them.
        dict(name="attention_tree_f32", kind="attention", B=5, rows=33, ragged=True, ctx=1999,
             tree=True, tail=3, n_q=16, n_kv=2, hd=256, gated=False, page=16, bf16=False, pad=8),
        # The second 2048 rows of a 4096-token prompt.
        dict(name="attention_prompt_2048", kind="attention", B=1, rows=2048, ragged=False, ctx=2048,
             tree=False, tail=0, n_q=16, n_kv=4, hd=128, gated=True, page=64, bf16=True, pad=0),
        # One sequence's tree of 16, the 9 attention layers of the 4B model.
        dict(name="commit_1x16", kind="commit", B=1, rows=16, ragged=False, ctx=600, tree=True,
             tail=0, n_kv=4, hd=128, page=64, bf16=True, layers=9),
        # A batch of 64 trees of up to 64 nodes.
        dict(name="commit_64x64", kind="commit", B=64, rows=64, ragged=True, ctx=1000, tree=True,
             tail=7, n_kv=4, hd=128, page=64, bf16=True, layers=9),
        # One sequence's tree of 16 through a 4B DeltaNet layer.
        dict(name="deltanet_1x16", kind="deltanet", B=1, rows=16, ragged=False, ctx=600, tree=True,
             tail=0, H=16, pad=0, commit=False),
        # Verification of 16 trees of up to 64 nodes in such a layer.
        dict(name="deltanet_16x64", kind="deltanet", B=16, rows=64, ragged=True, ctx=1000,
             tree=True, tail=2, H=16, pad=4, commit=False),
        # The accepted paths of 16 trees of up to 64 nodes into their states.
        dict(name="deltanet_commit_16x64", kind="deltanet", B=16, rows=64, ragged=True, ctx=1000,
             tree=True, tail=2, H=16, pad=4, commit=True),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["append", "attention", "attention", "commit", "deltanet"])
    ragged, tail = rng.random() < 0.5, rng.choice([0, 0, rng.randint(1, 9)])
    page = rng.choice([16, 32, 64, 128, 256])
    bf16 = rng.random() < 0.6
    hd = rng.choice([128, 128, 256])
    n_kv = rng.choice([1, 2, 4, 8])
    n_q = n_kv * rng.choice([1, 2, 4, 8])
    pad = rng.choice([0, 0, 4 * rng.randint(1, 16)])
    if kind == "append":
        tree = rng.random() < 0.5
        B = _log(rng, 1, 64)
        rows = _log(rng, 1, TREE) if tree else _log(rng, 1, 2048)
        rows = max(1, min(rows, 2048 * 24 * 128 // (B * (n_q + 2 * n_kv) * hd)))
        return dict(kind=kind, B=B, rows=rows, ragged=ragged, ctx=rng.randint(0, 1500), tree=tree,
                    tail=tail, n_q=n_q, n_kv=n_kv, hd=hd, rot=2 * rng.randint(0, hd // 2),
                    axes=rng.choice([1, 2, 3]), gated=rng.random() < 0.5, page=page, bf16=bf16,
                    pad=pad)
    if kind == "attention":
        form = rng.choice(["decode", "tree", "prompt"])
        ctx, B = _log(rng, 1, 32768) - 1, _log(rng, 1, 64)
        size = n_kv * hd * (1 if bf16 else 2)
        B = max(1, min(B, MAX_KV * 4 * 128 // (2 * size * (ctx + 1))))
        rows = 1 if form == "decode" else _log(rng, 1, TREE) if form == "tree" else _log(rng, 1, 2048)
        rows = max(1, min(rows, MAX_FLOPS // (4 * hd * n_q * B * (ctx + rows))))
        return dict(kind=kind, B=B, rows=rows, ragged=ragged, ctx=ctx, tree=form == "tree",
                    tail=tail, n_q=n_q, n_kv=n_kv, hd=hd, gated=rng.random() < 0.5, page=page,
                    bf16=bf16, pad=pad)
    if kind == "commit":
        return dict(kind=kind, B=_log(rng, 1, 64), rows=_log(rng, 1, TREE), ragged=ragged,
                    ctx=rng.randint(0, 1000), tree=True, tail=tail, n_kv=min(n_kv, 4), hd=hd,
                    page=page, bf16=bf16, layers=rng.randint(1, 9) if hd == 128 else rng.randint(1, 4))
    H, rows = rng.choice([1, 2, 4, 16, 32]), _log(rng, 1, TREE)
    return dict(kind=kind, B=_log(rng, 1, max(1, min(32, 16384 // (H * rows)))), rows=rows,
                ragged=ragged, ctx=rng.randint(0, 1000), tree=rng.random() < 0.8, tail=tail, H=H,
                pad=pad, commit=rng.random() < 0.4)


# ---- inputs --------------------------------------------------------------------


def _lens(case):
    """Each sequence's new rows and its keys before them, of the case alone."""
    B, rows, ctx = case["B"], case["rows"], case["ctx"]
    if not case["ragged"]:
        return [rows] * B, [ctx] * B
    n = [max(1, rows * ((7 * b + 3) % 16) // 15) if rows == 1 or b == 0
         else rows * ((7 * b + 3) % 16) // 15 for b in range(B)]
    return n, [ctx * (1 + (11 * b + 5) % 32) // 32 for b in range(B)]


def _normal(g, *shape, mean=0.0, std=1.0):
    t = torch.randn(*shape, generator=g, device=DEV, dtype=F32)
    return t.mul_(std).add_(mean)


def _ints(values):
    return torch.tensor(np.asarray(values, np.int32), device=DEV)


def _trees(n, host):
    """Parents of each sequence's nodes: a root, then a drafter's branches, the
    deepest ones grown most. The last of every fifth node up to the end of a
    sequence of more than 20 are padding (-2)."""
    parent = []
    for k in n:
        p = [-1] + [host.randint(max(0, i - 9), i - 1) for i in range(1, k)]
        if k > 20:
            p[k - k // 10:] = [-2] * (k // 10)
        parent += p[:k]
    return parent


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    host = random.Random(seed)
    n, ctx = _lens(case)
    B, total = case["B"], sum(n)
    start = [0] * (B + 1)
    for b in range(B):
        start[b + 1] = start[b] + n[b]
    parent = _trees(n, host) if case["tree"] else None
    all_rows = total + case["tail"]
    st = dict(case=case, n=n, ctx=ctx, start=start, total=total, all_rows=all_rows)
    st["row_start"], st["ctx_len"] = _ints(start), _ints(ctx)
    st["parent"] = None if parent is None else _ints(parent + [-2] * case["tail"])
    if case["kind"] == "deltanet":
        return _prepare_deltanet(case, st, g, host, parent)
    # the pools: pages in any order, a few of them of other sequences
    page, n_kv, hd = case["page"], case["n_kv"], case["hd"]
    room = [c + max(k, TREE if case["kind"] == "commit" else 1) for c, k in zip(ctx, n)]
    pages = [-(-r // page) for r in room]
    st["ld_table"] = max(pages)
    n_pages = sum(pages) + 3
    order = torch.randperm(n_pages, generator=g, device=DEV).to(I32)
    table = torch.zeros(B, st["ld_table"], dtype=I32, device=DEV)
    at = 0
    for b in range(B):
        table[b, :pages[b]] = order[at:at + pages[b]]
        at += pages[b]
    st["table"], st["n_pages"] = table, n_pages
    layers = case.get("layers", 1)
    dt = BF16 if case["bf16"] else F32
    for name in ("k", "v"):
        st[name] = _normal(g, layers, n_pages, n_kv, page, hd).to(dt)
    if case["kind"] == "commit":
        tokens = torch.randint(0, 151936, (all_rows,), generator=g, device=DEV, dtype=I32)
        st["tokens"], st["picks"] = tokens, _picks(n, start, parent, tokens, host)
        st["path"] = torch.zeros(B, TREE, dtype=I32, device=DEV)
        for name in ("accepted", "next", "new_len"):
            st[name] = torch.zeros(B, dtype=I32, device=DEV)
        return st
    n_q, head = case["n_q"], hd * (2 if case["gated"] else 1)
    if case["kind"] == "append":
        rot, axes = case["rot"], case["axes"]
        st["ld"] = n_q * head + 2 * n_kv * hd + case["pad"]
        st["qkv"] = _normal(g, all_rows, st["ld"])
        st["qn"], st["kn"] = _normal(g, hd, std=0.2), _normal(g, hd, std=0.2)
        st["n_pos"] = max(room) + 8
        inv = 1e6 ** (-torch.arange(0, max(rot, 2), 2, dtype=F64, device=DEV) / max(rot, 2))
        angle = torch.arange(st["n_pos"], dtype=F64, device=DEV)[:, None] * inv
        st["cos"], st["sin"] = torch.cos(angle).to(F32), torch.sin(angle).to(F32)
        st["positions"] = st["pair_axis"] = None
        if axes > 1:
            # text has one position for all axes, an image its row and column too
            st["positions"] = torch.randint(0, st["n_pos"], (axes, all_rows), generator=g,
                                            device=DEV, dtype=I32)
            st["pair_axis"] = _ints([j % axes for j in range(max(rot // 2, 1))])
        st["q_out"] = torch.zeros(all_rows, n_q * hd + case["pad"], dtype=F32, device=DEV)
        return st
    st["q"] = _normal(g, all_rows, n_q * hd + case["pad"])
    # queries that look at some of the keys harder than at others
    st["q"] *= torch.rand(all_rows, 1, generator=g, device=DEV) * 2 + 0.5
    st["qkv"] = _normal(g, all_rows, n_q * head) if case["gated"] else None
    st["out"] = torch.zeros(all_rows, n_q * hd + case["pad"], dtype=F32, device=DEV)
    return st


def _picks(n, start, parent, tokens, host):
    """The target's greedy tokens: most nodes are followed by one of their
    children's, as a drafter that is often right has it."""
    picks = [host.randrange(151936) for _ in range(tokens.shape[0])]
    drafted = tokens.tolist()
    for b, k in enumerate(n):
        kids = {}
        for i in range(1, k):
            kids.setdefault(parent[start[b] + i], []).append(i)
        for i, c in kids.items():
            if i >= 0 and host.random() < 0.85:
                picks[start[b] + i] = drafted[start[b] + host.choice(c)]
    return _ints(picks)


def _prepare_deltanet(case, st, g, host, parent):
    B, H = case["B"], case["H"]
    C = 3 * H * D
    st["ldp"] = 4 * H * D + 2 * H + case["pad"]
    st["proj"] = _normal(g, st["all_rows"], st["ldp"])
    st["conv"] = _normal(g, B, 3, C)
    st["conv_w"] = _normal(g, 4, C, std=0.4)
    st["A_log"] = torch.log(torch.rand(H, generator=g, device=DEV) * 15 + 1)
    dt = torch.exp(torch.rand(H, generator=g, device=DEV) * math.log(100.0) + math.log(1e-3))
    st["dt"] = torch.log(torch.expm1(dt))
    st["norm"] = 1 + _normal(g, D, std=0.1)
    st["state"] = _normal(g, B, H, D, D, std=0.1)
    st["out"] = torch.zeros(st["all_rows"], H * D, dtype=F32, device=DEV)
    if case["commit"]:
        # paths from the roots down, of any length up to the deepest node's
        path, accepted = [], []
        for b, k in enumerate(st["n"]):
            one, cur = [], -1
            for i in range(k):
                p = parent[st["start"][b] + i] if parent else i - 1
                if p == cur and host.random() < 0.9:
                    one.append(i)
                    cur = i
            path.append(one + [-1] * (TREE - len(one)))
            accepted.append(len(one))
        st["path"], st["accepted"], st["paths"] = _ints(path), _ints(accepted), accepted
    return st


# ---- the framework's calls -----------------------------------------------------


def _ptr(t):
    return None if t is None else t.data_ptr()


def _batch(hip, st):
    if "batch" not in st:
        st["batch"] = hip.RowBatch(st["case"]["B"], st["all_rows"], _ptr(st["row_start"]),
                                   _ptr(st["ctx_len"]), _ptr(st["parent"]))
    return st["batch"]


def _pages(hip, st):
    if "pages" not in st:
        c = st["case"]
        st["pages"] = hip.KvPages(_ptr(st["k"]), _ptr(st["v"]), 1 if c["bf16"] else 0,
                                  st["n_pages"], c["page"], c["n_kv"], c["hd"], _ptr(st["table"]),
                                  st["ld_table"])
    return st["pages"]


def _work(st, hip, query, *sizes):
    """The workspace that a program keeps for its calls of one size."""
    if "work" not in st:
        n = getattr(hip.lib(), query)(*sizes)
        st["work"] = torch.empty(max(n, 16), dtype=torch.uint8, device=DEV)
    return st["work"]


def _run_own(st):
    from quicklm_amd import hip

    c, stream = st["case"], torch.cuda.current_stream().cuda_stream
    batch = _batch(hip, st)
    if c["kind"] == "append":
        hip.call("qlm_paged_append", _ptr(st["qkv"]), st["ld"], _ptr(st["qn"]), _ptr(st["kn"]),
                 _ptr(st["cos"]), _ptr(st["sin"]), st["n_pos"], c["rot"], _ptr(st["positions"]),
                 st["all_rows"], _ptr(st["pair_axis"]), c["axes"], batch, _pages(hip, st),
                 _ptr(st["q_out"]), st["q_out"].shape[1], c["n_q"], c["gated"], stream)
        return [st["q_out"], st["k"], st["v"]]
    if c["kind"] == "attention":
        work = _work(st, hip, "qlm_paged_attention_workspace_bytes", st["all_rows"], c["B"],
                     c["n_q"], c["n_kv"], c["hd"], st["ld_table"] * c["page"])
        gate = st["qkv"][:, c["hd"]:] if c["gated"] else None
        hip.call("qlm_paged_attention", _ptr(st["q"]), st["q"].shape[1], batch, _pages(hip, st),
                 _ptr(gate), gate.stride(0) if c["gated"] else 0, 2 * c["hd"], _ptr(st["out"]),
                 st["out"].shape[1], c["n_q"], _ptr(work), work.numel(), stream)
        return [st["out"]]
    if c["kind"] == "commit":
        hip.call("qlm_tree_commit", _ptr(st["tokens"]), _ptr(st["picks"]), batch, _pages(hip, st),
                 c["layers"], st["k"].stride(0), _ptr(st["path"]), TREE, _ptr(st["accepted"]),
                 _ptr(st["next"]), _ptr(st["new_len"]), stream)
        return [st["path"], st["accepted"], st["next"], st["new_len"], st["k"], st["v"]]
    H = c["H"]
    if c["commit"]:
        hip.call("qlm_deltanet_tree_commit", _ptr(st["proj"]), st["ldp"], batch, _ptr(st["path"]),
                 TREE, _ptr(st["accepted"]), _ptr(st["conv"]), _ptr(st["conv_w"]),
                 _ptr(st["A_log"]), _ptr(st["dt"]), _ptr(st["state"]), H, D, stream)
        return [st["state"], st["conv"]]
    work = _work(st, hip, "qlm_deltanet_tree_workspace_bytes", st["all_rows"], H, D)
    hip.call("qlm_deltanet_tree", _ptr(st["proj"]), st["ldp"], batch, _ptr(st["conv"]),
             _ptr(st["conv_w"]), _ptr(st["A_log"]), _ptr(st["dt"]), _ptr(st["norm"]),
             _ptr(st["state"]), _ptr(st["out"]), H * D, H, D, _ptr(work), work.numel(), stream)
    return [st["out"]]


# ---- the plain forms -----------------------------------------------------------


def _family(st):
    """[B, T, T] truth values: node j is i or above it (all rows of a sequence
    in order where there is no tree), and [B, T]: the rows that are in the tree."""
    B, T = st["case"]["B"], max(max(st["n"]), 1)
    at = torch.arange(T, device=DEV)
    rows = st["row_start"][:-1, None].to(I64) + at
    live = at < (st["row_start"][1:] - st["row_start"][:-1])[:, None]
    if st["parent"] is None:
        return live[:, :, None] & (at[:, None] >= at), live
    parent = st["parent"][rows.clamp(max=st["all_rows"] - 1)].to(I64)
    parent = torch.where(live, parent, torch.full_like(parent, -2))
    up = (parent[:, :, None] == at).to(F32)
    up = up + torch.eye(T, device=DEV)
    for _ in range(max(T - 1, 1).bit_length()):
        up = (up @ up).clamp(max=1.0)
    live = live & ((up * (parent == -1)[:, None].to(F32)).sum(2) > 0)
    return (up > 0) & live[:, :, None], live


def _slots(st, b, first, count):
    """Page and place of `count` positions of sequence b."""
    page = st["case"]["page"]
    p = torch.arange(first, first + count, device=DEV)
    return st["table"][b].to(I64)[p // page], p % page


def _append(st):
    c = st["case"]
    hd, n_q, n_kv, rot = c["hd"], c["n_q"], c["n_kv"], c["rot"]
    total, half = st["total"], c["rot"] // 2
    x = st["qkv"][:total]
    head = hd * (2 if c["gated"] else 1)
    q = x[:, :n_q * head].reshape(total, n_q, head)[:, :, :hd]
    k = x[:, n_q * head:n_q * head + n_kv * hd].reshape(total, n_kv, hd)
    v = x[:, n_q * head + n_kv * hd:n_q * head + 2 * n_kv * hd].reshape(total, n_kv, hd)
    q = q * torch.rsqrt(q.square().mean(2, keepdim=True) + EPS) * (1 + st["qn"])
    k = k * torch.rsqrt(k.square().mean(2, keepdim=True) + EPS) * (1 + st["kn"])
    if half:
        if st["positions"] is not None:
            axis = st["pair_axis"].to(I64)
            pos = st["positions"][:, :total].to(I64)[axis].t()
        else:
            family, live = _family(st)
            depth = family.sum(2) - 1
            pos = torch.cat([st["ctx"][b] + depth[b, :st["n"][b]] for b in range(c["B"])])
            pos = pos[:, None].expand(total, half)
        j = torch.arange(half, device=DEV)
        cos, sin = st["cos"][pos, j][:, None], st["sin"][pos, j][:, None]
        q, k = ([torch.cat([t[..., :half] * cos - t[..., half:rot] * sin,
                            t[..., half:rot] * cos + t[..., :half] * sin, t[..., rot:]], 2)
                 for t in (q, k)])
    live = torch.cat([l[:m] for l, m in zip(_family(st)[1], st["n"])]) if c["tree"] else None
    if live is not None:
        q = torch.where(live[:, None, None], q, torch.zeros_like(q))
    st["q_out"][:total, :n_q * hd] = q.reshape(total, n_q * hd)
    for b in range(c["B"]):
        s, m = st["start"][b], st["n"][b]
        page, place = _slots(st, b, st["ctx"][b], m)
        for pool, new in (("k", k), ("v", v)):
            rows = new[s:s + m].to(st[pool].dtype)
            if live is not None:
                rows = torch.where(live[s:s + m, None, None], rows, st[pool][0, page, :, place])
            st[pool][0, page, :, place] = rows
    return [st["q_out"], st["k"], st["v"]]


def _attention(st):
    c = st["case"]
    hd, n_q, n_kv = c["hd"], c["n_q"], c["n_kv"]
    family, live = _family(st)
    for b in range(c["B"]):
        s, m, ctx = st["start"][b], st["n"][b], st["ctx"][b]
        if m == 0:
            continue
        page, place = _slots(st, b, 0, ctx + m)
        k, v = (st[p][0, page, :, place].to(F32).permute(1, 0, 2) for p in ("k", "v"))
        q = st["q"][s:s + m, :n_q * hd].reshape(m, n_kv, -1, hd).permute(1, 2, 0, 3)
        seen = torch.ones(m, ctx + m, dtype=torch.bool, device=DEV)
        seen[:, ctx:] = family[b, :m, :m]
        score = q @ k[:, None].transpose(2, 3).contiguous() / math.sqrt(hd)
        score = torch.where(seen, score, torch.full_like(score, float("-inf")))
        p = torch.exp(score - score.amax(3, keepdim=True))
        o = (p @ v[:, None]) / p.sum(3, keepdim=True)
        o = torch.where(live[b, :m, None], o, torch.zeros_like(o))
        o = o.permute(2, 0, 1, 3).reshape(m, n_q, hd)
        if c["gated"]:
            gate = st["qkv"][s:s + m].reshape(m, n_q, 2 * hd)[:, :, hd:]
            o = o / (1 + torch.exp(-gate))
        st["out"][s:s + m, :n_q * hd] = o.reshape(m, n_q * hd)
    return [st["out"]]


def _commit(st):
    c = st["case"]
    B, T, page = c["B"], max(max(st["n"]), 1), c["page"]
    at = torch.arange(T, device=DEV)
    rows = (st["row_start"][:-1, None] + at).to(I64).clamp(max=st["all_rows"] - 1)
    n = (st["row_start"][1:] - st["row_start"][:-1])[:, None]
    parent = torch.where(at < n, st["parent"][rows], torch.full_like(rows, -2, dtype=I32))
    tokens, picks = st["tokens"][rows], st["picks"][rows]
    b = torch.arange(B, device=DEV)
    # the root is the token that the last step chose: accepted as it is
    cur = torch.where(parent[:, 0] == -1, 0, -1).to(I64)
    st["path"].fill_(-1)
    st["next"].fill_(-1)
    count = torch.zeros(B, dtype=I64, device=DEV)
    for step in range(T):
        there = cur >= 0
        st["path"][:, step] = cur.to(I32)
        count += there
        pick = picks[b, cur.clamp(min=0)]
        st["next"].copy_(torch.where(there, pick, st["next"]))
        child = (parent == cur[:, None]) & (tokens == pick[:, None]) & there[:, None] & (at > 0)
        first = torch.where(child, at, torch.full_like(at, T)).amin(1)
        cur = torch.where(first < T, first, torch.full_like(first, -1))
    st["accepted"].copy_(count)
    st["new_len"].copy_(st["ctx_len"] + count)
    # places beyond the path keep what they hold
    step = torch.arange(T, device=DEV)
    taken = (step < count[:, None]) & (step > 0)
    to = st["ctx_len"][:, None].to(I64) + step
    frm = torch.where(taken, st["ctx_len"][:, None] + st["path"][:, :T], to.to(I32)).to(I64)
    tp, fp = (torch.gather(st["table"].to(I64), 1, x // page) for x in (to, frm))
    for pool in ("k", "v"):
        st[pool][:, tp, :, to % page] = st[pool][:, fp, :, frm % page]
    return [st["path"], st["accepted"], st["next"], st["new_len"], st["k"], st["v"]]


def _silu(x):
    return x / (1 + torch.exp(-x))


def _deltanet(st):
    c = st["case"]
    B, H, commit = c["B"], c["H"], c["commit"]
    T = max(max(st["paths"]) if commit else max(st["n"]), 1)
    at = torch.arange(T, device=DEV)
    base = st["row_start"][:-1, None].to(I64)
    if commit:
        node = st["path"][:, :T].to(I64)
        live = at < st["accepted"][:, None]
        parent = torch.where(live, at - 1, torch.full_like(at, -2)).to(I64)
        rows = (base + node.clamp(min=0)).clamp(max=st["all_rows"] - 1)
    else:
        family, live = _family(st)
        rows = (base + at).clamp(max=st["all_rows"] - 1)
        parent = (at - 1).expand(B, T) if st["parent"] is None else st["parent"][rows].to(I64)
        parent = torch.where(live, parent, torch.full_like(parent, -2))
    C = 3 * H * D
    x = st["proj"][rows]  # [B, T, ldp]
    b = torch.arange(B, device=DEV)
    # the ring: row (position + j) % 3 holds the input j - 3 places back
    ring = torch.stack([st["conv"][b, (st["ctx_len"].to(I64) + j) % 3] for j in range(3)], 1)
    past = [x[:, :, :C]]
    for k in range(1, 4):  # inputs k places above each node
        up = past[-1][b[:, None], parent.clamp(min=0)]
        past.append(torch.where((parent >= 0)[:, :, None], up, ring[:, 3 - k, None]))
    y = sum(past[3 - j] * st["conv_w"][j] for j in range(4))
    y = _silu(y).reshape(B, T, 3, H, D)
    q, k, v = y[:, :, 0], y[:, :, 1], y[:, :, 2]
    q = q / torch.sqrt(q.square().sum(3, keepdim=True) + EPS)
    k = k / torch.sqrt(k.square().sum(3, keepdim=True) + EPS)
    z = x[:, :, C:C + H * D].reshape(B, T, H, D)
    beta = 1 / (1 + torch.exp(-x[:, :, 4 * H * D:4 * H * D + H]))
    dt = x[:, :, 4 * H * D + H:4 * H * D + 2 * H] + st["dt"]
    soft = torch.where(dt > 20, dt, torch.log1p(torch.exp(dt.clamp(max=20))))
    decay = torch.exp(-torch.exp(st["A_log"]) * soft)
    states = None if commit else x.new_empty(B, T, H, D, D)
    S, outs = st["state"], []
    for t in range(T):
        if not commit:
            p = parent[:, t]
            S = torch.where((p >= 0)[:, None, None, None], states[b, p.clamp(min=0)], st["state"])
        was = S
        S = S * decay[:, t, :, None, None]
        w = (v[:, t] - (S * k[:, t, :, :, None]).sum(2)) * beta[:, t, :, None]
        S = S + k[:, t, :, :, None] * w[:, :, None, :]
        if commit:
            S = torch.where(live[:, t, None, None, None], S, was)
        else:
            states[:, t] = S
        outs.append((S * q[:, t, :, :, None]).sum(2) / math.sqrt(D))
    if commit:
        st["state"].copy_(S)
        count, pos = st["accepted"].to(I64), st["ctx_len"].to(I64)
        line = torch.cat([ring, x[:, :, :C]], 1)  # the last three before the path, then it
        for j in range(3):
            st["conv"][b, (pos + count + j) % 3] = line[b, count + j]
        return [st["state"], st["conv"]]
    o = torch.stack(outs, 1)
    o = o * torch.rsqrt(o.square().mean(3, keepdim=True) + EPS) * st["norm"] * _silu(z)
    o = torch.where(live[:, :, None, None], o, torch.zeros_like(o)).reshape(B, T, H * D)
    for i, m in enumerate(st["n"]):
        st["out"][st["start"][i]:st["start"][i] + m] = o[i, :m]
    return [st["out"]]


def run(state: dict):
    if own:
        return _run_own(state)
    return dict(append=_append, attention=_attention, commit=_commit,
                deltanet=_deltanet)[state["case"]["kind"]](state)


def work(case: dict) -> dict:
    n, ctx = _lens(case)
    total, size = sum(n), 2 if case.get("bf16") else 4
    if case["kind"] == "append":
        hd, heads = case["hd"], case["n_q"] + 2 * case["n_kv"]
        return {"bytes": total * hd * (4 * heads + 4 * case["n_q"] + 2 * case["n_kv"] * size),
                "flops": 8 * total * hd * (case["n_q"] + case["n_kv"])}
    if case["kind"] == "attention":
        hd, n_q, n_kv = case["hd"], case["n_q"], case["n_kv"]
        keys = sum(c + m for c, m in zip(ctx, n) if m)
        pairs = sum(m * c + m * (m + 1) // 2 for c, m in zip(ctx, n))
        return {"bytes": 2 * keys * n_kv * hd * size
                + 4 * total * n_q * hd * (3 if case["gated"] else 2),
                "flops": 4 * hd * n_q * pairs}
    if case["kind"] == "commit":
        # a path's rows read and written: of a tree of k nodes about 4 log2 k
        moved = sum(min(k - 1, int(2 * math.log2(k))) for k in n if k > 1)
        row = 2 * 2 * case["layers"] * case["n_kv"] * case["hd"] * size
        return {"bytes": moved * row + 16 * sum(n), "flops": sum(n)}
    H, B = case["H"], case["B"]
    inputs, state = 4 * (4 * H * D + 2 * H), 4 * H * D * D
    if case["commit"]:
        moved = sum(min(k, 1 + int(2 * math.log2(k))) for k in n if k)
        return {"bytes": moved * 4 * (3 * H * D + 2 * H) + 2 * B * state + 8 * 9 * B * H * D,
                "flops": 6 * D * D * H * moved}
    return {"bytes": total * (inputs + 4 * H * D) + B * state + 4 * 9 * B * H * D,
            "flops": 6 * D * D * H * total}


# ---- the definitions in 64 bits ------------------------------------------------


def _above(st, b):
    """For each row of sequence b the rows from its root down to itself, or
    None for a row outside the tree; found on the host, a row at a time."""
    s, m = st["start"][b], st["n"][b]
    if st["parent"] is None:
        return [list(range(i + 1)) for i in range(m)]
    parent, chains = st["parent"][s:s + m].tolist(), []
    for i, p in enumerate(parent):
        if p == -1:
            chains.append([i])
        elif 0 <= p < i and chains[p] is not None:
            chains.append(chains[p] + [i])
        else:
            chains.append(None)
    return chains


def _exact_append(st):
    c = st["case"]
    hd, n_q, n_kv, half = c["hd"], c["n_q"], c["n_kv"], c["rot"] // 2
    head = hd * (2 if c["gated"] else 1)
    q_out, pools = st["q_out"].double(), [st["k"].double(), st["v"].double()]
    for b in range(c["B"]):
        chains = _above(st, b) if c["tree"] else None
        live = [i for i in range(st["n"][b]) if not c["tree"] or chains[i] is not None]
        if not live:
            continue
        at = torch.tensor(live, device=DEV)
        x = st["qkv"][st["start"][b] + at].double()
        if st["positions"] is None:
            depth = [len(chains[i]) - 1 for i in live] if c["tree"] else live
            pos = (torch.tensor(depth, device=DEV) + st["ctx"][b])[:, None].expand(-1, half)
        else:
            pos = st["positions"][:, st["start"][b] + at].long()
            pos = torch.stack([pos[a] for a in st["pair_axis"].tolist()], 1)[:, :half]
        # a pair of elements is a complex number, turned by its position's angle
        j = torch.arange(half, device=DEV)
        turn = torch.complex(st["cos"][pos, j].double(), st["sin"][pos, j].double())
        k0 = n_q * head
        parts = [(x[:, i * head:i * head + hd], st["qn"], ("q", i)) for i in range(n_q)]
        parts += [(x[:, k0 + i * hd:k0 + (i + 1) * hd], st["kn"], ("k", i)) for i in range(n_kv)]
        k0 += n_kv * hd
        parts += [(x[:, k0 + i * hd:k0 + (i + 1) * hd], None, ("v", i)) for i in range(n_kv)]
        slot = at + st["ctx"][b]
        page, place = st["table"][b].long()[slot // c["page"]], slot % c["page"]
        for t, gain, (name, i) in parts:
            if gain is not None:
                t = t / torch.sqrt((t * t).sum(1, keepdim=True) / hd + EPS) * (gain.double() + 1)
                turned = torch.complex(t[:, :half].contiguous(),
                                       t[:, half:2 * half].contiguous()) * turn
                t = torch.cat([turned.real, turned.imag, t[:, 2 * half:]], 1)
            if name == "q":
                q_out[st["start"][b] + at, i * hd:(i + 1) * hd] = t
            else:
                pools[name == "v"][0, page, i, place] = t
    return [q_out] + pools


def _exact_attention(st):
    c = st["case"]
    hd, n_q, n_kv, page = c["hd"], c["n_q"], c["n_kv"], c["page"]
    G = n_q // n_kv
    out = st["out"].double()
    for b in range(c["B"]):
        s, m, ctx = st["start"][b], st["n"][b], st["ctx"][b]
        if not m:
            continue
        bias = torch.full((m, ctx + m), -math.inf, dtype=F64)
        if c["tree"]:
            chains = _above(st, b)
            for i, chain in enumerate(chains):
                bias[i, :ctx] = 0
                bias[i, [ctx + j for j in chain or range(m)]] = 0
            dead = torch.tensor([chain is None for chain in chains], device=DEV)
        else:
            bias = torch.triu(bias, ctx + 1).nan_to_num(nan=0.0, neginf=-math.inf)
            dead = torch.zeros(m, dtype=torch.bool, device=DEV)
        bias = bias.to(DEV)
        pages = -(-(ctx + m) // page)
        for g in range(n_kv):
            k, v = (st[p][0, st["table"][b, :pages].long(), g].reshape(pages * page, hd)
                    [:ctx + m].double() for p in ("k", "v"))
            for h in range(g * G, (g + 1) * G):
                e = torch.mm(st["q"][s:s + m, h * hd:(h + 1) * hd].double(), k.t().contiguous())
                o = torch.mm(torch.softmax(e * hd ** -0.5 + bias, 1), v)
                if c["gated"]:
                    o = o * torch.sigmoid(
                        st["qkv"][s:s + m, (2 * h + 1) * hd:(2 * h + 2) * hd].double())
                out[s:s + m, h * hd:(h + 1) * hd] = o.masked_fill(dead[:, None], 0.0)
    return [out]


def _exact_commit(st):
    c = st["case"]
    tokens, picks = st["tokens"].tolist(), st["picks"].tolist()
    parent = st["parent"].tolist()
    path, accepted, nxt = [], [], []
    k, v = st["k"].double(), st["v"].double()
    for b in range(c["B"]):
        s, m, ctx = st["start"][b], st["n"][b], st["ctx"][b]
        one = [0] if m and parent[s] == -1 else []
        while one:
            kids = [i for i in range(1, m) if parent[s + i] == one[-1]
                    and tokens[s + i] == picks[s + one[-1]]]
            if not kids:
                break
            one.append(kids[0])
        table = st["table"][b].tolist()
        for pool in (k, v):
            was = [pool[:, table[(ctx + i) // c["page"]], :, (ctx + i) % c["page"]].clone()
                   for i in one]
            for i, row in enumerate(was):
                pool[:, table[(ctx + i) // c["page"]], :, (ctx + i) % c["page"]] = row
        path.append(one + [-1] * (TREE - len(one)))
        accepted.append(len(one))
        nxt.append(picks[s + one[-1]] if one else -1)
    return [_ints(path), _ints(accepted), _ints(nxt),
            _ints([a + x for a, x in zip(accepted, st["ctx"])]), k, v]


def _exact_deltanet(st):
    c = st["case"]
    H, C = c["H"], 3 * c["H"] * D
    out, state, conv = st["out"].double(), st["state"].double(), st["conv"].double()
    w = st["conv_w"].double()
    for b in range(c["B"]):
        s, m, ctx = st["start"][b], st["n"][b], st["ctx"][b]
        if c["commit"]:
            nodes = st["path"][b, :st["paths"][b]].tolist()
            chains = [list(range(i + 1)) for i in range(len(nodes))]
        else:
            whole = _above(st, b)
            nodes = [i for i in range(m) if whole[i] is not None]
            new = {i: j for j, i in enumerate(nodes)}
            chains = [[new[i] for i in whole[k]] for k in nodes]
        n = len(nodes)
        if not n:
            continue
        x = st["proj"][[s + i for i in nodes]].double()
        old = [conv[b, (ctx + j) % 3].clone() for j in range(3)]
        # each node's line of four inputs
        y = torch.stack([sum(w[3 - i] * r for i, r in enumerate(
            ([x[j, :C] for j in reversed(chain)] + old[::-1])[:4])) for chain in chains])
        y = (y * torch.sigmoid(y)).reshape(n, 3, H, D).permute(1, 2, 0, 3)  # [3, H, n, D]
        q, k = (t / torch.sqrt((t * t).sum(2, keepdim=True) + EPS) for t in (y[0], y[1]))
        beta = torch.sigmoid(x[:, 4 * H * D:4 * H * D + H]).t()
        alpha = -(torch.exp(st["A_log"].double())
                  * torch.nn.functional.softplus(x[:, 4 * H * D + H:4 * H * D + 2 * H]
                                                 + st["dt"].double())).t()
        above = torch.zeros(n, n, dtype=F64)
        for i, chain in enumerate(chains):
            above[i, chain] = 1
        above = above.to(DEV)
        # all nodes at once: S_t = g_t S + sum over its line of (g_t / g_s) k_s u_s
        g = torch.matmul(alpha, above.t().contiguous())  # [H, n], logarithms
        ratio = torch.exp(torch.where(above > 0, g[:, :, None] - g[:, None], -math.inf))
        S0 = state[b]
        kk = torch.matmul(k, k.transpose(1, 2).contiguous()) * ratio
        A = torch.tril(beta[:, :, None] * kk, -1) + torch.eye(n, dtype=F64, device=DEV)
        rhs = beta[:, :, None] * (y[2] - torch.exp(g)[:, :, None] * torch.matmul(k, S0))
        u = torch.linalg.solve_triangular(A, rhs, upper=False, unitriangular=True)
        if c["commit"]:
            end = ratio[:, -1, :, None]
            state[b] = (torch.exp(g[:, -1])[:, None, None] * S0
                        + torch.matmul((k * end).transpose(1, 2).contiguous(), u))
            line = old + [x[j, :C] for j in range(n)]
            for j in range(3):
                conv[b, (ctx + n + j) % 3] = line[n + j]
            continue
        o = torch.exp(g)[:, :, None] * torch.matmul(q, S0)
        o = o + torch.matmul(torch.matmul(q, k.transpose(1, 2).contiguous()) * ratio, u)
        o = o / math.sqrt(D)
        o = o / torch.sqrt((o * o).sum(2, keepdim=True) / D + EPS) * st["norm"].double()
        z = x[:, C:C + H * D].reshape(n, H, D).permute(1, 0, 2)
        o = o * z * torch.sigmoid(z)
        out[s:s + m] = 0.0
        out[[s + i for i in nodes]] = o.permute(1, 0, 2).reshape(n, H * D)
    return [state, conv] if c["commit"] else [out]


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    return dict(append=_exact_append, attention=_exact_attention, commit=_exact_commit,
                deltanet=_exact_deltanet)[case["kind"]](st)
