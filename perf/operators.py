"""Operators for scoring a prompt with activations in 8 bits, as measurable
cases.

  norm      residual addition, RMSNorm and an output in 8 bits with one scale
            a row (qlm_add_rms_norm_q8)
  matmul    matrix product of 8-bit rows and 8-bit weights with one scale a row
            and one a channel (qlm_matmul_a8)
  logprobs  log probabilities of given tokens, entropy and the top alternatives
            of rows of logits (qlm_token_logprobs)

`run` computes the operators' plain form with elementary torch operations, or,
where `own` is true, calls the kernel library.
"""

from __future__ import annotations

import random

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
EPS = 1e-6
STORE, RESIDUAL, SWIGLU = 0, 1, 2
F32, F64, I8, I32, I64 = torch.float32, torch.float64, torch.int8, torch.int32, torch.int64

MAX_NORM = 8192 * 4096  # elements of the largest norm
MAX_MATMUL = 2 * 4096 * 12288 * 4096  # operations of the largest product
MAX_LOGITS = 2047 * 151936  # logits of the largest scoring call


def listed():
    return [
        # One decode step of a 4B-class model (hidden 2560): pure latency.
        dict(name="norm_1x2560", kind="norm", rows=1, n=2560, pad=0, add=True),
        # The norm before a 2048-token prompt's MLP.
        dict(name="norm_2048x2560", kind="norm", rows=2048, n=2560, pad=0, add=True),
        # The first norm of a batch of odd rows taken out of wider ones.
        dict(name="norm_333x1001_strided", kind="norm", rows=333, n=1001, pad=37, add=False),
        # Several prompts packed into one prefill of a wider model.
        dict(name="norm_8192x4096", kind="norm", rows=8192, n=4096, pad=0, add=True),
        # One decode step's gate/up projection: the weights' stream.
        dict(name="matmul_1x9728x2560_swiglu", kind="matmul", M=1, N=9728, K=2560, pad=0,
             epilogue=SWIGLU),
        # A serving batch of 16: the down projection into the residual stream.
        dict(name="matmul_16x2560x9728_residual", kind="matmul", M=16, N=2560, K=9728, pad=0,
             epilogue=RESIDUAL),
        # A short ragged prompt through an odd-sized projection, rows padded.
        dict(name="matmul_77x5003x1088", kind="matmul", M=77, N=5003, K=1088, pad=13,
             epilogue=STORE),
        # A 2048-token prompt's gate/up projection.
        dict(name="matmul_2048x9728x2560_swiglu", kind="matmul", M=2048, N=9728, K=2560, pad=0,
             epilogue=SWIGLU),
        # The widest isolated product of the benchmark shapes, for packed prompts.
        dict(name="matmul_4096x12288x4096", kind="matmul", M=4096, N=12288, K=4096, pad=0,
             epilogue=STORE),
        # Sampling: the alternatives beside one decoded token.
        dict(name="logprobs_1x151936_top20", kind="logprobs", rows=1, vocab=151936, pad=0, ids=1,
             top=20, masked=False),
        # Constrained decoding of a batch: most tokens masked to -inf, one row
        # with fewer tokens left than alternatives asked for, one with none.
        dict(name="logprobs_37x32003_masked", kind="logprobs", rows=37, vocab=32003, pad=5, ids=4,
             top=64, masked=True),
        # Scoring a 2048-token prompt: every next token's log probability.
        dict(name="logprobs_2047x151936_top5", kind="logprobs", rows=2047, vocab=151936, pad=0,
             ids=1, top=5, masked=False),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["norm", "matmul", "logprobs"])
    if kind == "norm":
        n = _log(rng, 64, 16384)
        return dict(kind=kind, rows=_log(rng, 1, min(8192, MAX_NORM // n)), n=n,
                    pad=rng.choice([0, 0, rng.randint(1, 64)]), add=rng.random() < 0.7)
    if kind == "matmul":
        N, K = _log(rng, 48, 12288), 64 * _log(rng, 1, 152)
        epilogue = rng.choice([STORE, RESIDUAL, SWIGLU])
        most = MAX_MATMUL // (2 * N * K * (2 if epilogue == SWIGLU else 1))
        return dict(kind=kind, M=_log(rng, 1, min(4096, most)), N=N, K=K,
                    pad=rng.choice([0, 0, rng.randint(1, 64)]), epilogue=epilogue)
    vocab = _log(rng, 1000, 151936)
    return dict(kind=kind, rows=_log(rng, 1, min(2047, MAX_LOGITS // vocab)), vocab=vocab,
                pad=rng.choice([0, 0, rng.randint(1, 64)]), ids=rng.choice([1, 1, 4, 8]),
                top=rng.choice([0, 1, 5, 20, 64]), masked=rng.random() < 0.3)


# ---- inputs --------------------------------------------------------------------


def _normal(g, *shape, mean=0.0, std=1.0):
    t = torch.randn(*shape, generator=g, device=DEV, dtype=F32)
    return t.mul_(std).add_(mean)


def _quantised(t):
    """Rows in 8 bits with one scale each, as the framework keeps its weights."""
    s = t.abs().amax(1, keepdim=True) / 127
    return torch.round(t / s).to(I8), s[:, 0].contiguous()


def _tile_major(w, halves):
    """The weight layout of qlm_mx_swizzle: 16-row x 64-column fragments, the
    rows of each half padded with zeros to whole tiles."""
    rows, K = w.shape[0] // halves, w.shape[1]
    tiles = -(-rows // 16)
    p = torch.zeros(halves, tiles * 16, K, dtype=I8, device=w.device)
    p[:, :rows] = w.view(halves, rows, K)
    return p.view(halves * tiles, 16, K // 64, 4, 16).permute(0, 2, 3, 1, 4).contiguous()


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    st = dict(case=case)
    pad = case["pad"]
    if case["kind"] == "norm":
        rows, n = case["rows"], case["n"]
        # a residual stream: a few channels much larger than the others
        x = _normal(g, rows, n + pad)
        x[:, ::251] *= 20.0
        st["x"] = x
        st["delta"] = _normal(g, rows, n + pad, std=0.5) if case["add"] else None
        st["w"] = _normal(g, n, std=0.1)
        st["sum"] = torch.empty_like(x) if case["add"] else None
        st["q"] = torch.zeros(rows, n + pad, dtype=I8, device=DEV)
        st["scales"] = torch.zeros(rows, dtype=F32, device=DEV)
        st["values"] = torch.zeros(rows, n, dtype=F32, device=DEV)
    elif case["kind"] == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        halves = 2 if case["epilogue"] == SWIGLU else 1
        st["w"], st["w_scales"] = _quantised(_normal(g, halves * N, K, std=0.02))
        st["tiles"] = _tile_major(st["w"], halves)
        # a row's 8-bit activations have their own scale; rows 16-byte aligned
        st["x"] = torch.zeros(M, K + 16 * (pad % 4), dtype=I8, device=DEV)
        st["x"][:, :K], st["x_scales"] = _quantised(_normal(g, M, K))
        st["y"] = _normal(g, M, N + pad)
    else:
        rows, V = case["rows"], case["vocab"]
        # rows from flat to peaked distributions
        logits = _normal(g, rows, V + pad)
        logits *= torch.rand(rows, 1, generator=g, device=DEV) * 5 + 1
        if case["masked"]:
            keep = torch.rand(rows, V + pad, generator=g, device=DEV) < 0.1
            keep[0] = False
            keep[0, [V // 3, V // 2, V - 1]] = True
            if rows > 1:
                keep[-1] = False
            logits.masked_fill_(~keep, float("-inf"))
        st["logits"] = logits
        st["ids"] = torch.randint(0, V, (rows, case["ids"]), generator=g, device=DEV, dtype=I32)
        st["logprobs"] = torch.zeros(rows, case["ids"], dtype=F32, device=DEV)
        st["entropy"] = torch.zeros(rows, dtype=F32, device=DEV)
        st["top_ids"] = torch.zeros(rows, case["top"], dtype=I32, device=DEV)
        st["top_logprobs"] = torch.zeros(rows, case["top"], dtype=F32, device=DEV)
    return st


# ---- the framework's calls -----------------------------------------------------


def _ptr(t):
    return None if t is None else t.data_ptr()


def _work(st, hip, query, *sizes):
    """The workspace that a program keeps for its calls of one size."""
    if "work" not in st:
        n = getattr(hip.lib(), query)(*sizes)
        st["work"] = torch.empty(max(n, 16), dtype=torch.uint8, device=DEV)
    return st["work"]


def _run_own(st):
    from quicklm_amd import hip

    c, stream = st["case"], torch.cuda.current_stream().cuda_stream
    if c["kind"] == "norm":
        ld = c["n"] + c["pad"]
        hip.call("qlm_add_rms_norm_q8", _ptr(st["x"]), ld, _ptr(st["delta"]), ld, _ptr(st["w"]),
                 EPS, _ptr(st["sum"]), ld, _ptr(st["q"]), ld, _ptr(st["scales"]), c["rows"],
                 c["n"], stream)
        # what the 8 bits stand for
        torch.mul(st["q"][:, :c["n"]], st["scales"][:, None], out=st["values"])
        out = [st["values"], st["scales"]]
        return out + [st["sum"][:, :c["n"]]] if c["add"] else out
    if c["kind"] == "matmul":
        M, N, K, e = c["M"], c["N"], c["K"], c["epilogue"]
        work = _work(st, hip, "qlm_matmul_a8_workspace_bytes", M, N, K, e)
        hip.call("qlm_matmul_a8", _ptr(st["x"]), st["x"].shape[1], _ptr(st["x_scales"]),
                 _ptr(st["tiles"]), _ptr(st["w_scales"]), _ptr(st["y"]), N + c["pad"], M, N, K, e,
                 _ptr(work), work.numel(), stream)
        return [st["y"][:, :N]]
    rows, V, top = c["rows"], c["vocab"], c["top"]
    work = _work(st, hip, "qlm_token_logprobs_workspace_bytes", rows, V, top)
    hip.call("qlm_token_logprobs", _ptr(st["logits"]), V + c["pad"], V, rows, _ptr(st["ids"]),
             c["ids"], _ptr(st["logprobs"]), _ptr(st["entropy"]), top,
             _ptr(st["top_ids"]) if top else None, _ptr(st["top_logprobs"]) if top else None,
             _ptr(work), work.numel(), stream)
    out = [st["logprobs"], st["entropy"]]
    return out + [st["top_ids"], st["top_logprobs"]] if top else out


# ---- the plain forms -----------------------------------------------------------


def _norm(st):
    c = st["case"]
    r = st["x"][:, :c["n"]]
    if c["add"]:
        r = r + st["delta"][:, :c["n"]]
    # the quotient next to a rounding border needs 64 bits
    r64 = r.to(F64)
    y = r64 * torch.rsqrt(r64.square().mean(1, keepdim=True) + EPS) * (1 + st["w"].to(F64))
    s = y.abs().amax(1, keepdim=True) / 127
    s = torch.where(s > 0, s, torch.ones_like(s))
    values = (torch.round(y / s) * s).to(F32)
    return [values, s[:, 0].to(F32), r] if c["add"] else [values, s[:, 0].to(F32)]


def _matmul(st):
    c = st["case"]
    N, K = c["N"], c["K"]
    p = st["x"][:, :K].to(F32) @ st["w"].to(F32).t()
    p = p * st["x_scales"][:, None] * st["w_scales"]
    y = st["y"][:, :N]
    if c["epilogue"] == SWIGLU:
        gate = p[:, :N]
        y.copy_(gate / (1 + torch.exp(-gate)) * p[:, N:])
    elif c["epilogue"] == RESIDUAL:
        y.add_(p)
    else:
        y.copy_(p)
    return [y]


def _logprobs(st):
    c = st["case"]
    logits = st["logits"][:, :c["vocab"]]
    d = logits - logits.amax(1, keepdim=True)
    p = torch.exp(d)
    z = p.sum(1, keepdim=True)
    logz = torch.log(z)
    # a masked token adds nothing: 0, not 0 * -inf
    pd = torch.where(p > 0, p * d, p)
    entropy = logz[:, 0] - pd.sum(1) / z[:, 0]
    out = [torch.gather(d, 1, st["ids"].to(I64)) - logz, entropy]
    if c["top"]:
        # one 64-bit key a logit, larger value first, then the lower id
        bits = (logits + 0.0).view(I32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(I64)
        at = torch.arange(c["vocab"], device=logits.device, dtype=I64)
        key = torch.topk(order * (1 << 32) + (0xFFFFFFFF - at), c["top"], dim=1).values
        ids = 0xFFFFFFFF - (key & 0xFFFFFFFF)
        out += [ids.to(I32), torch.gather(d, 1, ids) - logz]
    return out


def run(state: dict):
    if own:
        return _run_own(state)
    return {"norm": _norm, "matmul": _matmul, "logprobs": _logprobs}[state["case"]["kind"]](state)


def work(case: dict) -> dict:
    if case["kind"] == "norm":
        rows, n = case["rows"], case["n"]
        each = 4 + 1 + (8 if case["add"] else 0)  # input, 8 bits; addend and sum
        return {"bytes": rows * n * each + 4 * n + 4 * rows, "flops": 8 * rows * n}
    if case["kind"] == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        ch = N * (2 if case["epilogue"] == SWIGLU else 1)
        y = 4 * M * N * (2 if case["epilogue"] == RESIDUAL else 1)
        return {"bytes": M * K + ch * K + 4 * M + 4 * ch + y, "flops": 2 * M * ch * K}
    rows, V, ids, top = case["rows"], case["vocab"], case["ids"], case["top"]
    return {"bytes": rows * (4 * V + 8 * ids + 4 + 8 * top), "flops": 5 * rows * V}


# ---- the definitions in 64 bits ------------------------------------------------


def _exact_norm(st):
    c = st["case"]
    x = st["x"][:, :c["n"]]
    if c["add"]:
        x = x + st["delta"][:, :c["n"]]  # the sum is stored in 32 bits
    x = x.double()
    t = x * (st["w"].double() + 1.0)
    top = t.abs().max(dim=1).values
    rms = torch.sqrt((x * x).sum(1) / c["n"] + EPS)
    scale = torch.where(top > 0, top / rms / 127.0, torch.ones_like(top))
    # the root mean square is a factor of both the values and the scale
    q = torch.round(127.0 * t / torch.where(top > 0, top, torch.ones_like(top))[:, None])
    out = [q * scale[:, None], scale]
    return out + [x] if c["add"] else out


def _exact_matmul(st):
    c = st["case"]
    N = c["N"]
    a = st["x"][:, :c["K"]].double() * st["x_scales"].double()[:, None]
    b = st["w"].double() * st["w_scales"].double()[:, None]
    y = torch.mm(a, b.t().contiguous())
    if c["epilogue"] == SWIGLU:
        return [y[:, :N] * torch.sigmoid(y[:, :N]) * y[:, N:]]
    if c["epilogue"] == RESIDUAL:
        return [st["y"][:, :N].double() + y]
    return [y]


def _exact_logprobs(st):
    c = st["case"]
    rows, V, top = c["rows"], c["vocab"], c["top"]
    lp, h, tl = [], [], []
    for r in range(0, rows, 256):
        x = st["logits"][r:r + 256, :V].double()
        lsm = x - torch.logsumexp(x, 1, keepdim=True)
        lp.append(torch.gather(lsm, 1, st["ids"][r:r + 256].long()))
        h.append(-(torch.exp(lsm) * lsm.clamp_min(-1e30)).sum(1))
        if top:
            tl.append(torch.topk(lsm, top, dim=1).values)
    out = [torch.cat(lp), torch.cat(h)]
    return out + [None, torch.cat(tl)] if top else out


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    kinds = {"norm": _exact_norm, "matmul": _exact_matmul, "logprobs": _exact_logprobs}
    return kinds[case["kind"]](st)
