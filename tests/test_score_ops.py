"""Refusals of the 8-bit norm, the 8-bit matrix product and the token log
probabilities: every check runs on the host before any launch, so none of the
fake pointers below is read. No GPU call is made."""

import math

import pytest

from quicklm_amd import hip

P = 1 << 20  # 16-byte aligned, never dereferenced
ARG, SHAPE = -1, -2


def norm(**kw):
    a = dict(x=P, ldx=64, delta=P, ldd=64, w=P, eps=1e-6, sum=2 * P, lds=64, q=P, ldq=64,
             scales=P, rows=2, n=64, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return hip.lib().qlm_add_rms_norm_q8(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(x=None), ARG), (dict(w=None), ARG), (dict(q=None), ARG), (dict(scales=None), ARG),
    (dict(rows=0), ARG), (dict(rows=-1), ARG), (dict(n=0), ARG),
    (dict(ldx=63), ARG), (dict(ldd=63), ARG), (dict(lds=63), ARG), (dict(ldq=63), ARG),
    (dict(delta=None), ARG),  # a sum of one term
    (dict(eps=-1e-6), ARG), (dict(eps=math.nan), ARG),
    (dict(sum=P, x=P, ldx=65, delta=3 * P), ARG),  # in place with other rows
    (dict(sum=P, x=3 * P, ldd=65), ARG),
    (dict(rows=(1 << 21) + 1), SHAPE),
])
def test_norm_q8_refusals(kw, rc):
    assert norm(**kw) == rc


def matmul(**kw):
    a = dict(x=P, ldx=128, sx=P, q=P, sw=P, y=P, ldy=32, M=2, N=32, K=128, epilogue=0, work=P,
             work_bytes=1 << 40, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return hip.lib().qlm_matmul_a8(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(x=None), ARG), (dict(sx=None), ARG), (dict(q=None), ARG), (dict(sw=None), ARG),
    (dict(y=None), ARG), (dict(M=0), ARG), (dict(N=0), ARG), (dict(K=0), ARG), (dict(M=-3), ARG),
    (dict(epilogue=3), ARG), (dict(epilogue=-1), ARG), (dict(ldx=112), ARG), (dict(ldy=31), ARG),
    (dict(K=96), SHAPE), (dict(K=1 << 17, ldx=1 << 17), SHAPE), (dict(ldx=136), SHAPE),
    (dict(ldx=1 << 23), SHAPE), (dict(x=P + 8), SHAPE), (dict(q=P + 4), SHAPE),
    (dict(work=P + 8), SHAPE),
])
def test_matmul_a8_refusals(kw, rc):
    assert matmul(**kw) == rc


@pytest.mark.parametrize("N,K", [(32, 128), (2560, 9728), (9728, 2560), (151936, 2560),
                                 (5003, 1088), (16, 131008)])
@pytest.mark.parametrize("epilogue", [0, 1, 2])
def test_matmul_a8_workspace(N, K, epilogue):
    """A workspace for the most rows serves every call of fewer, and a short
    or missing one is refused."""
    L, last = hip.lib(), 0
    for M in [1, 2, 5, 16, 17, 32, 33, 64, 65, 100, 128, 129, 256, 300, 512, 1000, 2048, 4096]:
        b = L.qlm_matmul_a8_workspace_bytes(M, N, K, epilogue)
        assert b >= last
        last = b
        if b:
            kw = dict(M=M, N=N, K=K, ldx=K, ldy=N, epilogue=epilogue)
            assert matmul(work_bytes=b - 1, **kw) == ARG
            assert matmul(work=None, **kw) == ARG
    for bad in [(0, N, K, 0), (1, 0, K, 0), (1, N, 0, 0), (1, N, K, 3), (1, N, K, -1),
                (1, N, 96, 0), (-1, N, K, 0)]:
        assert L.qlm_matmul_a8_workspace_bytes(*bad) == 0


def logprobs(**kw):
    a = dict(logits=P, ldl=100, n=100, rows=2, ids=P, n_ids=1, lp=P, entropy=P, top=5, top_ids=P,
             top_lp=P, work=P, work_bytes=1 << 40, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return hip.lib().qlm_token_logprobs(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(logits=None), ARG), (dict(work=None), ARG), (dict(rows=0), ARG), (dict(n=0), ARG),
    (dict(ldl=99), ARG), (dict(n_ids=-1), ARG), (dict(ids=None), ARG), (dict(lp=None), ARG),
    (dict(top=-1), ARG), (dict(top_ids=None), ARG), (dict(top_lp=None), ARG),
    (dict(top=101), ARG),  # more alternatives than tokens
    (dict(n_ids=0, top=0, entropy=None), ARG),  # nothing asked for
    (dict(work_bytes=0), ARG), (dict(top=65), SHAPE),
    (dict(n=(1 << 21) + 1, ldl=1 << 22), SHAPE), (dict(rows=(1 << 23) + 1), SHAPE),
    (dict(work=P + 8), SHAPE),
])
def test_token_logprobs_refusals(kw, rc):
    assert logprobs(**kw) == rc


def test_token_logprobs_workspace():
    L = hip.lib()
    for rows, n, top in [(1, 1, 1), (1, 151936, 20), (37, 32003, 64), (2047, 151936, 5)]:
        b = L.qlm_token_logprobs_workspace_bytes(rows, n, top)
        assert b > 0
        assert logprobs(rows=rows, n=n, ldl=n, top=top, work_bytes=b - 1) == ARG
        assert 0 < L.qlm_token_logprobs_workspace_bytes(rows, n, 0) <= b
    for bad in [(0, 5, 1), (1, 0, 1), (1, 5, -1), (1, (1 << 21) + 1, 1), (-1, 5, 1)]:
        assert L.qlm_token_logprobs_workspace_bytes(*bad) == 0


def test_engine_score_refuses_a_null_handle():
    from quicklm_amd import engine

    L = engine.lib()
    assert L.qlm_engine_score(None, None, 0, 0, 0, None, None, None, None) == 1
    assert b"null engine handle" in L.qlm_engine_last_error()


@pytest.mark.parametrize("call,kw", [
    (matmul, dict(M=1 << 20)), (matmul, dict(N=1 << 23, ldy=1 << 23)),
    (logprobs, dict(rows=(1 << 21) + 1)),
    (logprobs, dict(rows=2 ** 31 - 1, n=1, ldl=1, top=1)),
])
def test_more_than_a_launch_can_number(call, kw):
    assert call(work_bytes=1 << 60, **kw) == SHAPE
