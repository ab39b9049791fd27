"""Scoring a prompt through the engine: qlm_engine_score against the logits of
the batched forward (64-bit log softmax of them), and the states it leaves."""

import os
import tempfile

import numpy as np
import pytest

from tests.util import say

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def engine(hip):
    from quicklm_amd import synth
    from quicklm_amd.engine import Engine

    base = "/dev/shm" if os.path.isdir("/dev/shm") else None
    with tempfile.TemporaryDirectory(dir=base) as d:
        say("writing tiny model", d)
        synth.write_model(d, "tiny")
        e = Engine(d, max_seq_len=512, max_batch=1, precision="int8")
    yield e
    e.close()


def reference(logits, tokens, top):
    """(logprobs, entropy, top_ids, top_logprobs) of rows of logits in 64 bits."""
    x = logits.astype(np.float64)
    d = x - x.max(axis=1, keepdims=True)
    e = np.exp(d)
    z = e.sum(axis=1, keepdims=True)
    lsm = d - np.log(z)
    ids = np.argsort(-x, axis=1, kind="stable")[:, :top]
    lp = np.append(lsm[np.arange(len(tokens) - 1), tokens[1:]], np.nan)
    ent = (np.log(z) - (e * d).sum(axis=1, keepdims=True) / z)[:, 0]
    return lp, ent, ids, np.take_along_axis(lsm, ids, 1), d


def check(got, logits, tokens, top):
    lp, ent, ti, tl = got
    rlp, rent, rti, rtl, d = reference(logits, tokens, top)
    # A term of z is off by 2 (|d| + 1) roundings, its sums by one a term added
    # in turn (chunks of 256 tokens, four to a lane) and 16 a join; log z by 4
    # of its size, and the difference by one of |d| and of the result. Entropy:
    # the same on both of its terms.
    chunks = -(-logits.shape[1] // 256)
    tol = U * (2 * np.abs(d).max() + 64 + 2 * chunks + 64)
    tol_h = tol * (2 + 3 * rent.max())
    assert np.isnan(lp[-1]) and np.array_equal(ti, rti)
    assert np.abs(lp[:-1] - rlp[:-1]).max(initial=0) <= tol
    assert np.abs(ent - rent).max() <= tol_h
    assert np.abs(tl - rtl).max(initial=0) <= tol


@pytest.mark.parametrize("n,top", [(1, 5), (2, 0), (9, 64), (70, 5), (200, 1)])
def test_score_matches_the_logits(engine, n, top):
    e = engine
    toks = np.random.default_rng(n).integers(0, e.vocab, 40 + n).astype(np.int32)
    say(f"score n={n} top={top}")
    e.reset()
    e.forward_batch(toks[:40], 0, argmax=False)
    _, logits = e.forward_batch(toks[40:], 40, argmax=True, logits=True)
    e.reset()
    e.forward_batch(toks[:40], 0, argmax=False)
    got = e.score(toks[40:], 40, top)
    check(got, logits, toks[40:], top)


def test_score_leaves_the_states_of_a_forward(engine):
    e = engine
    toks = np.random.default_rng(7).integers(0, e.vocab, 120).astype(np.int32)
    say("states after score")
    e.reset()
    e.forward_batch(toks[:100], 0, argmax=True)
    want = [e.forward_greedy(int(t), 100 + i) for i, t in enumerate(toks[100:])]
    logits = e.last_logits(0)
    e.reset()
    e.score(toks[:100], 0, 3)
    assert [e.forward_greedy(int(t), 100 + i) for i, t in enumerate(toks[100:])] == want
    assert np.array_equal(e.last_logits(0), logits)


def test_score_in_pieces(engine):
    """A text in pieces of one, a few and many tokens: each piece against its
    own logits, buffers growing and shrinking between the calls."""
    e = engine
    toks = np.random.default_rng(8).integers(0, e.vocab, 200).astype(np.int32)
    say("score in pieces")
    cuts = [0, 1, 5, 130, 131, 200]
    logits = []
    e.reset()
    for a, b in zip(cuts, cuts[1:]):
        logits.append(e.forward_batch(toks[a:b], a, argmax=True, logits=True)[1])
    e.reset()
    for i, (a, b) in enumerate(zip(cuts, cuts[1:])):
        check(e.score(toks[a:b], a, 2 * i), logits[i], toks[a:b], 2 * i)


def test_score_refusals(engine):
    from quicklm_amd.engine import EngineError

    e = engine
    t = np.arange(8, dtype=np.int32)
    say("score refusals")
    e.reset()
    for call in (lambda: e.score(t, 510), lambda: e.score(t, -1), lambda: e.score(t, 0, 65),
                 lambda: e.score(t, 0, -1), lambda: e.score([0, e.vocab], 0),
                 lambda: e.score([-1, 0], 0)):
        with pytest.raises(EngineError):
            call()
    lp, ent, ti, tl = e.score([], 0, 3)  # nothing to score
    assert lp.size == ent.size == 0 and ti.shape == tl.shape == (0, 3)


def test_score_refuses_a_position_whose_sum_overflows(engine):
    from quicklm_amd.engine import EngineError

    say("score at the largest position")
    with pytest.raises(EngineError):
        engine.score(np.arange(8, dtype=np.int32), 2 ** 31 - 1)
