"""qlm_engine_score at every weight precision, and over more rows than one pass
through the layers takes, against the logits of the batched forward."""

import tempfile

import numpy as np
import pytest

from tests.test_score_gpu import check
from tests.util import say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model_dir(hip):
    from quicklm_amd import synth

    with tempfile.TemporaryDirectory() as d:
        synth.write_model(d, "micro")
        yield d


def both(e, toks, first, top):
    """The logits of toks[first:] after the others, and their scores."""
    out = []
    for scored in (False, True):
        e.reset()
        if first:
            e.forward_batch(toks[:first], 0, argmax=False)
        out.append(e.score(toks[first:], first, top) if scored else
                   e.forward_batch(toks[first:], first, argmax=True, logits=True)[1])
    return out


@pytest.mark.parametrize("precision", ["int8", "int8_row", "int4", "bf16"])
def test_score_at_every_precision(model_dir, precision):
    from quicklm_amd.engine import Engine

    e = Engine(model_dir, max_seq_len=256, max_batch=2, precision=precision)
    try:
        toks = np.random.default_rng(3).integers(0, e.vocab, 140).astype(np.int32)
        for first, n, top in ((0, 1, 3), (20, 1, 0), (20, 9, 64), (30, 64, 1), (0, 140, 5)):
            say(f"score {precision} first={first} n={n} top={top}")
            logits, got = both(e, toks[:first + n], first, top)
            check(got, logits, toks[first:first + n], top)
    finally:
        e.close()


def test_score_over_several_passes(model_dir):
    """2500 rows take two passes through the layers and 40 of the head; a
    generation before and after them is the same."""
    from quicklm_amd.engine import Engine

    e = Engine(model_dir, max_seq_len=2600, max_batch=1, precision="int8")
    try:
        toks = np.random.default_rng(4).integers(0, e.vocab, 2507).astype(np.int32)
        prompt = toks[None, :50]
        say("score of 2500 rows")
        before = e.generate(prompt, 12)[0]
        logits, got = both(e, toks, 7, 4)
        check(got, logits, toks[7:], 4)
        assert np.array_equal(e.generate(prompt, 12)[0], before)
    finally:
        e.close()


def test_score_without_some_outputs(model_dir):
    """Outputs that are not wanted may be null; alternatives need both arrays."""
    from quicklm_amd.engine import Engine, lib

    e = Engine(model_dir, max_seq_len=128, max_batch=1, precision="int8")
    try:
        toks = np.random.default_rng(5).integers(0, e.vocab, 70).astype(np.int32)
        say("score without some outputs")
        e.reset()
        lp, ent, ti, tl = e.score(toks, 0, 3)
        want = e.forward_greedy(1, 70)

        def call(top, *outs):
            e.reset()
            return lib().qlm_engine_score(e.h, toks.ctypes.data, toks.size, 0, top,
                                          *(None if a is None else a.ctypes.data for a in outs))

        a, b = np.empty_like(lp), np.empty_like(ent)
        ids, lps = np.empty_like(ti), np.empty_like(tl)
        for top, outs, wants in ((0, (None,) * 4, ()), (0, (a, None, None, None), ((a, lp),)),
                                 (0, (None, b, None, None), ((b, ent),)),
                                 (3, (None, None, ids, lps), ((ids, ti), (lps, tl)))):
            for o in (a, b, ids, lps):
                o.fill(-7)
            assert call(top, *outs) == 0
            for got, w in wants:
                assert np.array_equal(got, w, equal_nan=got.dtype == np.float32)
            assert e.forward_greedy(1, 70) == want
        assert call(3, a, b, None, lps) != 0 and call(3, a, b, ids, None) != 0
    finally:
        e.close()
