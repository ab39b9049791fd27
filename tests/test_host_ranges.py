"""Positions and counts that the engine refuses on the host, also where their
sum passes 2^31: tests/model_probe.cpp calls the model with its sizes set and
nothing loaded. Run where no GPU is visible, as the host's other refusals: a
call that came past its check would end at the missing device."""

import ctypes as C
import os
import subprocess

import pytest

from quicklm_amd import hip

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "quicklm_amd")
BIG = 2 ** 31 - 1
MAX_SEQ = 512
BATCH, STEPS, TOKENS, GENERATE, SCORE, LOGITS, WIDE = range(7)


@pytest.fixture(scope="module")
def call(tmp_path_factory):
    hip.lib()
    if hip.device_count() > 0:
        pytest.skip("host-only refusal tests run where no GPU is visible")
    so = str(tmp_path_factory.mktemp("model_probe") / "libmodelprobe.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I",
                    os.path.join(PKG, "csrc", "host"), "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "model_probe.cpp"), "-o", so, "-L", PKG,
                    "-lqlm_engine", "-lqlm_hip", f"-Wl,-rpath,{PKG}"], check=True)
    L = C.CDLL(so)

    def run(which, a, b):
        err = C.create_string_buffer(256)
        L.model_ranges(which, MAX_SEQ, a, b, err, len(err))
        return err.value.decode()

    return run


EXCEEDED = f"context length exceeded max_seq_len ({MAX_SEQ})"
OUTSIDE = "tokens: range outside the token stream"


@pytest.mark.parametrize("which,a,b,text", [
    (BATCH, 8, BIG, EXCEEDED), (BATCH, 8, BIG - 7, EXCEEDED), (BATCH, 2, BIG - 1, EXCEEDED),
    (BATCH, 8, MAX_SEQ - 7, EXCEEDED), (BATCH, 8, -1, EXCEEDED), (BATCH, 8, -BIG - 1, EXCEEDED),
    (BATCH, MAX_SEQ + 1, 0, EXCEEDED),
    (SCORE, 8, BIG, EXCEEDED), (SCORE, 8, MAX_SEQ - 7, EXCEEDED), (SCORE, 8, -1, EXCEEDED),
    (STEPS, BIG, 1, EXCEEDED), (STEPS, BIG, MAX_SEQ, EXCEEDED), (STEPS, MAX_SEQ, 1, EXCEEDED),
    (TOKENS, 8, BIG, OUTSIDE), (TOKENS, BIG, 1, OUTSIDE), (TOKENS, 8, MAX_SEQ - 6, OUTSIDE),
    (TOKENS, 8, -1, OUTSIDE),
    (GENERATE, 8, BIG, EXCEEDED), (GENERATE, 8, MAX_SEQ - 6, EXCEEDED),
    (GENERATE, BIG, BIG, EXCEEDED), (GENERATE, MAX_SEQ + 1, 0, EXCEEDED)])
def test_a_range_past_the_context_is_refused(call, which, a, b, text):
    assert call(which, a, b) == text


@pytest.mark.parametrize("which,a,b", [
    (BATCH, 8, MAX_SEQ - 8), (SCORE, 8, MAX_SEQ - 8), (STEPS, 2, MAX_SEQ - 2),
    (TOKENS, 8, MAX_SEQ - 7), (GENERATE, 8, MAX_SEQ - 7)])
def test_a_range_that_fits_reaches_the_device(call, which, a, b):
    assert call(which, a, b) not in (EXCEEDED, OUTSIDE, "no error")


@pytest.mark.parametrize("which,a,b,text", [
    # a negative number of steps would move the count of positions back
    (STEPS, -1, 5, "steps: negative count"), (STEPS, -BIG - 1, 0, "steps: negative count"),
    (TOKENS, -1, 5, OUTSIDE), (TOKENS, -BIG - 1, 0, OUTSIDE),
    (LOGITS, -1, 0, "last_logits: no such sequence"),
    (LOGITS, 1, 0, "last_logits: no such sequence"),
    (LOGITS, BIG, 0, "last_logits: no such sequence")])
def test_a_negative_count_or_another_sequence_is_refused(call, which, a, b, text):
    assert call(which, a, b) == text


@pytest.mark.parametrize("vocab,top,text", [
    ((1 << 21) + 1, 0, "score: vocabulary too large"), (BIG, 5, "score: vocabulary too large"),
    (1 << 21, 65, "score: top out of range"), (4, 5, "score: top out of range"),
    (4, -1, "score: top out of range")])
def test_score_names_what_it_refuses(call, vocab, top, text):
    assert call(WIDE, vocab, top) == text
