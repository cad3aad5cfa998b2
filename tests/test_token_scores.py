"""Token scorers: what is refused before any device work (CPU)."""
import ctypes

import numpy as np
import pytest

from llambda_amd import native
from llambda_amd.sampling import HipTokenScorer, SamplingError


@pytest.mark.parametrize("args, message", [
    ((0, 1, 0), "vocab 0 out of range"),
    ((262145, 1, 0), "vocab 262145 out of range"),
    ((100, 0, 0), "max_rows 0 out of range"),
    ((100, 65536, 0), "max_rows 65536 out of range"),
    ((100, 1, 65), "max_top 65 out of range"),
    ((100, 1, -1), "max_top -1 is negative"),
    ((-5, 1, 0), "vocab -5 is negative"),
])
def test_scorers_that_are_refused(args, message):
    with pytest.raises(SamplingError, match=message):
        HipTokenScorer(*args)


def test_given_tokens_are_checked():
    scorer = HipTokenScorer.__new__(HipTokenScorer)
    scorer._h = None
    x = np.zeros((2, 10), np.float32)
    for given, message in [([1, 10], "not all in 0..9"), ([[1], [-1]], "not all in 0..9"), ([1.0, 2.0], "whole numbers"),
                           ([1, 2, 3], r"of shape \(3,\)"), (np.zeros((2, 2, 2), int), "of shape")]:
        with pytest.raises(SamplingError, match=message):
            scorer.score(x, given)
    with pytest.raises(SamplingError, match="top -1 is negative"):
        scorer.score(x, top=-1)
    with pytest.raises(SamplingError, match="1 dimensions"):
        scorer.score(x[0])
    with pytest.raises(SamplingError, match="null scorer"):
        scorer.score(x, [1, 2])


def test_null_pointers_fail():
    L = native.lib()
    L.llambda_hip_token_scorer_destroy(None)
    L.llambda_hip_attention_session_destroy(None)
    out = native.TokenScores()
    assert L.llambda_hip_token_scorer_score_device(None, None, 0, 1, 1, None, 0, 0, ctypes.byref(out), None) == -1
    assert "null scorer" in native.last_error()
    assert L.llambda_hip_token_scorer_create(100, 1, 0, None) == -1
    assert "null result" in native.last_error()
    assert L.llambda_hip_attention_session_create(None, None) == -1
    assert "null result" in native.last_error()
    handle = ctypes.c_void_p()
    assert L.llambda_hip_attention_session_create(None, ctypes.byref(handle)) == -1
    assert "null description" in native.last_error()
    assert L.llambda_hip_attention_session_sync(None, None) == -1
    assert "null session" in native.last_error()
