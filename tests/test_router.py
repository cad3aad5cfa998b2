"""Routers and batch samplers: what their creation refuses before any device work."""
import ctypes

import numpy as np
import pytest

from llambda_amd import native
from llambda_amd.hip_backend import HipBackendError
from llambda_amd.moe import HipRouter, Routing
from llambda_amd.sampling import HipBatchSampler, SamplingError, _per_row, _random_per_row


@pytest.mark.parametrize("kw,text", [
    (dict(experts=0, top_k=1), "expert_count 0"), (dict(experts=1025, top_k=1), "expert_count 1025"),
    (dict(experts=8, top_k=0), "top_k 0"), (dict(experts=8, top_k=9), "top_k 9 is not in 1..8"),
    (dict(experts=128, top_k=65), "top_k 65 is not in 1..64"),
    (dict(experts=8, top_k=1, groups=0), "groups 0"), (dict(experts=8, top_k=1, groups=3), "3 groups do not divide"),
    (dict(experts=256, top_k=1, groups=128), "groups 128 is not in 1..64"),
    (dict(experts=8, top_k=1, groups=2, top_groups=3), "top_groups 3"),
    (dict(experts=8, top_k=5, groups=2, top_groups=1), "top_k 5 is not in 1..4"),
    (dict(experts=8, top_k=1, group_rank=3), "group_rank 3"), (dict(experts=8, top_k=1, group_rank=0), "group_rank 0"),
    (dict(experts=8, top_k=1, weights_scale=np.inf), "weights_scale"), (dict(experts=8, top_k=1, score="relu"), "relu"),
    (dict(experts=8, top_k=1, bias=np.zeros(7, np.float32)), "bias has 7 elements, not 8"),
])
def test_routings_that_are_refused(kw, text):
    with pytest.raises(HipBackendError, match=text):
        HipRouter(Routing(**kw))


def test_null_arguments():
    L = native.lib()
    assert L.llambda_hip_router_create(None, None) == -1
    assert L.llambda_hip_router_create(None, ctypes.byref(ctypes.c_void_p())) == -1
    d = native.RouterDesc(score=7, expert_count=8, top_k=1, groups=1, top_groups=1, group_rank=1)
    assert L.llambda_hip_router_create(ctypes.byref(d), ctypes.byref(ctypes.c_void_p())) == -1
    assert "unknown score 7" in native.last_error()
    assert L.llambda_hip_router_run(None, None, 0, None, None, 1) == -1
    assert L.llambda_hip_router_run_device(None, None, None, None, 1, None) == -1
    assert L.llambda_hip_moe_session_set_router(None, None) == -1
    L.llambda_hip_router_destroy(None)
    L.llambda_hip_batch_sampler_destroy(None)
    assert L.llambda_hip_batch_sampler_create(10, 1, None) == -1
    assert L.llambda_hip_batch_sampler_sample(None, None, 1, 1, None, None) == -1
    assert L.llambda_hip_batch_sampler_sample_device(None, None, 1, 1, None, None, None) == -1


@pytest.mark.parametrize("vocab,rows,text", [(0, 1, "vocab 0"), (262145, 1, "vocab 262145"), (10, 0, "max_rows 0"),
                                             (10, 65536, "max_rows 65536")])
def test_batch_samplers_that_are_refused(vocab, rows, text):
    with pytest.raises(SamplingError, match=text):
        HipBatchSampler(vocab, rows)


def test_parameters_of_rows():
    """Random numbers of more digits than float32 stay below 1; counts are whole and do not wrap around."""
    last = np.float32(1 - 2.0 ** -24)
    assert _random_per_row(1 - 2.0 ** -40, 2).tolist() == [last, last]
    assert _random_per_row([0.25, 0.99999999], 2).tolist() == [0.25, last]
    assert _random_per_row([1.0, -1e-9], 2).tolist() == [1.0, np.float32(-1e-9)]  # (refused by the call)
    assert np.isnan(_random_per_row(np.nan, 1)[0])
    assert _per_row(np.array([2 ** 40, -2 ** 40, 7]), 3, np.int32).tolist() == [2 ** 31 - 1, -2 ** 31, 7]
    assert _per_row(2 ** 40, 2, np.int32).tolist() == [2 ** 31 - 1] * 2
    assert _per_row(np.uint64(2 ** 63), 1, np.int32).tolist() == [2 ** 31 - 1]
    assert _per_row(np.array([40.0, 1e30, -1e30]), 3, np.int32).tolist() == [40, 2 ** 31 - 1, -2 ** 31]
    assert _per_row(np.float32(7), 1, np.int32).tolist() == [7] and _per_row(True, 1, np.int32).tolist() == [1]
    for v in (2.5, [1, 2.25], np.nan, "3", None):
        with pytest.raises(SamplingError, match="TOP-K must be whole numbers"):
            _per_row(v, 2, np.int32)
    assert _per_row([0.5], 2, np.float32).tolist() == [0.5, 0.5]
