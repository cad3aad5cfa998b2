"""Mamba-2 mixer layers: what session creation refuses before any device work,
and layers read from a model's tensors."""
import ctypes
import dataclasses

import numpy as np
import pytest

import ssm_reference
from llambda_amd import ggml, native, projection
from llambda_amd.hip_backend import HipBackendError
from llambda_amd.ssm import HipSsmSession, ssm_layer_from_model, synthetic_ssm


def _layer(**kw):
    return synthetic_ssm(np.random.default_rng(1), **{**dict(heads=4, head_dim=32, groups=2, state=16), **kw})


@pytest.mark.parametrize("change,text", [
    (dict(head_dim=24), "head_dim 24 is not a multiple of 16"),
    (dict(head_dim=144), "head_dim 144 is not in 16..128"),
    (dict(groups=3), "3 groups do not divide 4 heads"),
    (dict(groups=5), "groups 5 is not in 1..4"),
    (dict(state=48), "state 48 is not a power of two"),
    (dict(state=512), "state 512 is not in"),
    (dict(conv_width=1), "conv_width 1 is not in 2..4"),
    (dict(conv_width=5), "conv_width 5 is not in 2..4"),
    (dict(heads=256, head_dim=128, groups=1, state=16), "channels of a norm group"),
])
def test_layouts_that_are_refused(change, text):
    with pytest.raises(HipBackendError, match=text):
        HipSsmSession(_layer(**change))


@pytest.mark.parametrize("kw,text", [
    (dict(slots=0), "slots 0"), (dict(max_tokens=0), "max_tokens 0"),
    (dict(max_tokens=1 << 21), "max_tokens"), (dict(max_sequences=0), "max_sequences 0"),
    (dict(max_sequences=65536), "max_sequences"),
    (dict(conv_states_ptr=4096), "one state pool"), (dict(conv_states_ptr=4096, ssm_states_ptr=4104), "aligned"),
])
def test_sizes_that_are_refused(kw, text):
    with pytest.raises(HipBackendError, match=text):
        HipSsmSession(_layer(), **kw)


@pytest.mark.parametrize("value", [0.5, np.inf, -np.inf, np.nan])
def test_growing_states_are_refused(value):
    layer = _layer()
    layer.a[2] = value
    with pytest.raises(HipBackendError, match=r"ssm_a\[2\]"):
        HipSsmSession(layer)


def test_other_refusals():
    for eps in (-1.0, np.nan, np.inf):
        with pytest.raises(HipBackendError, match="norm_epsilon"):
            HipSsmSession(dataclasses.replace(_layer(), norm_epsilon=eps))
    with pytest.raises(HipBackendError, match="norm has 127 elements, not 128"):
        HipSsmSession(dataclasses.replace(_layer(), norm=np.ones(127, np.float32)))
    with pytest.raises(HipBackendError, match="null weights"):
        HipSsmSession(dataclasses.replace(_layer(), d=None))
    L = native.lib()
    assert L.llambda_hip_ssm_session_create(None, None) == -1
    assert "null result" in native.last_error()
    assert L.llambda_hip_ssm_session_create(None, ctypes.byref(ctypes.c_void_p())) == -1
    L.llambda_hip_ssm_session_destroy(None)
    assert L.llambda_hip_ssm_session_input_element_count(None) == 0
    assert L.llambda_hip_ssm_session_output_element_count(None) == 0
    for call in (L.llambda_hip_ssm_session_step_device(None, None, None, 1, None, None, None),
                 L.llambda_hip_ssm_session_run(None, 0, None, 0, None, 0, 1),
                 L.llambda_hip_ssm_session_reset(None, 0), L.llambda_hip_ssm_session_sync(None, None)):
        assert call == -1


def test_layer_from_model():
    want = _layer()
    t = projection.TensorInfo

    def info(name, a):
        return t(f"blk.3.{name}", ggml.F32, tuple(reversed(a.shape)), np.ascontiguousarray(a).view(np.uint8).reshape(-1))

    tensors = [info("ssm_conv1d.weight", want.conv_weight), info("ssm_conv1d.bias", want.conv_bias),
               info("ssm_dt.bias", want.dt_bias), info("ssm_a", want.a.reshape(-1, 1)), info("ssm_d", want.d),
               info("ssm_norm.weight", want.norm.reshape(2, -1))]
    got = ssm_layer_from_model(projection.ProjectionModel(tensors, layer_count=4), 3, heads=4, groups=2)
    for f in dataclasses.fields(want):
        assert np.array_equal(getattr(got, f.name), getattr(want, f.name)), f.name
    assert (got.row, got.channels, got.inner) == (2 * 128 + 64 + 4, 192, 128)
    with pytest.raises(HipBackendError, match="do not fit"):
        ssm_layer_from_model(projection.ProjectionModel(tensors, layer_count=4), 3, heads=5, groups=2)
    with pytest.raises(KeyError, match="ssm_conv1d.weight"):
        ssm_layer_from_model(projection.ProjectionModel(tensors[1:], layer_count=4), 3, heads=4, groups=2)


@pytest.mark.parametrize("names", ["xBCs", "x", "B", "C", "s"])
@pytest.mark.parametrize("kw", [dict(heads=4, head_dim=64, groups=2, state=128), dict(heads=4, head_dim=32, state=16),
                                dict(heads=2, head_dim=128, groups=1, state=256)], ids=str)
def test_operands_of_half_the_digits_are_seen(kw, names):
    """An operand of 16 bits leaves what a call's outputs may differ by together."""
    rng = np.random.default_rng(7)
    layer = _layer(**kw)
    x = rng.normal(size=(129, layer.row)).astype(np.float32)
    conv = rng.normal(size=(layer.conv_width - 1, layer.channels)).astype(np.float32)
    ssm = rng.normal(size=(layer.heads, layer.head_dim, layer.state)).astype(np.float32)

    def rounded(bits):
        def operand(name, v):
            if name not in names:
                return v
            m, e = np.frexp(v)
            return np.ldexp(np.round(m * 2.0 ** bits), e - bits)
        return operand

    want = ssm_reference.sequence(layer, x, conv, ssm)
    few, all_ = (ssm_reference.with_operands(layer, x, conv, ssm, rounded(bits)) for bits in (16, 24))
    assert ssm_reference.together(few[0], want[0]) > ssm_reference.TOGETHER
    assert ssm_reference.together(all_[0], want[0]) < ssm_reference.TOGETHER / 4
    if "x" in names or "B" in names:
        assert ssm_reference.together(few[1], want[2]) > ssm_reference.TOGETHER
    exact = ssm_reference.with_operands(layer, x, conv, ssm, lambda name, v: v)
    for got, of in ((exact[0], want[0]), (exact[1], want[2])):
        assert ssm_reference.together(got, of) < 1e-8  # (the epsilon of one is rounded to float32)
