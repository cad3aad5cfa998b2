"""Attention sessions: what is refused before any device work (CPU), and the reference of the GPU tests against
itself."""
import numpy as np
import pytest

import attention_reference as ref
from llambda_amd.attention import AttentionLayout, HipAttentionSession
from llambda_amd.hip_backend import HipBackendError

GOOD = dict(heads=8, kv_heads=2, head_dim=64)
ROOM = dict(pages=4, page_tokens=16, max_context=64)


@pytest.mark.parametrize("change, room, message", [
    (dict(heads=0), {}, "heads 0 is not in 1..1024"),
    (dict(heads=2048), {}, "heads 2048 is not in 1..1024"),
    (dict(kv_heads=3), {}, "3 kv_heads do not divide 8 heads"),
    (dict(kv_heads=16), {}, "kv_heads 16 is not in 1..8"),
    (dict(head_dim=72), {}, "head_dim 72 is not a multiple of 16"),
    (dict(head_dim=272), {}, "head_dim 272 is not in 16..256"),
    (dict(row_type="f64"), {}, "no type 'f64'"),
    (dict(row_type="f16", cache_type="f32"), {}, "no rows of type 1 over a cache of type 0"),
    (dict(row_type="bf16", cache_type="f16"), {}, "no rows of type 30 over a cache of type 1"),
    (dict(scale=-1.0), {}, "scale -1.0 is not positive"),
    (dict(scale=0.0), {}, "scale 0.0 is not positive"),
    (dict(scale=float("nan")), {}, "scale nan is not positive"),
    (dict(scale=float("inf")), {}, "scale inf"),
    ({}, dict(page_tokens=8), "page_tokens 8 is not in 16.."),
    ({}, dict(page_tokens=48), "page_tokens 48 is not a power of two"),
    ({}, dict(pages=0), "pages 0 is not in 1.."),
    ({}, dict(max_context=0), "max_context 0 is not in 1.."),
    ({}, dict(max_tokens=0), "max_tokens 0 is not in 1.."),
    ({}, dict(max_sequences=65536), "max_sequences 65536 is not in 1..65535"),
    ({}, dict(layers=0), "layers 0 is not in 1.."),
    ({}, dict(key_pages_ptr=4096), "one pool without the other"),
    ({}, dict(key_pages_ptr=4096, value_pages_ptr=4104), "pools must be 16-byte aligned"),
    ({}, dict(pages=2 ** 31 - 1, page_tokens=2 ** 20), "a pool of"),
])
def test_descriptions_that_are_refused(change, room, message):
    with pytest.raises(HipBackendError, match=message):
        HipAttentionSession(AttentionLayout(**{**GOOD, **change}), **{**ROOM, **room})


def test_closed_session_is_refused():
    session = HipAttentionSession.__new__(HipAttentionSession)
    session.pointer = None
    with pytest.raises(HipBackendError, match="closed"):
        session.sync()


def test_bf16_bits():
    rng = np.random.default_rng(0)
    a = rng.normal(size=1000).astype(np.float32)
    b = ref.rounded(a, "bf16")
    assert np.all(np.abs(a - b) <= np.abs(a) * 2.0 ** -8)
    assert np.array_equal(ref.rounded(b, "bf16"), b)
    assert ref.rounded(np.float32([1 + 2 ** -8, 1 + 3 * 2 ** -8]), "bf16").tolist() == [1.0, 1 + 2 ** -6]


def test_a_chain_sees_what_causal_rows_see():
    assert np.array_equal(ref.sees(7, 3), ref.sees(7, 3, [-1, 0, 1, 2, 3, 4, 5]))
