"""Lists of pages and parents that are no whole numbers of 32 bits are refused before any device work (CPU)."""
import numpy as np
import pytest

from llambda_amd.attention import AttentionLayout, HipAttentionSession
from llambda_amd.hip_backend import HipBackendError


@pytest.fixture
def session():
    """As far as its lists go: the native session is not reached."""
    s = HipAttentionSession.__new__(HipAttentionSession)
    s.pointer, s.layout, s.page_tokens = None, AttentionLayout(4, 2, 16), 16
    return s


ROWS = [np.zeros((2, heads, 16), np.float32) for heads in (4, 2, 2)]


@pytest.mark.parametrize("table, message", [
    ([0.0, 1.0], "table must be whole numbers, not float64"),
    (np.array([0.5], np.float32), "table must be whole numbers, not float32"),
    ([True, False], "table must be whole numbers, not bool"),
    (["0"], "table must be whole numbers"),
    ([2 ** 32], "table holds 4294967296, which does not fit"),
    (np.array([2 ** 32 + 1, 0], np.int64), "table holds 4294967297"),
    (np.array([2 ** 31], np.uint32), "table holds 2147483648"),
    (np.array([2 ** 64 - 1], np.uint64), "table holds 18446744073709551615"),
    ([-2 ** 31 - 1], "table holds -2147483649"),
    ([2 ** 80], "table must be whole numbers, not object"),
])
def test_tables(session, table, message):
    with pytest.raises(HipBackendError, match=message):
        session.run(*ROWS, table)
    with pytest.raises(HipBackendError, match=message):
        session.read(table, 0, 2)
    with pytest.raises(HipBackendError, match=message):
        session.write(table, 0, *(np.zeros((2, 2, 16), np.float16) for _ in range(2)))


@pytest.mark.parametrize("parents, message", [
    ([-1.0, 0.0], "parents must be whole numbers, not float64"),
    (np.array([-1, 2 ** 32 - 1]), "parents holds 4294967295"),
    ([-1], "1 parents of 2 rows"),
])
def test_parents(session, parents, message):
    with pytest.raises(HipBackendError, match=message):
        session.run(*ROWS, [0, 1], parents=parents)


def test_lists_that_fit(session):
    """What is behind the entries in use is not looked at."""
    for table in ([3], (3, 4), np.array([3, -1], np.int8), np.array([3, 2 ** 40]), np.array([[3], [5]], np.uint64), range(3, 5)):
        t = session._table(table, 16)
        assert t.dtype == np.int32 and t[0] == 3 and t.flags.c_contiguous
    assert session._table([], 0).size == 0
    with pytest.raises(HipBackendError, match="closed"):
        session.run(*ROWS, np.array([0, 1], np.int64), parents=np.array([-1, 0], np.int16))


def test_a_scale_that_is_zero_in_single_precision():
    """It would be taken for the default."""
    with pytest.raises(HipBackendError, match="scale 1e-60 is not positive"):
        HipAttentionSession(AttentionLayout(4, 2, 16, scale=1e-60), pages=1, max_context=16)
