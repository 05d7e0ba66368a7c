"""cs1_kv_rows_if_room refuses what cs1_kv_rows does, and a missing status, before any device work."""
import pytest

from qwen3_5_native import hip
from test_decode_refusals import BAD_TABLES, table

INVALID = hip.HIP_ERROR_INVALID_VALUE
N = None
A = 1 << 20  # an aligned address that is never followed: every call here returns before a launch


@pytest.mark.parametrize("bad", BAD_TABLES + [dict(npages=(1 << 30) + 1), dict(npages=1 << 27)], ids=str)
def test_bad_tables(bad):
    assert hip.load().cs1_kv_rows_if_room(table(**bad), N, A, 0, 4, A, A, A, N) == INVALID


def test_arguments():
    call = hip.load().cs1_kv_rows_if_room
    for n in (-1, 8193):
        assert call(table(), N, A, n, 4, A, A, A, N) == INVALID
    assert call(N, N, A, 1, 4, A, A, A, N) == INVALID
    assert call(table(), N, N, 1, 4, A, A, A, N) == INVALID   # no offsets
    assert call(table(), N, A, 1, -1, A, A, A, N) == INVALID
    assert call(table(), N, A, 1, 4, N, A, A, N) == INVALID   # no status
    assert call(table(), N, A, 1, 0, N, A, A, N) == INVALID
    assert call(table(), N, A, 1, 4, A, N, A, N) == INVALID
    assert call(table(), N, A, 1, 4, A, A, N, N) == INVALID
    assert call(table(), N, N, 1, 0, A, N, N, N) == 0
