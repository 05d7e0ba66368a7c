"""The operations on several new tokens of a sequence refuse sizes past what their kernels count in 32 bits, before any
device work."""
import ctypes

import pytest

from qwen3_5_native import hip
from test_decode_refusals import table

INVALID = hip.HIP_ERROR_INVALID_VALUE
N = None
A = 1 << 20  # an aligned address that is never followed: every call here returns before a launch


@pytest.mark.parametrize("n,nseq,max_pages", [(17, 8192, 1 << 27), (8192, 17, 1 << 27), (8192, 8192, 1 << 18), (32, 32, 1 << 26)])
def test_extend_of_more_pages_than_32_bits_count(n, nseq, max_pages):
    """Offsets that fall and rise again may ask each entry's whole row of the table: 17 rows of 2^27 pages, 2^31 and more in
    all, came out as a negative number, and lengths grew with no page behind them."""
    t = table(nseq=nseq, max_pages=max_pages - (max_pages == 1 << 27), page=16)
    assert hip.load().cs1_kv_extend(t, N, A, n, A, N) == INVALID


def test_prep_of_more_rows_than_a_launch_has():
    rot = hip.Rotary(A, 64, 0, 1.0)
    for dh, ld in ((128, 8192), (256, 10240)):
        for T in (1 << 24, 2 ** 31 - 1):
            assert hip.load().cs1_attn_prep_paged(A, A, A, ld, A, A, 1e-6, ctypes.byref(rot), table(), A, A, A, A, A, A, T, 16, 4, dh, N) == INVALID


@pytest.mark.parametrize("rows", [1 << 23, 1 << 24, 2 ** 31 - 1])
def test_log_probabilities_of_more_rows_than_a_launch_has(rows):
    for V in (1, 2, 9, 1000):
        assert hip.load().cs1_token_logprobs(A, 0, V, A, rows, V, 1, A, A, A, A, A, N) == INVALID
