"""cs1_token_logprobs_workspace_bytes: what is enough for `rows` rows is enough for any fewer, needs no device."""
import pytest

from qwen3_5_native import hip


@pytest.fixture(scope="module")
def size():
    return hip.load().cs1_token_logprobs_workspace_bytes


@pytest.mark.parametrize("V", [1, 2048, 2049, 4096, 4097, 40000, 65537, 70008, 131072, 151936, 248320, 1 << 24, 1 << 28])
def test_serves_fewer_rows(size, V):
    for k in (0, 1, 20, 32):
        sizes = [size(rows, V, k) for rows in range(1, 1024)]
        assert sizes == sorted(sizes), (V, k)
        # sums of 16 bytes and k keys of 8 for each part, and never many of them
        assert all(s % (16 + 8 * k) == 0 for s in sizes) and sizes[-1] <= 2046 * (16 + 8 * k)
        assert (sizes[0] == 0) == (sizes[-1] == 0)


def test_serves_fewer_alternatives_and_tokens(size):
    for rows in (1, 7, 300, 511, 512, 1023):
        for V in (3000, 131072, 131073, 248320):
            sizes = [size(rows, V, k) for k in range(33)]
            assert sizes == sorted(sizes)
        sizes = [size(rows, V, 20) for V in range(1000, 300000, 331)]
        assert sizes == sorted(sizes)


def test_many_rows_need_none(size):
    for rows in (1024, 1025, 5000, 1 << 20):
        assert size(rows, 151936, 20) == 0
