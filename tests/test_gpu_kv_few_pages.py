"""cs1_kv_extend and cs1_kv_reserve that need few pages: found in the first scan of the counts and taken by the lanes of the waves
that find them, wherever in a wave's 256 pages they are; one more than that, and such that lie behind the first scan."""
import numpy as np
import pytest

from decode_ref import ints
from gpu_helpers import get, say, stream
from qwen3_5_native import hip
from test_gpu_kv_free_pages import pool
from test_gpu_kv_rows import Cache

pytestmark = pytest.mark.gpu

SPOTS = {
    "a wave's borders": [0, 63, 64, 127, 128, 191, 192, 255, 256, 319, 511, 512, 4095],
    "every 64th": list(range(5, 4096, 64)),
    "every 63rd": list(range(0, 4096, 63)),
    "sixteen a wave": list(range(0, 4096, 16)),
    "a run": list(range(250, 330)),
    "the end of the first scan": list(range(4060, 4130)),
    "behind the first scan": [1, 2, 4096, 4097, 20479, 20480, 29999],
    "none": [],
}


@pytest.mark.parametrize("where", SPOTS)
@pytest.mark.parametrize("npages", [4096, 4100, 30000])
def test_few_pages(where, npages):
    free = [p for p in SPOTS[where] if p < npages]
    say(f"few pages: {where}, {len(free)} of {npages}")
    rng = np.random.default_rng(npages + len(free))
    for total in sorted({1, 2, 13, 63, 64, 65, len(free) - 1, len(free), len(free) + 1}):
        if total < 1 or total > 300:
            continue
        n = min(total, 9)
        c = Cache(pool(rng, npages, free))
        new = 16 * (1 + rng.multinomial(total - n, np.ones(n) / n))
        want = c.extend(rng.permutation(40)[:n], np.concatenate([[0], np.cumsum(new)]))
        assert (want == 0) == (total <= len(free))


def test_single_tokens():
    say("few pages: single tokens of 1 to 70 sequences")
    rng = np.random.default_rng(1)
    for n in (1, 2, 40, 64, 65, 70):
        c = Cache(pool(rng, 3000, 200, nseq=80))
        for _ in range(2):  # the second one has room already
            b = ints(rng.permutation(80)[:n])
            seqs = get(b, np.int32, n)
            hip.check(hip.api().cs1_kv_reserve(c.d.ref, b.at(0), None, n, c.status.at(0), stream().handle), "reserve")
            assert c.answer() == c.t.reserve(seqs)
            c.d.check()
