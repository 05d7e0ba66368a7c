"""cs1_kv_extend and cs1_kv_reserve where free pages are few among many, or many: the scans over the pages' counts, and what they
collect before it is taken."""
import numpy as np
import pytest

from decode_ref import Table, ints
from gpu_helpers import get, say, stream
from qwen3_5_native import hip
from test_gpu_kv_rows import Cache

pytestmark = pytest.mark.gpu


def pool(rng, npages, free, nseq=40, max_pages=6000):
    """All pages are someone's but `free` (numbers, or how many of them at random)."""
    t = Table(nseq, max_pages, npages, 16)
    t.refs[:] = 1
    t.refs[rng.choice(npages, free, replace=False) if isinstance(free, int) else free] = 0
    return t


@pytest.mark.parametrize("npages,free", [(4095, 50), (4097, 300), (20480, 700), (20481, 700), (36865, 900), (60000, 1200), (60000, [59999, 4096, 4095, 0]),
                                         (60000, list(range(20470, 20490))), (30000, 29000), (60000, 60000)])
def test_few_among_many(npages, free):
    say(f"free pages: {free if isinstance(free, int) else len(free)} of {npages}")
    rng = np.random.default_rng(npages)
    c = Cache(pool(rng, npages, free))
    n = free if isinstance(free, int) else len(free)
    for share in (0.01, 0.3, 0.5):  # some of them, again, and then more than are left
        new = np.maximum(1, rng.multinomial(max(1, int(n * share)) * 16, np.ones(20) / 20))
        seqs, cu = rng.permutation(40)[:20], np.concatenate([[0], np.cumsum(new)])
        if c.extend(seqs, cu) == 0:
            c.rows(seqs, cu, int(min(cu[-1], 5000)))
    c.extend([0], [0, 6000 * 16 - int(c.t.lens[0])])  # as much as a row of the table holds
    lens = c.t.lens.copy()
    b = ints(np.arange(40))
    hip.check(hip.api().cs1_kv_reserve(c.d.ref, b.at(0), None, 40, c.status.at(0), stream().handle), "reserve")
    want = c.t.reserve(list(range(40)))
    assert get(c.status, np.int32, 1)[0] == want
    c.d.check()
    assert (c.t.lens == lens).all() or want == 0
