"""cs1_attention_paged_varlen for many entries whose columns are more than few: windows of the search, items that lie whole in a
stretch, and stretches that begin inside one item and end inside another."""
import numpy as np
import pytest

import decode_ref as R
from gpu_helpers import say
from test_gpu_attention_chunk import Call, handle, run  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,longest,most,hq,hk,dh", [(130, 900, 3, 17, 1, 256), (300, 700, 3, 17, 1, 128), (2100, 60, 2, 17, 1, 128), (700, 300, 9, 4, 2, 256),
                                                     (65, 2500, 40, 6, 2, 128), (8192, 4, 2, 20, 1, 128)])
def test_many_entries(handle, n, longest, most, hq, hk, dh):  # noqa: F811
    say(f"attention: {n} entries up to {longest}, heads {hq}/{hk} Dh={dh}")
    rng = np.random.default_rng(n)
    lens = rng.integers(0, longest + 1, n)
    new = np.minimum(lens, rng.integers(0, most + 1, n))
    t = R.scattered(rng, n, lens.tolist(), 16 if n > 1000 else 48)
    order = rng.permutation(n)
    run(Call(handle, rng, t, order, new[order], hq, hk, dh, pad=1, lse=n < 1000, gate=n != 300))


@pytest.mark.parametrize("lens,new,hq,hk,dh", [([20000], [700], 24, 4, 256), ([30000], [300], 16, 1, 128), ([9000, 12000], [400, 500], 16, 4, 256),
                                               ([3000] * 40, [64] * 40, 16, 4, 128), ([40000, 1, 30, 20000], [200, 1, 30, 65], 32, 8, 128),
                                               ([4000], [900], 40, 8, 256), ([3500, 20], [2600, 17], 32, 8, 128)],
                         ids=lambda l: f"{len(l)}x{max(l)}" if isinstance(l, list) else str(l))
def test_long_stretches(handle, lens, new, hq, hk, dh):  # noqa: F811
    """Stretches of more keys than an item has, whose first item's end comes last."""
    say(f"attention: long stretches, {len(lens)} sequences up to {max(lens)}, heads {hq}/{hk} Dh={dh}")
    rng = np.random.default_rng(sum(lens))
    t = R.scattered(rng, len(lens), lens, 208)
    run(Call(handle, rng, t, np.arange(len(lens)), new, hq, hk, dh))
