"""cs1_token_logprobs with a workspace that was made for more rows: batches of any smaller size stay inside of it."""
import numpy as np
import pytest

import decode_ref as R
from gpu_helpers import dev, empty, get, say, stream
from qwen3_5_native import hip
from test_gpu_logprobs import reference, values

pytestmark = pytest.mark.gpu
GUARD = 4096


@pytest.mark.parametrize("most,V,k", [(512, 151936, 20), (1023, 20000, 32), (70, 248320, 1)])
def test_fewer_rows(most, V, k):
    rng = np.random.default_rng(most)
    api = hip.api()
    need = api.cs1_token_logprobs_workspace_bytes(most, V, k)
    distinct = 5  # rows; row r of the batch is number r % 5
    x = values(rng, distinct, V, 2.0, False)
    buf = dev(R.O.f32_to_bf16(x[np.arange(most) % distinct].reshape(-1)))
    target = 77
    t = dev(np.full(most, target, np.int32))
    lp, ent, top, ids = empty(4 * most), empty(4 * most), empty(4 * most * k), empty(4 * most * k)
    (wl, tl), (we, te), wi, (wt, tt) = reference(x, np.full(distinct, target), k)
    for rows in sorted({1, 2, 3, 37, most // 3, most // 2, most - 1, most}):
        say(f"logprobs: {rows} rows of {V} in a workspace for {most}")
        assert api.cs1_token_logprobs_workspace_bytes(rows, V, k) <= need
        pattern = rng.integers(0, 256, need + GUARD).astype(np.uint8)
        ws = dev(pattern)
        hip.check(api.cs1_token_logprobs(buf.at(0), 0, V, t.at(0), rows, V, k, lp.at(0), ent.at(0), ids.at(0), top.at(0), ws.at(0),
                                         stream().handle), "token_logprobs")
        of = np.arange(rows) % distinct
        np.testing.assert_array_equal(get(ids, np.int32, rows * k).reshape(rows, k), wi[of])
        R.close(get(lp, np.float32, rows).astype(np.float64), wl[of], tl[of], "logprob")
        R.close(get(ent, np.float32, rows).astype(np.float64), we[of], te[of], "entropy")
        R.close(get(top, np.float32, rows * k).reshape(rows, k).astype(np.float64), wt[of], tt[of], "top")
        np.testing.assert_array_equal(get(ws, np.uint8, need + GUARD)[need:], pattern[need:])
