"""cs1_token_logprobs from 2^26 logits on, where blocks have 512 threads: parts that are joined and rows in one part,
both types, rows on odd addresses, rows without a distribution, ties and full lists."""
import numpy as np
import pytest

import decode_ref as R
from decode_ref import E32
from gpu_helpers import dev, empty, get, say, stream
from qwen3_5_native import hip
from test_gpu_logprobs import values

pytestmark = pytest.mark.gpu
THREADS = 512


def reference(x):
    """Float64 log-probabilities [rows, V], entropies, and the bounds on a float32 computation of these.

    A difference d from the largest is off by E32 |d| and its product with log2 e by two more, so e^d by 3 E32 |d| of itself
    and the exponential's step of 2 E32.  A thread sums up to n = V / 512 values (a part of a row: fewer) and moves its base
    at most once for the 16 values or more that it has under way, and under 100 more sums and 20 more changes of base (an
    exponential and two products: 6 E32) join it with the others of a block, and blocks.  The weighted sum has the
    same and a product.  The logarithm and the two differences that are left are a step of what they give each."""
    V = x.shape[1]
    x = x.astype(np.float64)
    n = V / THREADS
    m = x.max(1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        d = x - m
        p = np.exp(d)
        z = p.sum(1, keepdims=True)
        D = np.abs(np.where(np.isneginf(d), 0.0, d))
        depth = (n + 100 + 6 * (n / 16 + 20)) * E32
        rel = (p * (3 * D + 3) * E32).sum(1) / z[:, 0] + depth
        w = (p * D).sum(1) / z[:, 0]
        werr = (p * D * (3 * D + 5) * E32).sum(1) / z[:, 0] + w * (depth + rel)
        logz = np.log(z[:, 0])
        logp = d - logz[:, None]
        ent = logz + w
    bad = ~(np.isfinite(z[:, 0]) & (z[:, 0] > 0))
    step = rel + 2 * E32 * (4 * np.abs(logz) + 1)
    tol = step[:, None] + 3 * E32 * np.abs(np.where(np.isfinite(logp), logp, 0))
    etol = step + werr + 3 * E32 * np.abs(ent)
    logp[bad], ent[bad], tol[bad], etol[bad] = np.nan, np.nan, 0, 0
    return logp, tol, ent, etol, bad


def rows_of_interest(rng, V, f32):
    x = values(rng, 11, V, 2.0, f32)
    x[1] = np.where(rng.random(V) < 10 / V, x[1], -np.inf)  # a few tokens allowed
    x[1, V // 2] = 0.25
    x[2] = -np.inf
    x[3, V - 2] = np.nan
    x[4, 1] = np.inf
    x[5] = 0.5  # ties: the lowest index first
    x[6] = np.where(rng.random(V) < 0.5, -0.0, 0.0)
    x[7] = np.floor(x[7])
    # large ones in a lane's loads alone, more than the list of candidates holds
    each = 4 if f32 else 8
    x[8] = np.where(np.arange(V) // each % 64 == 7, 40.0, -1.0)
    x[9] = np.where(np.arange(V) // each % 64 == 63, np.arange(V) % 97, -1.0)
    return x


@pytest.mark.parametrize("rows,V,k,pad,off,f32", [
    (500, 151936, 32, 0, 0, False),   # three parts a row
    (500, 151936, 20, 1, 3, False),   # rows on odd addresses
    (460, 151936, 32, 3, 1, True),
    (1100, 70001, 32, 0, 0, True),    # one part a row
    (1100, 70001, 5, 5, 7, False),
    (1100, 70001, 0, 0, 0, False),
    (1100, 70000, 0, 0, 0, True),
    (1100, 70000, 32, 8, 0, False),   # rows on whole loads: full lists
    (300, 248320, 1, 0, 0, True),
], ids=str)
def test_rows(rows, V, k, pad, off, f32):
    assert rows * V >= 1 << 26
    say(f"logprobs: {rows} rows of {V}, k={k}, pad {pad}, from {off}, f32={f32}")
    rng = np.random.default_rng(rows + V + k)
    x = rows_of_interest(rng, V, f32)
    distinct, ld = len(x), V + pad
    of = np.arange(rows) % distinct  # the row that a row of the batch repeats
    full = np.full(off + rows * ld, 1e30, np.float32)  # what is no logit would be the best one
    full[off:].reshape(rows, ld)[:, :V] = x[of]
    buf = dev(full if f32 else R.O.f32_to_bf16(full))
    targets = rng.integers(0, V, rows).astype(np.int32)
    targets[20:30] = [-1, V, 0, V - 1, 2 ** 31 - 1, -2 ** 31, V // 2, 1, 2, V - 2]
    t = dev(targets)
    lp, ent = dev(np.full(rows + 1, 77, np.float32)), dev(np.full(rows + 1, 77, np.float32))
    top, ids = dev(np.full(rows * k + 1, 77, np.float32)), dev(np.full(rows * k + 1, 77, np.int32))
    need = hip.api().cs1_token_logprobs_workspace_bytes(rows, V, k)
    ws = empty(need) if need else None

    def launch():
        hip.check(hip.api().cs1_token_logprobs(buf.at(off * (4 if f32 else 2)), int(f32), ld, t.at(0), rows, V, k, lp.at(0), ent.at(0),
                                               ids.at(0) if k else None, top.at(0) if k else None, ws.at(0) if ws else None,
                                               stream().handle), "token_logprobs")
        got = [get(lp, np.float32, rows + 1), get(ent, np.float32, rows + 1), get(ids, np.int32, rows * k + 1),
               get(top, np.float32, rows * k + 1)]
        assert all(g[-1] == 77 for g in got), "written behind the last row"
        return [g[:-1] for g in got]

    first = launch()
    for a, b in zip(first, launch()):
        np.testing.assert_array_equal(a, b)
    logp, tol, went, etol, bad = reference(x)
    there = (targets >= 0) & (targets < V)
    at = np.clip(targets, 0, V - 1)
    R.close(first[0].astype(np.float64), np.where(there, logp[of, at], 0.0), np.where(there, tol[of, at], 0.0), "logprob")
    R.close(first[1].astype(np.float64), went[of], etol[of], "entropy")
    order = np.argsort(-x, axis=1, kind="stable")[:, :k]
    best, btol = np.take_along_axis(logp, order, 1), np.take_along_axis(tol, order, 1)
    order[bad] = -1
    np.testing.assert_array_equal(first[2].reshape(rows, k), order[of])
    R.close(first[3].reshape(rows, k).astype(np.float64), best[of], btol[of], "top")
