"""cs1_token_logprobs against log-softmax, entropy and a stable sort in float64."""
import numpy as np
import pytest

import decode_ref as R
from decode_ref import E32
from gpu_helpers import dev, empty, get, say, stream
from qwen3_5_native import hip

pytestmark = pytest.mark.gpu


def reference(x, targets, k):
    """Float64 results and bounds on a float32 computation's error.

    A difference d = x - m is off by E32 |d|, its product with log2 e by two more, so e^d by 3 E32 |d| of itself and the
    exponential's step of 2 E32.  A thread of 512 sums V / 512 values, and less than 100 more sums and changes of base (an
    exponential and two products, 6 E32 each) join it with the others; the weighted sum has the same and a product.  A base
    changes at most every 16 values of a thread."""
    rows, V = x.shape
    x = x.astype(np.float64)
    m = x.max(1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        d = x - m
        p = np.exp(d)
        z = p.sum(1, keepdims=True)
        D = np.where(np.isneginf(d), 0.0, d)
        depth = (V / 512 + 100 + 6 * (V / 512 / 16 + 20)) * E32
        rel = (p * (3 * np.abs(D) + 3) * E32).sum(1) / z[:, 0] + depth
        w = (p * np.abs(D)).sum(1) / z[:, 0]
        werr = (p * np.abs(D) * (3 * np.abs(D) + 5) * E32).sum(1) / z[:, 0] + w * (depth + rel)
        logz = np.log(z[:, 0])
        logp = d - logz[:, None]
        ent = logz - (p * D).sum(1) / z[:, 0]
    bad = ~(np.isfinite(z[:, 0]) & (z[:, 0] > 0))
    t_ok = (targets >= 0) & (targets < V)
    lp = np.where(t_ok, logp[np.arange(rows), np.clip(targets, 0, V - 1)], 0.0)
    step = 2 * E32 * (4 * np.abs(logz) + 1)
    ltol = rel + step + 3 * E32 * np.abs(np.where(np.isfinite(lp), lp, 0))
    etol = rel + step + werr + 3 * E32 * np.abs(ent)
    lp[bad & t_ok] = np.nan
    ent[bad] = np.nan
    order = np.argsort(-x, axis=1, kind="stable")[:, :k]
    n = order.shape[1]
    ids, top = np.full((rows, k), -1), np.full((rows, k), np.nan)
    ids[:, :n], top[:, :n] = order, np.take_along_axis(logp, order, 1)
    ids[bad], top[bad] = -1, np.nan
    ttol = (rel + step)[:, None] + 3 * E32 * np.abs(np.where(np.isfinite(top), top, 0))
    for tol in (ltol, etol, ttol):
        tol[bad] = 0  # NaN or 0, and nothing near them
    return (lp, ltol), (ent, etol), ids, (top, ttol)


class Call:
    """x: float values that the type holds; rows of `ld`, the first `off` values of the buffer left out."""

    def __init__(self, x, k, f32, targets=None, pad=0, off=0, rng=None, ent=True):
        self.x, self.k, self.f32, self.off, self.ent = x.astype(np.float32), k, f32, off, ent
        self.rows, self.V = x.shape
        self.ld = self.V + pad
        rng = rng or np.random.default_rng(0)
        self.targets = rng.integers(0, self.V, self.rows).astype(np.int32) if targets is None else np.asarray(targets, np.int32)

    def upload(self):
        full = np.full(off_end(self), 1e30, np.float32)  # what is no logit would be the best one
        full[self.off:].reshape(-1)[: self.rows * self.ld].reshape(self.rows, self.ld)[:, :self.V] = self.x
        self.size = 4 if self.f32 else 2
        self.buf = dev(full if self.f32 else R.O.f32_to_bf16(full))
        self.t = dev(self.targets)
        fill = lambda n: dev(np.full(n + 1, 77.0, np.float32))  # noqa: E731
        self.lp, self.e, self.top = fill(self.rows), fill(self.rows), fill(self.rows * self.k)
        self.ids = dev(np.full(self.rows * self.k + 1, 77, np.int32))
        need = hip.api().cs1_token_logprobs_workspace_bytes(self.rows, self.V, self.k)
        self.ws = empty(need) if need else None

    def launch(self, st=None):
        hip.check(hip.api().cs1_token_logprobs(
            self.buf.at(self.off * self.size), int(self.f32), self.ld, self.t.at(0), self.rows, self.V, self.k, self.lp.at(0),
            self.e.at(0) if self.ent else None, self.ids.at(0) if self.k else None, self.top.at(0) if self.k else None,
            self.ws.at(0) if self.ws else None, st or stream().handle), "token_logprobs")

    def results(self):
        n = self.rows * self.k
        out = [get(b, np.float32, c + 1) for b, c in ((self.lp, self.rows), (self.e, self.rows), (self.top, n))]
        ids = get(self.ids, np.int32, n + 1)
        assert all(o[-1] == 77 for o in out) and ids[-1] == 77, "written behind the last row"
        return out[0][:-1], out[1][:-1], ids[:-1].reshape(self.rows, self.k), out[2][:-1].reshape(self.rows, self.k)

    def check(self):
        lp, ent, ids, top = self.results()
        (wl, tl), (we, te), wi, (wt, tt) = reference(self.x, self.targets, self.k)
        R.close(lp.astype(np.float64), wl, tl, "logprob")
        if self.ent:
            R.close(ent.astype(np.float64), we, te, "entropy")
        else:
            assert (ent == 77).all()
        np.testing.assert_array_equal(ids, wi)
        R.close(top.astype(np.float64), wt, tt, "top")


def off_end(c):
    return c.off + c.rows * c.ld


def values(rng, rows, V, std, f32):
    x = (rng.standard_normal((rows, V)) * std).astype(np.float32)
    return x if f32 else R.f64(R.O.f32_to_bf16(x.reshape(-1))).reshape(rows, V).astype(np.float32)


def run(c):
    c.upload()
    c.launch()
    c.check()


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 33, 500, 4095, 4096, 4097, 40000, 151936, 248320])
def test_vocabularies(V, f32):
    say(f"logprobs V={V} f32={f32}")
    rng = np.random.default_rng(V)
    for rows, k, pad in ((1, 32, 0), (3, 5, 1), (2, 1, 24), (5, 0, 3)):
        run(Call(values(rng, rows, V, 3.0, f32), k, f32, pad=pad, rng=rng, ent=k != 1))


@pytest.mark.parametrize("rows,V", [(300, 6000), (1025, 700), (1500, 9001), (70, 33000)])
def test_many_rows(rows, V):
    say(f"logprobs {rows} rows of {V}")
    rng = np.random.default_rng(rows)
    run(Call(values(rng, rows, V, 2.0, False), 20, False, pad=rows % 8, rng=rng))


@pytest.mark.parametrize("off", range(1, 8))
def test_addresses(off):
    say(f"logprobs: from value {off} on, rows of an odd length")
    rng = np.random.default_rng(off)
    for f32 in (False, True):
        run(Call(values(rng, 4, 5003, 2.0, f32), 7, f32, off=off, rng=rng))


@pytest.mark.parametrize("rows", [2, 1100])
@pytest.mark.parametrize("V", [40, 5000])
def test_masked_logits(rows, V):
    """A few tokens allowed, all others -inf; some rows with none, a NaN or an infinity."""
    say(f"logprobs: masks, {rows} rows of {V}")
    rng = np.random.default_rng(V)
    x = values(rng, rows, V, 2.0, True)
    for r in range(rows):
        allowed = rng.permutation(V)[:1 + r % 9]
        keep = np.full(V, -np.inf, np.float32)
        keep[allowed] = x[r, allowed]
        x[r] = keep
    if rows > 2:
        x[5] = -np.inf
        x[6, 3] = np.nan
        x[7, V - 1] = np.inf
        x[8] = np.nan
        x[9, 0] = np.float32(-3.4e38)  # a mask of the type's lowest value
        x[10] = np.where(np.isneginf(x[10]), np.float32(-3.4e38), x[10])
    run(Call(x, 16, True, rng=rng))
    if rows > 2:
        lowest = R.f64(np.array([0xff7f], np.uint16))[0]
        x[9, 0], x[10] = lowest, np.where(x[10] < -1e38, lowest, R.f64(R.O.f32_to_bf16(x[10])))
    y = np.where(np.isfinite(x), R.f64(R.O.f32_to_bf16(np.where(np.isfinite(x), x, 0).reshape(-1))).reshape(x.shape), x)
    run(Call(y, 16, False, rng=rng))


@pytest.mark.parametrize("V", [64, 5000, 200000])
def test_equal_logits(V):
    """The lowest index first: all equal, two values, zeros of both signs."""
    say(f"logprobs: ties, V={V}")
    rng = np.random.default_rng(V)
    x = np.zeros((4, V), np.float32)
    x[0] = 1.5
    x[1] = rng.integers(0, 2, V)
    x[2] = np.where(rng.random(V) < 0.5, -0.0, 0.0)
    x[3] = np.floor(rng.standard_normal(V) * 2)
    for f32 in (False, True):
        run(Call(x, 32, f32, rng=rng))


@pytest.mark.parametrize("V", [3000, 150000])
def test_orders(V):
    """Rising, falling, and the large ones in few threads' loads (more than the list holds)."""
    say(f"logprobs: orders, V={V}")
    x = np.zeros((5, V), np.float32)
    x[0] = np.linspace(-5, 5, V)
    x[1] = np.linspace(5, -5, V)
    lane = np.arange(V) // 4 % 64  # the lane of a float32 load in the block
    x[2] = np.where(lane == 7, 50.0 + np.arange(V) % 1000 / 8, 0.0)
    x[3] = np.where(lane < 20, 9.0, 0.0) + np.arange(V) % 3
    x[4] = np.where(lane == 63, np.arange(V), -1.0)
    run(Call(x, 32, True))
    many = np.repeat(x[2:3], 1024, 0) + np.arange(1024, dtype=np.float32)[:, None] / 16 if V < 10000 else x[2:3]
    run(Call(many.astype(np.float32), 20, True))


def test_large_list_of_one_part():
    say("logprobs: one part, thousands above the threshold")
    V = 60000
    rows = 1024  # a part a row
    x = np.zeros((rows, V), np.float32)
    lane = (np.arange(V) // 4 + 1) % 64
    x[:] = np.where(lane == 3, 40.0, -1.0)[None]
    x[::2, 17::64] += 1.0
    x[3] = np.where(lane == 9, np.arange(V) % 977, -1.0)
    assert hip.api().cs1_token_logprobs_workspace_bytes(rows, V, 9) == 0
    run(Call(x, 9, True))


@pytest.mark.parametrize("shift", [0.0, 1e4, -3e4, 1e30])
def test_large_logits(shift):
    """The values' common part costs nothing but their own bits."""
    say(f"logprobs: around {shift}")
    rng = np.random.default_rng(3)
    x = values(rng, 6, 7000, 2.0, True) + np.float32(shift)
    x[4:, ::3] = shift - 500
    run(Call(x, 8, True, rng=rng))


def test_targets_out_of_range():
    say("logprobs: no target")
    rng = np.random.default_rng(5)
    c = Call(values(rng, 6, 100, 2.0, False), 2, False, targets=[-1, 99, 100, 2 ** 31 - 1, -2 ** 31, 0])
    run(c)
    lp = c.results()[0]
    assert (lp[[0, 2, 3, 4]] == 0).all() and (lp[[1, 5]] < 0).all()


def test_no_targets_and_no_entropy():
    say("logprobs: alternatives only")
    rng = np.random.default_rng(6)
    c = Call(values(rng, 3, 9000, 2.0, False), 4, False, ent=False)
    c.upload()
    hip.check(hip.api().cs1_token_logprobs(c.buf.at(0), 0, c.ld, None, 3, c.V, 4, None, None, c.ids.at(0), c.top.at(0), c.ws.at(0),
                                           stream().handle), "token_logprobs")
    lp, _, ids, _ = c.results()
    assert (lp == 77).all()
    np.testing.assert_array_equal(ids, reference(c.x, c.targets, 4)[2])


def test_offsets_past_32_bits():
    say("logprobs: rows past 8 GiB")
    V, rows = 1 << 20, 4200
    rng = np.random.default_rng(7)
    buf = hip.DeviceBuffer(rows * V * 2)
    x = values(rng, 1, V, 2.0, False)
    row = R.O.f32_to_bf16(x.reshape(-1))
    at = [0, 2047, 2048, 4095, 4199]
    c = Call(np.repeat(x, len(at), 0), 6, False, rng=rng)
    ids, top, lp, e = empty(4 * rows * 6), empty(4 * rows * 6), empty(4 * rows), empty(4 * rows)
    t = dev(np.full(rows, 12345, np.int32))
    for r in at:
        hip.upload(buf, row, stream(), offset=r * V * 2)
    assert hip.api().cs1_token_logprobs_workspace_bytes(rows, V, 6) == 0
    hip.check(hip.api().cs1_token_logprobs(buf.at(0), 0, V, t.at(0), rows, V, 6, lp.at(0), e.at(0), ids.at(0), top.at(0), None,
                                           stream().handle), "token_logprobs")
    (wl, tl), _, wi, _ = reference(c.x, np.full(len(at), 12345), 6)
    np.testing.assert_array_equal(get(ids, np.int32, rows * 6).reshape(rows, 6)[at], wi)
    R.close(get(lp, np.float32, rows)[at].astype(np.float64), wl, tl, "logprob")


def test_graph_replays_and_repeats():
    say("logprobs: replays give the same bits")
    rng = np.random.default_rng(8)
    for rows in (2, 1200):
        c = Call(values(rng, rows, 12000, 2.0, False), 10, False, rng=rng)
        c.upload()
        c.launch()
        first = c.results()
        graph = hip.Graph(stream(), c.launch)
        for _ in range(3):
            graph.launch(stream())
            for a, b in zip(first, c.results()):
                np.testing.assert_array_equal(a, b)
        c.check()
