"""cs1_attn_prep_paged against norm and rotation in float64, within bounds that follow from float32's and one bfloat16
rounding (rows_ref.turned)."""
import ctypes

import numpy as np
import pytest

import decode_ref as R
import rows_ref as W
from gpu_helpers import dev, get, get_bf16, say, stream
from qwen3_5_native import hip

pytestmark = pytest.mark.gpu
EPS = 1e-6


class Call:
    def __init__(self, rng, T, hq, hk, dh, dims, interleaved=False, gate=True, norm=True, magnitude=1.0, base=1e7, far=5000, page=16,
                 pad=0, std=1.0):
        self.T, self.hq, self.hk, self.dh, self.dims, self.inter = T, hq, hk, dh, dims, interleaved
        self.mag = float(np.float32(magnitude))
        self.wq, self.ld = hq * dh * (2 if gate else 1), hq * dh * (2 if gate else 1) + 2 * hk * dh + 8
        self.x = R.bf16(rng, T, self.ld, std=std)
        self.gate = gate
        self.w = [R.bf16(rng, dh, std=0.2) for _ in range(2)] if norm else [None, None]
        self.freqs = base ** (-np.arange(0, max(dims, 2), 2) / max(dims, 2))
        self.npages, self.page = R.cdiv(T, page) + 2, page
        self.pos = rng.integers(0, far, T).astype(np.int32)
        self.slot = rng.permutation(self.npages * page)[:T].astype(np.int32)
        if pad:
            self.pos[-pad:], self.slot[-pad:] = -1, -1

    def upload(self):
        T, hq, hk, dh = self.T, self.hq, self.hk, self.dh
        self.d = {"x": dev(self.x), "pos": dev(self.pos), "slot": dev(self.slot), "freqs": dev(self.freqs)}
        for name, w in zip(("qw", "kw"), self.w):
            self.d[name] = dev(w) if w is not None else None
        fill = lambda n: dev(np.full(n + 8, 0x7fc1, np.uint16))  # noqa: E731
        self.q, self.g = fill(T * hq * dh), fill(T * hq * dh)
        self.pools = [fill(self.npages * self.page * hk * dh) for _ in range(2)]

    def launch(self, st=None):
        d, x = self.d, self.d["x"]
        rot = hip.Rotary(d["freqs"].at(0) if self.dims else None, self.dims, int(self.inter), self.mag)
        pages = hip.PageTable(None, None, None, 1, 1, self.npages, self.page)
        ptr = lambda b: b.at(0) if b is not None else None  # noqa: E731
        hip.check(hip.api().cs1_attn_prep_paged(
            x.at(0), x.at(2 * self.wq), x.at(2 * (self.wq + self.hk * self.dh)), self.ld, ptr(d["qw"]), ptr(d["kw"]), EPS,
            ctypes.byref(rot), ctypes.byref(pages), d["pos"].at(0), d["slot"].at(0), self.q.at(0), self.g.at(0) if self.gate else None,
            self.pools[0].at(0), self.pools[1].at(0), self.T, self.hq, self.hk, self.dh, st or stream().handle), "prep")

    def check(self):
        T, hq, hk, dh = self.T, self.hq, self.hk, self.dh
        live = self.pos >= 0
        n = T * hq * dh
        q, g = get_bf16(self.q, n + 8), get_bf16(self.g, n + 8)
        assert (q[n:] == 0x7fc1).all() and (g[n:] == 0x7fc1).all()
        q, g = q[:n].reshape(T, hq, dh), g[:n].reshape(T, hq, dh)
        assert (q[~live] == 0x7fc1).all() and (g[~live] == 0x7fc1).all(), "rows of no one are written"
        raw = self.x[:, :self.wq].reshape(T, hq, -1)
        if self.gate:
            np.testing.assert_array_equal(g[live], raw[live][..., dh:])
        else:
            assert (g == 0x7fc1).all()

        def want(x, w):
            return W.turned(R.f64(np.ascontiguousarray(x[live])), R.f64(w) if w is not None else None, EPS, self.pos[live], self.freqs,
                            self.dims, self.inter, self.mag)

        y, tol = want(raw[..., :dh], self.w[0])
        R.close(R.f64(q[live]), y, tol, "q")
        kv = self.x[:, self.wq:self.wq + 2 * hk * dh].reshape(T, 2, hk, dh)
        m = self.npages * self.page
        kp, vp = (get_bf16(b, m * hk * dh + 8) for b in self.pools)
        assert (kp[-8:] == 0x7fc1).all() and (vp[-8:] == 0x7fc1).all()
        kp, vp = kp[:-8].reshape(m, hk, dh), vp[:-8].reshape(m, hk, dh)
        put = live & (self.slot >= 0) & (self.slot < m)
        rest = np.setdiff1d(np.arange(m), self.slot[put])
        assert (kp[rest] == 0x7fc1).all() and (vp[rest] == 0x7fc1).all(), "slots of no row are written"
        np.testing.assert_array_equal(vp[self.slot[put]], kv[put, 1])
        y, tol = want(kv[:, 0], self.w[1])
        at = put[live]
        R.close(R.f64(kp[self.slot[put]]), y[at], tol[at], "k")


@pytest.mark.parametrize("hq,hk,dh", [(16, 4, 128), (16, 4, 256), (24, 4, 256), (1, 1, 128), (1, 1, 256), (6, 2, 128), (40, 8, 256), (71, 3, 128)])
@pytest.mark.parametrize("dims,interleaved", [(0, False), (16, False), (16, True), (64, False), (96, True), (128, False), (128, True), (112, False)])
def test_heads_and_layouts(hq, hk, dh, dims, interleaved):
    say(f"prep paged heads {hq}/{hk} Dh={dh} dims={dims} interleaved={interleaved}")
    c = Call(np.random.default_rng(hq + dims), 5, hq, hk, dh, dims, interleaved, gate=hq % 3 != 0, norm=dims % 32 == 0)
    c.upload()
    c.launch()
    c.check()


@pytest.mark.parametrize("interleaved", [False, True])
def test_whole_heads_of_256(interleaved):
    say("prep paged: all 256 dims")
    c = Call(np.random.default_rng(2), 33, 8, 2, 256, 256, interleaved, magnitude=1.2079)
    c.upload()
    c.launch()
    c.check()


@pytest.mark.parametrize("far", [1, 2 ** 20, 2 ** 31 - 1])
def test_positions(far):
    """First tokens, and positions whose angles float32 does not hold."""
    say(f"prep paged: positions below {far}")
    c = Call(np.random.default_rng(far % 97), 130, 4, 2, 128, 128, far == 1, norm=far > 1, far=far, base=1e4, magnitude=1.1)
    if far > 1:
        c.pos[:2] = far - 1, 0
    c.upload()
    c.launch()
    c.check()


def test_one_weight_only():
    say("prep paged: norm of q alone, of k alone")
    for which in range(2):
        c = Call(np.random.default_rng(which), 9, 4, 4, 256, 64)
        c.w[which] = None
        c.upload()
        c.launch()
        c.check()


@pytest.mark.parametrize("T,pad", [(1, 1), (300, 45), (2000, 1)])
def test_rows_of_no_one(T, pad):
    say(f"prep paged: {pad} of {T} rows padding, slots out of range")
    rng = np.random.default_rng(T)
    c = Call(rng, T, 16, 4, 128, 32, pad=pad, page=48)
    for i, bad in enumerate((-1, -2 ** 31, c.npages * 48, 2 ** 31 - 1)):
        if i < T - pad:
            c.slot[i] = bad
    c.upload()
    c.launch()
    c.check()


@pytest.mark.parametrize("std", [1e-18, 3e-4, 1e4])
def test_sizes_of_values(std):
    say(f"prep paged: values of {std}")
    c = Call(np.random.default_rng(4), 17, 4, 2, 256, 64, std=std)
    c.upload()
    c.launch()
    c.check()


def test_pool_past_4_gib():
    say("prep paged: slots past 4 GiB")
    c = Call(np.random.default_rng(5), 6, 4, 16, 256, 64, page=256)
    T, hk, dh, npages = c.T, c.hk, c.dh, 2100  # 4.4 GB a pool
    c.slot = np.array([0, 524287, 524288, 524289, npages * 256 - 1, 300000], np.int32)
    c.upload()
    c.npages, c.pools = npages, [hip.DeviceBuffer(npages * 256 * hk * dh * 2) for _ in range(2)]
    assert (c.slot < c.npages * c.page).all() and all(b.nbytes == c.npages * c.page * hk * dh * 2 for b in c.pools)
    c.launch()
    kv = c.x[:, c.wq:c.wq + 2 * hk * dh].reshape(T, 2, hk, dh)
    y, tol = W.turned(R.f64(np.ascontiguousarray(kv[:, 0])), R.f64(c.w[1]), EPS, c.pos, c.freqs, c.dims, False, 1.0)
    for i, s in enumerate(c.slot):
        at = int(s) * hk * dh * 2
        np.testing.assert_array_equal(get(c.pools[1], np.uint16, hk * dh, at).reshape(hk, dh), kv[i, 1])
        R.close(R.f64(get(c.pools[0], np.uint16, hk * dh, at).reshape(hk, dh)), y[i], tol[i], f"k of slot {s}")


def test_rows_from_the_map():
    """Positions and slots as cs1_kv_rows leaves them, several sequences in one call."""
    say("prep paged behind kv_rows, in a graph")
    rng = np.random.default_rng(6)
    t = R.scattered(rng, 5, [50, 3, 0, 130, 17], 16)
    d = R.DeviceTable(t)
    seqs, cu = [3, 1, -1, 0, 4], np.array([0, 20, 23, 25, 30, 47], np.int32)
    c = Call(rng, 50, 8, 2, 128, 128)
    c.npages = t.npages
    c.pos, c.slot = W.rows_of(t, seqs, cu, 50)
    c.upload()
    hip.upload(c.d["pos"], np.zeros(50, np.int32), stream())
    hip.upload(c.d["slot"], np.zeros(50, np.int32), stream())
    b, off = R.ints(seqs), R.ints(cu)

    def record():
        hip.check(hip.api().cs1_kv_rows(d.ref, b.at(0), off.at(0), 5, 50, c.d["pos"].at(0), c.d["slot"].at(0), stream().handle), "rows")
        c.launch()

    graph = hip.Graph(stream(), record)
    for _ in range(3):
        graph.launch(stream())
        c.check()
        hip.upload(c.q, np.full(50 * 8 * 128 + 8, 0x7fc1, np.uint16), stream())
