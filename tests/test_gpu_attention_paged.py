"""cs1_attention_paged against attention in float64 (decode_ref.attention), within bounds that follow from
the roundings of float32 sums and one bfloat16 output."""
import ctypes

import numpy as np
import pytest

import decode_ref as R
from decode_ref import DeviceTable, ints
from gpu_helpers import dev, empty, get, get_bf16, say, stream
from qwen3_5_native import hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def handle():
    stream()
    h = hip.api().cs1_attention_paged_create()
    assert h
    yield h
    hip.api().cs1_attention_paged_destroy(h)


class Call:
    def __init__(self, handle, rng, t, seqs, hq, hk, dh, gate=True, lse=True, std=1.0):
        self.handle, self.t, self.seqs, self.hq, self.hk, self.dh = handle, t, np.asarray(seqs, np.int32), hq, hk, dh
        B = len(seqs)
        self.q, self.gate = R.bf16(rng, B, hq, dh, std=std), R.bf16(rng, B, hq, dh) if gate else None
        self.kp, self.vp = R.bf16(rng, t.npages, t.page, hk, dh, std=std), R.bf16(rng, t.npages, t.page, hk, dh)
        self.lse = lse

    def upload(self):
        self.d = DeviceTable(self.t)
        self.bufs = [dev(x) for x in (self.q, self.kp, self.vp, self.seqs)]
        self.g = dev(self.gate) if self.gate is not None else None
        B = len(self.seqs)
        self.out, self.l = dev(np.full(B * self.hq * self.dh + 8, 0x7fc1, np.uint16)), dev(np.full(B * self.hq + 1, 5.0, np.float32))

    def launch(self, st=None, null=False):
        q, kp, vp, seqs = self.bufs
        hip.check(hip.api().cs1_attention_paged(
            self.handle, q.at(0), kp.at(0), vp.at(0), self.d.ref, None if null else seqs.at(0), self.g.at(0) if self.g else None,
            self.out.at(0), self.l.at(0) if self.lse else None, len(self.seqs), self.hq, self.hk, self.dh, self.dh ** -0.5,
            st or stream().handle), "attention_paged")

    def results(self):
        B = len(self.seqs)
        n = B * self.hq * self.dh
        out, l = get_bf16(self.out, n + 8), get(self.l, np.float32, B * self.hq + 1)
        assert (out[n:] == 0x7fc1).all() and l[-1] == 5.0, "written behind the last row"
        return out[:n].reshape(B, self.hq, self.dh), l[:-1].reshape(self.hq, B)

    def check(self, seqs=None):
        out, l = self.results()
        want, wl, tol, ltol = R.attention(self.t, self.seqs if seqs is None else seqs, self.q, self.kp, self.vp, self.gate,
                                          self.hk, self.dh ** -0.5)
        R.close(R.f64(out), want, tol, "out")
        if self.lse:
            R.close(l.astype(np.float64), wl, ltol, "lse")


@pytest.mark.parametrize("hq,hk,dh", [(16, 4, 128), (16, 4, 256), (24, 4, 256), (4, 4, 128), (16, 1, 256), (6, 2, 128), (32, 1, 128),
                                      (17, 1, 256), (40, 2, 128), (1, 1, 256)])
@pytest.mark.parametrize("page", [16, 48, 64])
def test_head_layouts(handle, hq, hk, dh, page):
    say(f"paged attention heads {hq}/{hk} Dh={dh} page={page}")
    rng = np.random.default_rng(hq * hk + page)
    lens = [1, 0, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 130, 257, 300]
    t = R.scattered(rng, len(lens) + 2, lens, page)
    c = Call(handle, rng, t, rng.permutation(len(lens) + 2), hq, hk, dh, gate=page != 64, lse=page != 16)
    c.upload()
    c.launch()
    c.check()


@pytest.mark.parametrize("lens", [[5000], [1, 4000], [700, 700, 700], [8191, 3, 0, 900], [127] * 70, [12000, 1, 1, 1, 1],
                                  list(range(1, 400, 7)), [2049], [40000]], ids=lambda l: f"{len(l)}x{max(l)}")
@pytest.mark.parametrize("hq,hk,dh,page", [(16, 4, 128, 16), (24, 4, 256, 208), (20, 1, 256, 32)])
def test_lengths(handle, lens, hq, hk, dh, page):
    """Sequences that fill the chip alone and together, split and whole."""
    say(f"paged attention {len(lens)} sequences up to {max(lens)}, heads {hq}/{hk} Dh={dh} page={page}")
    rng = np.random.default_rng(sum(lens) + dh)
    t = R.scattered(rng, len(lens), lens, page)
    c = Call(handle, rng, t, rng.permutation(len(lens)), hq, hk, dh)
    c.upload()
    c.launch()
    c.check()


def test_padding_repeats_and_no_list(handle):
    say("paged attention: padding rows, a sequence twice, no list")
    rng = np.random.default_rng(3)
    t = R.scattered(rng, 5, [70, 0, 33, 500, 16], 16)
    c = Call(handle, rng, t, [3, -1, 0, 5, 0, 2 ** 31 - 1, 1, -2 ** 31, 4, 3], 8, 2, 128)
    c.upload()
    c.launch()
    c.check()
    out, l = c.results()
    for r in (1, 3, 5, 6, 7):
        assert (out[r] == 0).all() and (l[:, r] == -np.inf).all()
    c.launch(null=True)  # row i is sequence i; rows from nseq on are padding
    c.check(seqs=list(range(5)) + [-1] * 5)


def test_what_is_not_held_is_not_read(handle):
    """NaN and infinities in every slot that no token of the sequence has, and in pages of others."""
    say("paged attention: NaN around")
    rng = np.random.default_rng(4)
    lens = [1, 17, 40, 129, 1000, 0]
    t = R.scattered(rng, 6, lens, 48)
    c = Call(handle, rng, t, range(6), 16, 4, 256)
    held = np.zeros((t.npages, t.page), bool)
    for s, n in enumerate(lens):
        for j in range(n):
            held[t.table[s, j // 48], j % 48] = True
    for pool, bits in ((c.kp, 0x7fc0), (c.vp, 0x7f80)):
        pool[~held] = bits
    c.vp[~held, :, ::2] = 0xffc0
    c.upload()
    c.launch()
    c.check()
    assert np.isfinite(R.f64(c.results()[0])).all()


def test_a_token_of_infinities_is_its_own_rows_matter(handle):
    say("paged attention: infinite values in one sequence")
    rng = np.random.default_rng(5)
    t = R.scattered(rng, 3, [40, 50, 300], 16)
    c = Call(handle, rng, t, range(3), 8, 4, 128)
    c.vp[t.table[1, 0], 5, 2, 7] = 0x7f80  # +inf in kv head 2, dim 7
    c.kp[t.table[2, 3], 0, 1] = 0x7fc0     # NaN keys in kv head 1
    c.upload()
    c.launch()
    out = R.f64(c.results()[0])
    assert np.isfinite(out[0]).all()
    hit = np.zeros((8, 128), bool)
    hit[4:6, 7] = True
    assert (out[1][hit] == np.inf).all() and np.isfinite(out[1][~hit]).all()
    assert np.isnan(out[2, 2:4]).all() and np.isfinite(out[2, :2]).all() and np.isfinite(out[2, 4:]).all()


@pytest.mark.parametrize("dh", [128, 256])
def test_a_key_without_weight_adds_nothing(handle, dh):
    """Values of bfloat16's largest size under keys whose weight is far below float32's range."""
    say(f"paged attention: the largest values without weight, Dh={dh}")
    rng = np.random.default_rng(15)
    t = R.scattered(rng, 2, [40, 700], 16)
    c = Call(handle, rng, t, range(2), 8, 4, dh)
    c.q[:], c.kp[:] = 0, 0
    c.q[..., 0] = R.O.f32_to_bf16(np.full(c.q[..., 0].size, 128.0, np.float32)).reshape(c.q[..., 0].shape)
    low = R.O.f32_to_bf16(np.array([-64.0], np.float32))[0]  # scores of 0 but for these: -512 and less
    for s, j in ((0, 5), (0, 39), (1, 0), (1, 321), (1, 699)):
        at = t.table[s, j // 16], j % 16
        c.kp[at][:, 0] = low
        c.vp[at] = np.where(rng.random((4, dh)) < 0.5, 0x7f7f, 0xff7f)
    c.upload()
    c.launch()
    c.check()


def test_weights_keep_all_their_bits(handle):
    """Three keys whose values cancel to 2^-18 of their size: what a weight loses below float32's last bits shows.

    Scores 0, S and 0 with one product each, exact up to the exponential's argument (two roundings of |S log2 e| < 1.5)
    and the exponential (one step): the weight of S is off by 4 E32.  Three products of three parts each are summed: 8
    sums, a step of the largest term at most, 16 E32.  The terms are of the size of the middle one, below 2."""
    say("paged attention: weights to the last bit")
    rng = np.random.default_rng(16)
    hk, dh = 4, 256
    t = R.scattered(rng, 1, [3], 16)
    c = Call(handle, rng, t, [0], hk, hk, dh, gate=False)
    c.q[:], c.kp[:] = 0, 0
    c.q[..., 0] = 0x4180  # 16, so that the score is the key's value
    grid = R.f64(np.arange(0xbe80, 0xbf80, dtype=np.uint16))  # -1/4 to -1
    w = np.exp(grid).astype(np.float32)
    rest = w - R.f64((w.view(np.uint32) >> 16).astype(np.uint16))
    lost = np.abs(rest - R.f64(R.O.f32_to_bf16(rest.astype(np.float32)).reshape(-1))) / w  # in two parts
    S = grid[np.argsort(lost)[-hk:]]
    bf = lambda x: R.O.f32_to_bf16(np.asarray(x, np.float32).reshape(-1)).reshape(np.shape(x))  # noqa: E731
    page = t.table[0, 0]
    c.kp[page, 1, :, 0] = bf(S)
    p = np.exp(S)[:, None]
    v1 = bf(rng.uniform(1, 2, (hk, dh)))
    v0 = bf(-p * R.f64(v1))
    v2 = bf(-(p * R.f64(v1) + R.f64(v0)))
    c.vp[page, 0], c.vp[page, 1], c.vp[page, 2] = v0, v1, v2
    want = (p * R.f64(v1) + R.f64(v0) + R.f64(v2)) / (p + 2)
    assert np.abs(want).max() < 2.0 ** -16
    c.upload()
    c.launch()
    out, _ = c.results()
    R.close(R.f64(out)[0], want, 20 * R.E32 * 2 / (p + 2) + 1.01 * R.E16 * np.abs(want), "out")


@pytest.mark.parametrize("std", [8.0, 40.0])
def test_large_scores(handle, std):
    """Scores of hundreds to tens of thousands: the maximum moves by far more than a float's exponent holds."""
    say(f"paged attention: large scores, std {std}")
    rng = np.random.default_rng(6)
    t = R.scattered(rng, 4, [3000, 100, 1, 650], 32)
    c = Call(handle, rng, t, range(4), 16, 4, 128, std=std)
    c.upload()
    c.launch()
    c.check()


def test_bad_page_numbers_are_masked(handle):
    say("paged attention: page numbers out of range")
    rng = np.random.default_rng(7)
    t = R.scattered(rng, 4, [100, 700, 30, 64], 16)
    t.table[0, 2], t.table[1, 0], t.table[1, 43], t.table[2] = t.npages, -1, 2 ** 31 - 1, -2 ** 31
    c = Call(handle, rng, t, range(4), 16, 4, 256)
    c.upload()
    c.launch()
    c.check()


def test_more_tokens_than_the_table_has_room_for(handle):
    say("paged attention: a length past the table's row")
    rng = np.random.default_rng(8)
    t = R.scattered(rng, 2, [64, 20], 16, max_pages=4)
    c = Call(handle, rng, t, range(2), 8, 4, 128)
    c.upload()
    lens = dev(np.array([2 ** 31 - 1, 20], np.int32))
    c.d.struct.lens = lens.at(0)
    c.launch()
    c.check()


def test_the_same_bits_every_time_and_in_a_graph(handle):
    """Repeated, captured and replayed calls; the graph serves other lengths when it is replayed."""
    say("paged attention: repeats and graphs")
    rng = np.random.default_rng(9)
    t = R.scattered(rng, 6, [9000, 5, 700, 64, 0, 2000], 64, spare=8)
    c = Call(handle, rng, t, [0, 5, 2, 3, 4, 1, -1], 16, 4, 256)
    c.upload()
    c.launch()
    c.check()
    first = c.results()
    for _ in range(3):
        c.launch()
        for a, b in zip(c.results(), first):
            np.testing.assert_array_equal(a, b)
    g = hip.Graph(stream(), c.launch)
    for lens in ([9000, 5, 700, 64, 0, 2000], [1, 0, 650, 33, 0, 1999], [8999, 5, 1, 64, 0, 2000]):
        t.lens[:] = lens
        hip.upload(c.d.lens, t.lens, stream())
        g.launch(stream())
        stream().sync()
        c.check()
        again = c.results()
        g.launch(stream())
        for a, b in zip(c.results(), again):
            np.testing.assert_array_equal(a, b)


def test_two_streams_with_a_handle_each(handle):
    say("paged attention: two streams, a handle each")
    rng = np.random.default_rng(10)
    other = hip.Stream()
    h2 = hip.api().cs1_attention_paged_create()
    t = R.scattered(rng, 4, [6000, 800, 3, 2500], 16)
    a, b = Call(handle, rng, t, range(4), 16, 4, 128), Call(h2, rng, t, range(4), 24, 4, 256)
    a.upload()
    b.upload()
    stream().sync()
    for _ in range(5):
        a.launch()
        b.launch(other.handle)
    other.sync()
    a.check()
    b.check()
    other.destroy()
    hip.api().cs1_attention_paged_destroy(h2)


def test_sizes_one_after_another_with_one_handle(handle):
    """A large call, a small one, a split one: nothing of the call before is left in the handle."""
    say("paged attention: sizes in turn")
    rng = np.random.default_rng(11)
    for lens, hq, hk, dh in (([3000] * 20, 24, 4, 256), ([5], 16, 4, 128), ([20000], 16, 1, 256), ([100, 4000], 32, 1, 128)):
        t = R.scattered(rng, len(lens), lens, 32)
        c = Call(handle, rng, t, range(len(lens)), hq, hk, dh)
        c.upload()
        c.launch()
        c.check()


def test_many_rows(handle):
    say("paged attention: 3000 rows")
    rng = np.random.default_rng(12)
    lens = rng.integers(0, 40, 100)
    t = R.scattered(rng, 100, lens.tolist(), 16)
    c = Call(handle, rng, t, rng.integers(-1, 101, 3000), 4, 2, 128)
    c.upload()
    c.launch()
    c.check()


@pytest.mark.parametrize("lens,hq,hk,dh,page", [
    ([3] * 299 + [7000], 4, 2, 128, 16),                                   # more rows than a block looks at together, one split
    ([900, 0, 31] * 86, 4, 1, 256, 64),                                     # 258 of them, several a block
    ([9000] + [1] * 256 + [5000, 0, 4097], 2, 2, 128, 48),
    ([40] * 513, 16, 16, 128, 16),                                          # thousands of kv heads, several a block
    ([2048, 2048], 48, 1, 256, 256),                                        # three tiles of a kv head
    ([5000, 4096, 4095, 4097], 16, 4, 256, 4096),                           # a page larger than a sequence
    ([70000], 2, 1, 128, 1024), ([1], 16, 4, 128, 65536),
], ids=lambda v: f"{len(v)}x{max(v)}" if isinstance(v, list) else str(v))
def test_many_rows_and_large_pages(handle, lens, hq, hk, dh, page):
    say(f"paged attention {len(lens)} sequences up to {max(lens)}, heads {hq}/{hk} Dh={dh} page={page}")
    rng = np.random.default_rng(len(lens))
    t = R.scattered(rng, len(lens), lens, page, spare=1)
    c = Call(handle, rng, t, rng.permutation(len(lens)), hq, hk, dh)
    c.upload()
    c.launch()
    c.check()


@pytest.mark.parametrize("lens,hq,hk", [
    ([300 + i * 37 % 601 for i in range(130)], 16, 4),              # 13.8 chunks a sequence, few of them cut
    ([300 + i * 37 % 601 for i in range(129)] + [30000], 16, 4),     # one over many blocks' stretches, with a join
    ([384] * 128, 16, 4),                                            # ten chunks each: the first that is halved
    ([384] * 127 + [320], 16, 4),                                    # one less: the last that is not
    ([0, 1500, 129, 128, 4096] * 26, 16, 4),                         # empty ones and whole ones among cut ones
    ([500 + 3 * i for i in range(64)], 32, 8),
    ([450] * 255 + [9000], 32, 1),                                   # two tiles of a kv head
    ([1000] * 9 + [8000], 64, 64),                                   # one q head each
], ids=["130", "129+30000", "at", "below", "mixed", "64x8", "tiles", "64 heads"])
def test_half_the_blocks_with_twice_the_stretch(handle, lens, hq, hk):
    """Heads of 128 and at least twice as many (sequence, kv head, tile) as CUs: half of the blocks do the work, if that is ten
    chunks or more a sequence on average."""
    say(f"paged attention, stretches for half the blocks: {len(lens)} sequences up to {max(lens)}, heads {hq}/{hk}")
    rng = np.random.default_rng(len(lens) + hk)
    t = R.scattered(rng, len(lens), lens, 48)
    c = Call(handle, rng, t, rng.permutation(len(lens)), hq, hk, 128)
    c.upload()
    c.launch()
    c.check()
    first = c.results()
    c.launch()
    for a, b in zip(c.results(), first):
        np.testing.assert_array_equal(a, b)


def test_offsets_past_32_bits(handle):
    """Keys and values behind 4 GiB of a pool."""
    say("paged attention: pools of 5 GiB")
    page, hk, dh, hq = 64, 8, 128, 16
    rng = np.random.default_rng(14)
    npages = (5 << 30) // (page * hk * dh * 2)
    t = R.Table(2, 3, npages, page)
    t.table[0], t.table[1, 0], t.lens[:] = [npages - 1, 3, npages - 2], npages - 5, [150, 9]
    small = R.Table(2, 3, 6, page)  # the same pages, numbered from 0
    order = [npages - 1, 3, npages - 2, npages - 5]
    small.table[0], small.table[1, 0], small.lens[:] = [0, 1, 2], 3, [150, 9]
    c = Call(handle, rng, small, [1, 0], hq, hk, dh)
    want, wl, tol, ltol = R.attention(small, c.seqs, c.q, c.kp, c.vp, c.gate, hk, dh ** -0.5)
    c.upload()
    c.t, c.d = t, DeviceTable(t)
    size = page * hk * dh * 2
    pools = [empty(npages * size), empty(npages * size)]
    for pool, arr in zip(pools, (c.kp, c.vp)):
        for i, p in enumerate(order):
            hip.upload(pool, arr[i], stream(), offset=p * size)
    c.bufs[1:3] = pools
    c.launch()
    out, l = c.results()
    R.close(R.f64(out), want, tol, "out")
    R.close(l.astype(np.float64), wl, ltol, "lse")


def test_refusals_with_a_handle(handle):
    say("paged attention: refusals")
    rng = np.random.default_rng(13)
    t = R.scattered(rng, 1, [5], 16)
    c = Call(handle, rng, t, [0], 4, 2, 128)
    c.upload()
    api, st = hip.api(), stream().handle
    q, kp, vp, seqs = (b.at(0) for b in c.bufs)
    out = c.out.at(0)

    def call(q=q, kp=kp, vp=vp, gate=None, out=out, B=1, hq=4, hk=2, dh=128):
        return api.cs1_attention_paged(handle, q, kp, vp, c.d.ref, seqs, gate, out, None, B, hq, hk, dh, 1.0, st)

    assert call(dh=64) == call(hq=5) == call(hk=0) == call(B=-1) == call(hq=0) == hip.HIP_ERROR_INVALID_VALUE
    assert call(q=None) == call(kp=None) == call(vp=None) == call(out=None) == hip.HIP_ERROR_INVALID_VALUE
    assert call(q=q + 8) == call(kp=kp + 2) == call(vp=vp + 4) == call(out=out + 8) == call(gate=q + 2) == hip.HIP_ERROR_INVALID_VALUE
    assert call(B=1 << 23) == hip.HIP_ERROR_INVALID_VALUE
    assert call(B=0, q=None) == 0
    big = hip.PageTable(c.d.table.at(0), c.d.lens.at(0), c.d.refs.at(0), 1, 1, 1 << 27, 16)  # 2^31 tokens in the pool
    c.d.ref = ctypes.byref(big)
    assert call() == hip.HIP_ERROR_INVALID_VALUE
    long = hip.PageTable(c.d.table.at(0), c.d.lens.at(0), c.d.refs.at(0), 1, 1 << 26, 4, 16)  # 2^25 units a row
    c.d.ref = ctypes.byref(long)
    assert call(B=64) == hip.HIP_ERROR_INVALID_VALUE
    (out_before, _) = c.results()
    assert (out_before == 0x7fc1).all()
