"""cs1_attention_paged_varlen against attention in float64 (rows_ref.attention), within bounds that follow from
float32's sums, probabilities rounded to bfloat16 and one bfloat16 output."""
import numpy as np
import pytest

import decode_ref as R
import rows_ref as W
from decode_ref import DeviceTable, ints
from gpu_helpers import dev, get, get_bf16, say, stream
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
    """new[i] rows for list entry i, of whose sequence t holds them already; `pad` rows are no one's."""

    def __init__(self, handle, rng, t, seqs, new, hq, hk, dh, gate=True, lse=True, std=1.0, pad=0, max_new=None):
        self.handle, self.t, self.seqs, self.hq, self.hk, self.dh = handle, t, np.asarray(seqs, np.int32), hq, hk, dh
        self.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = B = int(self.cu[-1]) + pad
        self.max_new = int(max(new, default=0)) if max_new is None else max_new
        self.q, self.gate = R.bf16(rng, B, hq, dh, std=std), R.bf16(rng, B, hq, dh) if gate else None
        self.kp, self.vp = R.bf16(rng, t.npages, t.page, hk, dh, std=std), R.bf16(rng, t.npages, t.page, hk, dh)
        self.lse, self.scale = lse, dh ** -0.5

    def upload(self):
        self.d = DeviceTable(self.t)
        self.bufs = [dev(x) for x in (self.q, self.kp, self.vp, self.seqs, self.cu)]
        self.g = dev(self.gate) if self.gate is not None else None
        self.clear()

    def clear(self):
        self.out = dev(np.full(self.rows * self.hq * self.dh + 8, 0x7fc1, np.uint16))
        self.l = dev(np.full(self.rows * self.hq + 1, 5.0, np.float32))

    def launch(self, st=None, null=False):
        q, kp, vp, seqs, cu = self.bufs
        hip.check(hip.api().cs1_attention_paged_varlen(
            self.handle, q.at(0), kp.at(0), vp.at(0), self.d.ref, None if null else seqs.at(0), cu.at(0), len(self.seqs), self.max_new,
            self.g.at(0) if self.g else None, self.out.at(0), self.l.at(0) if self.lse else None, self.rows, self.hq, self.hk, self.dh,
            self.scale, st or stream().handle), "attention_paged_varlen")

    def results(self):
        n = self.rows * self.hq * self.dh
        out, l = get_bf16(self.out, n + 8), get(self.l, np.float32, self.rows * self.hq + 1)
        assert (out[n:] == 0x7fc1).all() and l[-1] == 5.0, "written behind the last row"
        return out[:n].reshape(self.rows, self.hq, self.dh), l[:-1].reshape(self.hq, self.rows)

    def check(self, seqs=None):
        out, l = self.results()
        want, wl, tol, ltol, ours = W.attention(self.t, self.seqs if seqs is None else seqs, self.cu, self.rows, self.max_new, self.q,
                                                self.kp, self.vp, self.gate, self.hk, self.scale)
        assert (out[~ours] == 0x7fc1).all(), "rows of no one are written"
        R.close(R.f64(out[ours]), want[ours], tol[ours], "out")
        if self.lse:
            assert (l[:, ~ours] == 5.0).all()
            R.close(l[:, ours].astype(np.float64), wl[:, ours], ltol[:, ours], "lse")
        return out, l


def run(c, **kw):
    c.upload()
    c.launch(**kw)
    return c.check()


HEADS = [(16, 4, 128), (16, 4, 256), (24, 4, 256), (4, 4, 128), (16, 1, 256), (6, 2, 128), (32, 1, 128), (17, 1, 256), (40, 2, 128), (1, 1, 256),
         (128, 1, 128), (10, 2, 256)]


@pytest.mark.parametrize("hq,hk,dh", HEADS)
@pytest.mark.parametrize("page", [16, 48, 64])
def test_head_layouts(handle, hq, hk, dh, page):
    say(f"attention chunk heads {hq}/{hk} Dh={dh} page={page}")
    rng = np.random.default_rng(hq * hk + page)
    lens = [1, 0, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 130, 257, 300]
    new = [min(n, int(k)) for n, k in zip(lens, rng.choice([1, 2, 3, 7, 40, 300], len(lens)))]
    t = R.scattered(rng, len(lens) + 2, lens, page)
    order = rng.permutation(len(lens))
    run(Call(handle, rng, t, order, np.array(new)[order], hq, hk, dh, gate=page != 64, lse=page != 16, pad=3))


@pytest.mark.parametrize("lens,new", [([5000], [4]), ([5000], [333]), ([1269], [333]), ([700], [700]), ([1, 4000], [1, 37]), ([700] * 3, [1, 250, 7]),
                                      ([8191, 3, 0, 900], [2, 3, 0, 900]), ([127] * 70, [1] * 70), ([12000, 1, 1, 1], [16, 1, 1, 1]),
                                      (list(range(1, 400, 7)), [1 + i % 5 if i else 1 for i in range(58)]), ([20000], [1]), ([2049], [2049]),
                                      ([64] * 9, [64] * 9), ([300] * 20, [4] * 20), ([3000] * 6, [1, 1, 100, 1, 1, 500])],
                         ids=lambda l: f"{len(l)}x{max(l)}")
@pytest.mark.parametrize("hq,hk,dh,page", [(16, 4, 128, 16), (6, 1, 256, 208), (20, 1, 256, 32), (8, 4, 128, 48)])
def test_lengths(handle, lens, new, hq, hk, dh, page):
    """Sequences that fill the chip alone and together, cut and whole."""
    say(f"attention chunk {len(lens)} sequences up to {max(lens)}, {sum(new)} rows, heads {hq}/{hk} Dh={dh} page={page}")
    rng = np.random.default_rng(sum(lens) + dh)
    t = R.scattered(rng, len(lens), lens, page)
    run(Call(handle, rng, t, np.arange(len(lens)), new, hq, hk, dh, gate=hq != 6))


def test_padding_repeats_and_no_list(handle):
    say("attention chunk: padding entries, a sequence twice, no list, rows before position 0")
    rng = np.random.default_rng(3)
    t = R.scattered(rng, 5, [70, 0, 33, 500, 16], 16)
    new = [3, 2, 70, 9, 70, 4, 3, 1, 20, 100]
    c = Call(handle, rng, t, [3, -1, 0, 5, 0, 2 ** 31 - 1, 1, -2 ** 31, 4, 3], new, 8, 2, 128, pad=5)
    out, l = run(c)
    for i in (1, 3, 5, 6, 7):
        rows = slice(c.cu[i], c.cu[i + 1])
        assert (out[rows] == 0).all() and (l[:, rows] == -np.inf).all()
    assert (out[c.cu[8]:c.cu[8] + 4] == 0).all()  # sequence 4 has 16 tokens and 20 rows
    c.clear()
    c.launch(null=True)  # entry i is sequence i; entries from nseq on are padding
    c.check(seqs=list(range(5)) + [-1] * 5)


def test_most_rows_and_no_rows(handle):
    say("attention chunk: rows behind max_new, entries without rows")
    rng = np.random.default_rng(4)
    t = R.scattered(rng, 4, [90, 40, 300, 7], 16)
    for dh in (128, 256):
        run(Call(handle, rng, t, [2, 0, 3, 1], [100, 0, 5, 40], 8, 4, dh, max_new=33, pad=2))
        run(Call(handle, rng, t, [2, 0], [1, 2], 8, 4, dh, max_new=1000))
    c = Call(handle, rng, t, [2, 0], [0, 0], 8, 4, 128, max_new=4, pad=6)
    run(c)


@pytest.mark.parametrize("dh", [128, 256])
def test_what_is_not_held_is_not_read(handle, dh):
    """NaN and infinities in every slot that no token of the sequence has, and in pages of others."""
    say(f"attention chunk: NaN around, Dh={dh}")
    rng = np.random.default_rng(4)
    lens = [1, 17, 40, 129, 1000, 0]
    t = R.scattered(rng, 6, lens, 48)
    c = Call(handle, rng, t, range(6), [1, 5, 40, 100, 3, 0], 16, 4, dh)
    held = np.zeros((t.npages, t.page), bool)
    for s, n in enumerate(lens):
        for j in range(n):
            held[t.table[s, j // 48], j % 48] = True
    for pool, bits in ((c.kp, 0x7fc0), (c.vp, 0x7f80)):
        pool[~held] = bits
    c.vp[~held, :, ::2] = 0xffc0
    out, _ = run(c)
    assert np.isfinite(R.f64(out)).all()


@pytest.mark.parametrize("dh", [128, 256])
@pytest.mark.parametrize("kind", ["nan", "inf"])
def test_later_rows_are_not_seen(handle, dh, kind):
    """NaN and infinities in the keys and values of new tokens: rows before them do not change."""
    say(f"attention chunk: {kind} in later rows, Dh={dh}")
    rng = np.random.default_rng(5)
    L = 150
    t = R.scattered(rng, 2, [400, 250], 16)
    c = Call(handle, rng, t, [0, 1], [L, 250], 8, 2, dh, gate=False)
    c.upload()
    c.launch()
    clean, cl = c.results()
    at = lambda s, p: (t.table[s, p // 16], p % 16)  # noqa: E731
    spots = [(0, 250 + 40, 0, 3), (0, 250 + 41, 1, 100), (1, 0, 1, 7), (1, 77, 0, 0), (1, 249, 0, dh - 1)]
    for s, p, h, d in spots:
        c.vp[at(s, p)][h, d] = {"nan": 0x7fc0, "inf": 0xff80 if d == 100 else 0x7f80}[kind]
    c.upload()
    c.launch()
    out, l = c.results()
    rep = 8 // 2
    hit = np.zeros(out.shape, bool)
    for s, p, h, d in spots:
        first = c.cu[s] + p - (int(t.lens[s]) - (c.cu[s + 1] - c.cu[s]))
        hit[first:c.cu[s + 1], h * rep:(h + 1) * rep, d] = True
    np.testing.assert_array_equal(out[~hit], clean[~hit])
    np.testing.assert_array_equal(l, cl)
    x = R.f64(out)[hit]
    assert np.isnan(x).all() if kind == "nan" else np.isinf(x).all()
    if kind == "inf":
        x = R.f64(out)
        assert (x[c.cu[0] + 41:c.cu[1], rep:, 100] == -np.inf).all() and (x[c.cu[1]:c.cu[2], rep:, 7] == np.inf).all()
    if kind == "nan":  # keys
        c.kp[at(0, 300)][1, 5] = 0x7fc0
        c.upload()
        c.launch()
        again = R.f64(c.results()[0])
        assert np.isnan(again[c.cu[0] + 50:c.cu[1], rep:]).all()
        np.testing.assert_array_equal(c.results()[0][:c.cu[0] + 50], out[:c.cu[0] + 50])


@pytest.mark.parametrize("dh", [128, 256])
def test_infinities_of_both_signs(handle, dh):
    say(f"attention chunk: infinities of both signs, Dh={dh}")
    rng = np.random.default_rng(6)
    t = R.scattered(rng, 1, [90], 16)
    c = Call(handle, rng, t, [0], [90], 4, 4, dh, gate=False)
    at = lambda p: (t.table[0, p // 16], p % 16)  # noqa: E731
    c.vp[at(20)][2, 9], c.vp[at(50)][2, 9] = 0x7f80, 0xff80
    c.upload()
    c.launch()
    x = R.f64(c.results()[0])
    assert np.isfinite(x[:20]).all() and (x[20:50, 2, 9] == np.inf).all() and np.isnan(x[50:, 2, 9]).all()
    x[20:, 2, 9] = 0
    assert np.isfinite(x).all()


def test_values_of_the_largest_size(handle):
    say("attention chunk: the largest values without weight")
    rng = np.random.default_rng(15)
    for dh in (128, 256):
        t = R.scattered(rng, 2, [40, 700], 16)
        c = Call(handle, rng, t, range(2), [20, 65], 8, 4, dh)
        c.q[:], c.kp[:] = 0, 0
        c.q[..., 0] = R.O.f32_to_bf16(np.full(c.q[..., 0].size, 128.0, np.float32)).reshape(c.q[..., 0].shape)
        low = R.O.f32_to_bf16(np.array([-64.0], np.float32))[0]  # scores of 0 but for these: -512 and less
        for s, j in ((0, 5), (0, 39), (1, 0), (1, 321), (1, 699)):
            at = t.table[s, j // 16], j % 16
            c.kp[at][:, 0] = low
            c.vp[at] = np.where(rng.random((4, dh)) < 0.5, 0x7f7f, 0xff7f)
        run(c)


@pytest.mark.parametrize("std", [8.0, 40.0])
@pytest.mark.parametrize("dh", [128, 256])
def test_large_scores(handle, std, dh):
    """Scores of hundreds to tens of thousands: the maximum moves by far more than a float's exponent holds."""
    say(f"attention chunk: large scores, std {std}")
    rng = np.random.default_rng(6)
    t = R.scattered(rng, 4, [3000, 100, 1, 650], 32)
    run(Call(handle, rng, t, range(4), [70, 100, 1, 5], 16, 4, dh, std=std))


def test_bad_page_numbers_are_masked(handle):
    say("attention chunk: page numbers out of range")
    rng = np.random.default_rng(7)
    for dh in (128, 256):
        t = R.scattered(rng, 4, [100, 700, 30, 64], 16)
        t.table[0, 2], t.table[1, 0], t.table[1, 43], t.table[2] = t.npages, -1, 2 ** 31 - 1, -2 ** 31
        run(Call(handle, rng, t, range(4), [50, 60, 30, 3], 16, 4, dh))


def test_more_tokens_than_the_table_has_room_for(handle):
    say("attention chunk: a length past the table's row")
    rng = np.random.default_rng(8)
    t = R.scattered(rng, 2, [96, 20], 16, max_pages=6)
    c = Call(handle, rng, t, [0, 1], [10, 20], 8, 2, 128)
    c.upload()
    hip.upload(c.d.lens, np.array([2 ** 31 - 1, 20], np.int32), stream())
    c.launch()
    c.check()


def test_rows_are_cut_off_and_offsets_fall(handle):
    """A program's mistakes: nothing behind the buffers is read or written."""
    say("attention chunk: odd offsets")
    rng = np.random.default_rng(9)
    t = R.scattered(rng, 3, [100, 50, 60], 16)
    c = Call(handle, rng, t, [0, 1, 2], [20, 20, 20], 8, 2, 128)
    c.upload()
    for cu in ([0, 20, 40, 2 ** 31 - 1], [0, 20, 10, 60], [-5, 20, 40, 60], [100, 200, 300, 400], [2 ** 31 - 1, -2 ** 31, 0, 7]):
        hip.upload(c.bufs[4], np.array(cu, np.int32), stream())
        c.launch()
        c.results()


def test_wide_batches(handle):
    """More entries than a window of the search, and than a wave has lanes for windows."""
    rng = np.random.default_rng(10)
    for n, most in ((65, 40), (700, 9), (4100, 2), (8192, 2)):
        say(f"attention chunk: {n} entries")
        lens = rng.integers(0, 40, n)
        new = np.minimum(lens, rng.integers(0, most + 1, n))
        t = R.scattered(rng, n, lens.tolist(), 16)
        run(Call(handle, rng, t, rng.permutation(n) if n == 8192 else np.arange(n), new, 2, 1, 128, pad=1, lse=n < 100))


def test_pool_past_4_gib(handle):
    say("attention chunk: pages past 4 GiB")
    rng = np.random.default_rng(11)
    hk, dh, page = 16, 256, 256
    t = R.Table(1, 4, 2100, page)  # 2.2 GB of 2 MiB pages a pool, the last past 4 GiB
    t.table[0, :3], t.lens[0] = [2099, 0, 2049], 700
    t.refs[t.table[0, :3]] = 1
    small = R.Table(1, 4, 3, page)
    small.table[0, :3], small.lens[0] = [0, 1, 2], 700
    c = Call(handle, rng, small, [0], [90], 16, hk, dh)
    c.upload()
    c.launch()
    want, _ = c.results()
    size = page * hk * dh * 2
    pools = [hip.DeviceBuffer(t.npages * size) for _ in range(2)]
    for pool, host in zip(pools, (c.kp, c.vp)):
        for i, p in enumerate(t.table[0, :3]):
            hip.upload(pool, host[i], stream(), offset=int(p) * size)
    c.d, c.bufs[1], c.bufs[2] = DeviceTable(t), pools[0], pools[1]
    c.clear()
    c.launch()
    np.testing.assert_array_equal(c.results()[0], want)


def test_one_graph_serves_other_batches(handle):
    say("attention chunk: replays with other lists and lengths")
    rng = np.random.default_rng(12)
    lens = [400, 33, 0, 1300, 90, 17]
    t = R.scattered(rng, 6, lens, 16)
    n, rows = 4, 300
    c = Call(handle, rng, t, [0] * n, [75] * n, 8, 2, 128, max_new=256)
    c.upload()
    graph = hip.Graph(stream(), c.launch)
    for ids, new in (([0, 3, 1, 4], [30, 200, 33, 1]), ([5, 5, -1, 2], [17, 3, 50, 2]), ([3, 0, 4, 1], [1, 1, 1, 1]), ([3, 3, 3, 3], [256, 0, 4, 40])):
        c.seqs, c.cu = np.array(ids, np.int32), np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        hip.upload(c.bufs[3], c.seqs, stream())
        hip.upload(c.bufs[4], c.cu, stream())
        hip.upload(c.out, np.full(rows * 8 * 128 + 8, 0x7fc1, np.uint16), stream())
        hip.upload(c.l, np.full(rows * 8 + 1, 5.0, np.float32), stream())
        graph.launch(stream())
        first = [x.copy() for x in c.check()]
        c.launch()  # and the same bits without it
        for a, b in zip(first, c.results()):
            np.testing.assert_array_equal(a, b)


def test_single_tokens_as_the_single_token_call(handle):
    say("attention chunk: one token each, beside cs1_attention_paged")
    rng = np.random.default_rng(13)
    lens = [700, 1, 64, 3000, 129]
    t = R.scattered(rng, 5, lens, 64)
    for dh in (128, 256):
        c = Call(handle, rng, t, range(5), [1] * 5, 16, 4, dh)
        out, _ = run(c)
        one = dev(np.zeros(5 * 16 * dh, np.uint16))
        q, kp, vp, seqs, _ = c.bufs
        hip.check(hip.api().cs1_attention_paged(handle, q.at(0), kp.at(0), vp.at(0), c.d.ref, seqs.at(0), c.g.at(0), one.at(0), None, 5, 16, 4,
                                                dh, c.scale, stream().handle), "attention_paged")
        a, b = R.f64(out), R.f64(get_bf16(one, 5 * 16 * dh)).reshape(out.shape)
        assert np.abs(a - b).max() <= 4 * R.E16 * np.abs(b).max()


def test_two_handles_on_two_streams():
    say("attention chunk: two calls at once")
    rng = np.random.default_rng(14)
    api, other = hip.api(), hip.Stream()
    calls = []
    for i, st in enumerate((stream(), other)):
        h = api.cs1_attention_paged_create()
        t = R.scattered(rng, 3, [2500, 300, 40], 16)
        calls.append((Call(h, rng, t, [0, 1, 2], [200 + i, 30, 40], 16, 4, 256), st, h))
        calls[-1][0].upload()
    stream().sync()
    for _ in range(3):
        for c, st, _h in calls:
            c.launch(st.handle)
    for c, st, h in calls:
        st.sync()
        c.check()
        api.cs1_attention_paged_destroy(h)
    other.destroy()
