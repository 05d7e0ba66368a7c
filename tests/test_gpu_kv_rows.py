"""cs1_kv_extend, cs1_kv_rows and cs1_kv_trim against the bookkeeping step by step."""
import numpy as np
import pytest

import decode_ref as R
import rows_ref as W
from decode_ref import DeviceTable, Table, ints
from gpu_helpers import dev, get, say, stream
from qwen3_5_native import hip

pytestmark = pytest.mark.gpu


class Cache:
    def __init__(self, t):
        self.t, self.d, self.status = t, DeviceTable(t), ints([77])

    def answer(self):
        return int(get(self.status, np.int32, 1)[0])

    def extend(self, seqs, cu, null=False):
        say(f"  extend {len(seqs)}")
        b, c = ints(seqs), ints(cu)
        hip.check(hip.api().cs1_kv_extend(self.d.ref, None if null else b.at(0), c.at(0), len(seqs), self.status.at(0),
                                          stream().handle), "extend")
        want = W.extend(self.t, seqs, cu)
        assert self.answer() == want
        self.d.check()
        return want

    def rows(self, seqs, cu, rows, null=False):
        say(f"  rows {rows} of {len(seqs)}")
        b, c = ints(seqs), ints(cu)
        out = dev(np.full(2 * (rows + 1), 99, np.int32))
        hip.check(hip.api().cs1_kv_rows(self.d.ref, None if null else b.at(0), c.at(0), len(seqs), rows, out.at(0),
                                        out.at(4 * (rows + 1)), stream().handle), "rows")
        got = get(out, np.int32, 2 * (rows + 1)).reshape(2, -1)
        assert (got[:, rows] == 99).all(), "written behind the last row"
        pos, slot = W.rows_of(self.t, seqs, cu, rows)
        np.testing.assert_array_equal(got[0, :rows], pos)
        np.testing.assert_array_equal(got[1, :rows], slot)
        return pos, slot

    def trim(self, seqs, drop, null=False):
        say(f"  trim {len(seqs)}")
        b, c = ints(seqs), ints(drop)
        hip.check(hip.api().cs1_kv_trim(self.d.ref, None if null else b.at(0), c.at(0), len(seqs), self.status.at(0),
                                        stream().handle), "trim")
        want = W.trim(self.t, seqs, drop)
        assert self.answer() == want
        self.d.check()
        return want


@pytest.mark.parametrize("seed", range(4))
def test_steps_of_a_server(seed):
    """Ragged growth with padding and repeats, rows mapped, some tokens taken back, sequences freed in between."""
    say(f"kv rows: steps, seed {seed}")
    rng = np.random.default_rng(seed)
    nseq, page = 12, [16, 48, 64, 16][seed]
    c = Cache(Table(nseq, 40, 90, page))
    for step in range(6):
        seqs = rng.integers(-2, nseq + 2, rng.integers(1, 12))
        new = rng.choice([0, 1, 2, 5, 17, 70], len(seqs))
        cu = np.concatenate([[0], np.cumsum(new)])
        if c.extend(seqs, cu) == 0:
            c.rows(seqs, cu, int(cu[-1]) + int(rng.integers(0, 4)))
            c.trim(seqs, rng.integers(-1, 30, len(seqs)))
        if step == 3:
            b = ints([3, 5])
            hip.check(hip.api().cs1_kv_free(c.d.ref, b.at(0), 2, stream().handle), "free")
            c.t.free([3, 5])
            c.d.check()


def test_no_list_and_nothing():
    say("kv rows: no list, no entries")
    c = Cache(Table(5, 6, 20, 16))
    cu = [0, 3, 3, 40, 41, 58, 60]
    c.extend(range(6), cu, null=True)  # entry 5 is past the table: padding
    c.rows(range(6), cu, 64, null=True)
    c.trim(range(6), [0, 5, 36, 1, 100, 3], null=True)
    one = ints([7])
    out = dev(np.full(6, 99, np.int32))
    api, st = hip.api(), stream().handle
    hip.check(api.cs1_kv_extend(c.d.ref, None, None, 0, c.status.at(0), st), "extend")
    assert c.answer() == 0
    hip.check(api.cs1_kv_trim(c.d.ref, None, None, 0, one.at(0), st), "trim")
    assert get(one, np.int32, 1)[0] == 0
    hip.check(api.cs1_kv_rows(c.d.ref, None, None, 0, 3, out.at(0), out.at(12), st), "rows")
    assert (get(out, np.int32, 6) == -1).all()
    c.d.check()


def test_too_little_room_changes_nothing():
    say("kv rows: no room")
    c = Cache(Table(4, 4, 6, 16))
    assert c.extend([0, 1], [0, 33, 50]) == 0
    assert c.extend([2, 0], [0, 20, 21]) > 0   # pages are missing
    assert c.extend([3, 1], [0, 1, 60]) == -1  # more than the table's row
    assert c.extend([0], [0, 2 ** 31 - 1]) == -1
    assert c.extend([2, 1], [0, 7, 8]) == 0


@pytest.mark.parametrize("n", [1025, 4000, 8192])
def test_long_lists(n):
    """More entries than a block has threads, single tokens and short drafts, half of them padding or repeats."""
    say(f"kv rows: {n} entries")
    rng = np.random.default_rng(n)
    nseq = 8192 if n == 8192 else 3000
    c = Cache(Table(nseq, 3, 20000, 16))
    seqs = rng.permutation(n).astype(np.int64) if n == 8192 else rng.integers(-3, nseq + 3, n)
    cu = np.concatenate([[0], np.cumsum(rng.integers(0, 4, n))])
    c.extend(seqs, cu)
    c.rows(seqs, cu, int(cu[-1]) + 5)
    c.extend(seqs, cu)
    c.trim(seqs, rng.integers(0, 6, n))


def test_offsets_that_fall_and_rows_that_are_cut():
    """Such offsets are a program's mistake: their rows are no one's, and nothing is read or written out of range."""
    say("kv rows: odd offsets")
    c = Cache(Table(6, 8, 40, 16))
    c.extend([0, 1, 2], [0, 30, 50, 53])
    c.rows([0, 1, 2], [0, 30, 50, 53], 40)  # fewer rows than offsets name
    c.extend([3, 4], [0, 9, 4])             # entry 4 has none
    b, cu, out = ints([0, 1, 2]), ints([0, 5, 2, 9]), dev(np.zeros(20, np.int32))
    hip.check(hip.api().cs1_kv_rows(c.d.ref, b.at(0), cu.at(0), 3, 10, out.at(0), out.at(40), stream().handle), "rows")
    got = get(out, np.int32, 20).reshape(2, 10)
    assert (got[:, 9] == -1).all() and (got[0] < 60).all() and (got[1] < 640).all() and (got >= -1).all()


def test_bad_pages_and_lengths():
    say("kv rows: pages out of range, lengths past the table")
    t = R.scattered(np.random.default_rng(1), 5, [40, 20, 33, 5, 16], 16)
    t.table[0, 1], t.table[1, 1], t.table[2, 0] = t.npages, -1, 2 ** 31 - 1
    c = Cache(t)
    c.rows(range(5), [0, 40, 60, 93, 98, 120], 125)  # sequence 4 has fewer tokens than rows
    t.lens[3] = 16 * t.max_pages + 9
    c = Cache(t)
    c.rows([3], [0, 16], 16)


def test_trim_beside_forks():
    """A page that others hold is not cut, whatever the order and also where the other one lets go of it in the same call."""
    say("kv rows: trim of forks")
    for order in ([0, 1, 2], [2, 1, 0], [1, 0, 2]):
        t = Table(4, 8, 30, 16)
        c = Cache(t)
        c.extend([0], [0, 70])
        src, dst = ints([0, 0]), ints([1, 2])
        ws = dev(np.zeros(400, np.int32))
        hip.check(hip.api().cs1_kv_fork(c.d.ref, src.at(0), dst.at(0), 2, None, 0, 16, ws.at(0), c.status.at(0), stream().handle),
                  "fork")
        t.fork([0, 0], [1, 2], [])
        c.d.check()
        drop = {0: 10, 1: 70, 2: 5}  # into a shared page, all of it, within its own page
        assert c.trim(order, [drop[s] for s in order]) == 1
        assert c.trim([0, 2], [6, 1]) == 0  # to its own page's start: nothing is cut
        assert c.trim([0], [16]) == 0       # to a page's end
        assert c.trim([0], [3]) == 1        # into a page that 2 holds


def test_many_pages_are_released():
    say("kv rows: thousands of pages")
    c = Cache(Table(3, 3000, 7000, 16))
    c.extend([2, 0], [0, 47000, 90001])
    assert c.trim([0, 1, 2], [43000, 4, 46999]) == 0
    c.rows([2, 0], [0, 1, 2], 2)


def test_replayed_step_follows_its_lists():
    say("kv rows: a captured step")
    rng = np.random.default_rng(9)
    c, api, s = Cache(Table(8, 20, 120, 16)), hip.api(), stream()
    n, rows = 5, 90
    seqs, cu, drop = ints([-1] * n), ints([0] * (n + 1)), ints([0] * n)
    out, st2 = dev(np.zeros(2 * rows, np.int32)), ints([5])

    def record():
        hip.check(api.cs1_kv_extend(c.d.ref, seqs.at(0), cu.at(0), n, c.status.at(0), s.handle), "extend")
        hip.check(api.cs1_kv_rows(c.d.ref, seqs.at(0), cu.at(0), n, rows, out.at(0), out.at(4 * rows), s.handle), "rows")
        hip.check(api.cs1_kv_trim(c.d.ref, seqs.at(0), drop.at(0), n, st2.at(0), s.handle), "trim")

    graph = hip.Graph(s, record)
    for step in range(5):
        ids, new = rng.permutation(9)[:n] - 1, rng.integers(0, 18, n)
        off, back = np.concatenate([[0], np.cumsum(new)]), rng.integers(0, 9, n)
        for buf, v in ((seqs, ids), (cu, off), (drop, back)):
            hip.upload(buf, v.astype(np.int32), s)
        graph.launch(s)
        assert c.answer() == W.extend(c.t, ids, off) == 0
        pos, slot = W.rows_of(c.t, ids, off, rows)
        got = get(out, np.int32, 2 * rows).reshape(2, rows)
        np.testing.assert_array_equal(got[0], pos)
        np.testing.assert_array_equal(got[1], slot)
        assert get(st2, np.int32, 1)[0] == W.trim(c.t, ids, back)
        c.d.check()
