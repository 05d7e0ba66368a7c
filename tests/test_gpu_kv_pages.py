"""The page operations (cs1_kv_*) against the bookkeeping step by step (decode_ref.Table): table, lengths,
counts and every byte of the pools are equal after each call."""
import numpy as np
import pytest

import decode_ref as R
from decode_ref import DeviceTable, Table, ints, pointers, pool_buffers, read_pool
from gpu_helpers import dev, empty, get, say, stream
from qwen3_5_native import hip

pytestmark = pytest.mark.gpu


class Cache:
    """A device table with pools, and the same on the host."""

    def __init__(self, t, rng, npools, width):
        self.t, self.d, self.width = t, DeviceTable(t), width
        self.pools = [R.bf16(rng, t.npages, t.page, width) for _ in range(npools)]
        self.bufs = pool_buffers(self.pools)
        self.ptrs = pointers(self.bufs)
        self.status = ints([77])
        self.ws = empty(hip.api().cs1_kv_workspace_bytes(t.npages, 8192))

    def check(self, what):
        self.d.check()
        for i, (b, p) in enumerate(zip(self.bufs, self.pools)):
            np.testing.assert_array_equal(read_pool(b, p), p, err_msg=f"{what}: pool {i}")

    def status_is(self, want):
        assert int(get(self.status, np.int32, 1)[0]) == want

    def reserve(self, seqs, cu=None, null=False):
        say(f"  reserve {len(seqs)} cu={cu is not None}")
        want = self.t.reserve(seqs, cu)
        b = ints(seqs) if len(seqs) else None
        hip.check(hip.api().cs1_kv_reserve(self.d.ref, None if null or b is None else b.at(0),
                                           cu.ctypes.data if cu is not None else None, len(seqs), self.status.at(0),
                                           stream().handle), "reserve")
        self.status_is(want)
        self.check("reserve")
        return want

    def write(self, seqs, cu, rng, layer=0, pad=(0, 8)):
        rows = len(seqs) if cu is None else int(cu[-1])
        say(f"  write {rows} rows of {len(seqs)} sequences")
        k, v = R.bf16(rng, rows, self.width + pad[0]), R.bf16(rng, rows, self.width + pad[1])
        kp, vp = 2 * layer, 2 * layer + 1
        self.t.write(seqs, cu, k[:, :self.width], v[:, :self.width], self.pools[kp], self.pools[vp])
        b, kb, vb = ints(seqs), dev(k), dev(v)
        hip.check(hip.api().cs1_kv_write(self.d.ref, b.at(0), cu.ctypes.data if cu is not None else None, len(seqs),
                                         kb.at(0), self.width + pad[0], vb.at(0), self.width + pad[1], self.bufs[kp].at(0),
                                         self.bufs[vp].at(0), self.width // 8, 8, stream().handle), "write")
        self.check("write")

    def fork(self, src, dst):
        say(f"  fork {len(src)}")
        want = self.t.fork(src, dst, self.pools)
        a, b = ints(src), ints(dst)
        hip.check(hip.api().cs1_kv_fork(self.d.ref, a.at(0), b.at(0), len(src), self.ptrs, len(self.bufs),
                                        2 * self.width, self.ws.at(0), self.status.at(0), stream().handle), "fork")
        self.status_is(want)
        self.check("fork")
        return want

    def free(self, seqs):
        say(f"  free {len(seqs)}")
        self.t.free(seqs)
        b = ints(seqs)
        hip.check(hip.api().cs1_kv_free(self.d.ref, b.at(0), len(seqs), stream().handle), "free")
        self.check("free")

    def compact(self):
        say("  compact")
        want = self.t.compact(self.pools)
        hip.check(hip.api().cs1_kv_compact(self.d.ref, self.ptrs, len(self.bufs), 2 * self.width, self.ws.at(0),
                                           self.status.at(0), stream().handle), "compact")
        self.status_is(want)
        self.check("compact")


@pytest.mark.parametrize("nseq,page,npages,max_pages,npools,width", [
    (1, 16, 5, 4, 2, 8), (6, 16, 40, 9, 2, 512), (13, 48, 61, 7, 4, 72), (40, 64, 150, 5, 6, 128), (9, 208, 30, 3, 2, 1024)])
def test_a_server_at_work(nseq, page, npages, max_pages, npools, width):
    """Random calls: ragged prompts and single tokens, forks, ends, compactions; pools that run out."""
    say(f"server nseq={nseq} page={page} npages={npages}")
    rng = np.random.default_rng(nseq * page)
    c = Cache(Table(nseq, max_pages, npages, page), rng, npools, width)
    seen = set()
    for step in range(30):
        kind = rng.choice(["prompt", "token", "token", "fork", "free", "compact"])
        pick = rng.permutation(nseq)[:rng.integers(1, nseq + 1)]
        # padding and a sequence named twice among them
        pick = np.concatenate([pick, [-1, nseq, pick[0]]])[rng.permutation(len(pick) + 3)]
        if kind == "prompt" and len(pick) <= 64:
            lens = rng.integers(0, 2 * page + 3, len(pick))
            cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
            got = c.reserve(pick, cu)
            if got == 0:
                c.write(pick, cu, rng, layer=int(rng.integers(npools // 2)))
            seen.add(("prompt", np.sign(got)))
        elif kind == "token":
            got = c.reserve(pick)
            if got == 0:
                c.write(pick, None, rng, layer=int(rng.integers(npools // 2)), pad=(16, 0))
            seen.add(("token", np.sign(got)))
        elif kind == "fork":
            src, dst = rng.integers(-1, nseq + 1, len(pick)), pick
            got = c.fork(src, dst)
            seen.add(("fork", np.sign(got)))
        elif kind == "free":
            c.free(pick[:max(1, len(pick) // 2)])
        else:
            c.compact()
    say(f"  seen {sorted((k, int(v)) for k, v in seen)}")


def test_what_reserve_says_when_room_is_short():
    say("reserve: short of pages, of a table's width, empty lists, null list")
    rng = np.random.default_rng(0)
    c = Cache(Table(4, 3, 6, 16), rng, 2, 8)
    assert c.reserve([0, 1], np.array([0, 48, 90], np.int32)) == 0  # three pages each: all six
    assert c.reserve([2, 3]) == 2
    assert c.reserve([0]) == -1
    assert c.reserve([1, 2, 0]) == -1
    assert c.reserve([1], np.array([0, 6], np.int32)) == 0  # fills its last page
    c.free([0])
    # 16 and 33 tokens need one page and three, of three that are free; 49 are more than a row's three pages hold
    assert c.reserve([2, 3, 2], np.array([0, 16, 49, 60], np.int32)) == 1
    assert c.reserve([2, 3, 2], np.array([0, 16, 65, 70], np.int32)) == -1
    assert c.reserve([2, 3], np.array([0, 16, 64], np.int32)) == 1
    assert c.reserve([2, 3], np.array([0, 16, 48], np.int32)) == 0
    assert c.reserve([]) == 0
    assert c.reserve([-1, 9, -5]) == 0
    c.free([0, 1, 2, 3])
    assert c.reserve([0, 1, 2, 3, 4, 5], null=True) == 0  # no list: row i is sequence i, rows from nseq on are padding


def test_long_lists_and_many_pages():
    """Lists of more entries than the planning block has threads, pages over several scans."""
    say("8192 sequences, 9001 pages")
    rng = np.random.default_rng(1)
    c = Cache(Table(8192, 3, 9001, 16), rng, 2, 8)
    every = rng.permutation(8192).astype(np.int32)
    assert c.reserve(every) == 0
    assert c.reserve(every[:1000]) == 0
    c.free(every[rng.permutation(8192)[:4000]])
    c.compact()
    src = every[rng.integers(0, 8192, 5000)]
    empties = np.flatnonzero(c.t.lens == 0)
    assert c.fork(src, np.resize(empties, 5000)) == 0
    for _ in range(17):
        c.reserve(every[:3000])
    c.compact()


@pytest.mark.parametrize("page,part", [(16, 0), (16, 1), (16, 15), (64, 33), (1024, 1000)])
def test_forks_share_whole_pages_and_copy_the_filled_rows(page, part):
    say(f"fork page={page} part={part}")
    rng = np.random.default_rng(part)
    c = Cache(Table(12, 4, 40, page), rng, 66, 24)  # more pools than one launch takes
    assert c.reserve([3, 5], np.array([0, 2 * page + part, 2 * page + part + 7], np.int32)) == 0
    assert c.fork([3, 3, 3, 5, 3, 0, 3, 8], [4, 6, 5, 7, 4, 9, 3, 10]) == 0
    # a source that is a destination, a destination twice, out of range
    assert c.fork([3, 0, 3, 3, -1, 3], [0, 1, 2, 2, 11, 12]) == 0
    c.free([3, 6, 4])
    c.compact()


def test_fork_without_room_changes_nothing():
    say("fork without room")
    rng = np.random.default_rng(5)
    c = Cache(Table(6, 4, 5, 16), rng, 2, 8)
    assert c.reserve([0], np.array([0, 40], np.int32)) == 0
    assert c.fork([0, 0, 0, 0], [1, 2, 3, 4]) == 2
    assert c.fork([0, 0], [1, 2]) == 0


def test_numbers_that_no_table_should_hold_are_not_followed():
    """Page numbers out of range in a table's row: no row is written there, no count changes."""
    say("bad page numbers")
    rng = np.random.default_rng(6)
    t = R.scattered(rng, 3, [40, 20, 17], 16)
    t.table[0, 1], t.table[1, 1], t.table[2, 1] = t.npages, -7, 2 ** 31 - 1
    c = Cache(t, rng, 2, 64)
    c.write([0, 1, 2], np.array([0, 40, 60, 77], np.int32), rng)
    c.write([0, 1, 2], np.array([0, 50, 90, 110], np.int32), rng)  # more rows than tokens: those before position 0 are left out


@pytest.mark.parametrize("bytes_,entries,npools", [(16, 9, 1), (48, 5, 3), (16384 + 16, 7, 70), (2 * 128 * 128 * 4, 6, 2)])
def test_copies_of_entries(bytes_, entries, npools):
    say(f"copy {bytes_} bytes, {entries} entries, {npools} pools")
    rng = np.random.default_rng(entries)
    pools = [R.bf16(rng, entries, bytes_ // 2) for _ in range(npools)]
    bufs = pool_buffers(pools)
    src = np.array([0, 1, 3, -1, 0, entries, 2, 4], np.int32)
    dst = np.array([2, 2, 1, 0, entries, 1, 3, 4], np.int32)
    want = [p.copy() for p in pools]
    for s, d in R.Table(entries, 1, 1, 16).pairs(src, dst, entries):
        for w, p in zip(want, pools):
            w[d] = p[s]
    a, b, ptrs = ints(src), ints(dst), pointers(bufs)
    hip.check(hip.api().cs1_kv_copy(ptrs, npools, bytes_, entries, a.at(0), b.at(0), len(src),
                                    stream().handle), "copy")
    for b, w in zip(bufs, want):
        np.testing.assert_array_equal(read_pool(b, w), w)


@pytest.mark.parametrize("bytes_,entries,npools,n", [(16384 + 16, 40, 64, 90), (16 * 700, 30, 3, 8192), (3 * 16384, 9, 66, 40)])
def test_copies_in_runs(bytes_, entries, npools, n):
    """So many blocks that each takes several pairs, in lists that name entries out of range, twice and as source and destination."""
    say(f"copy {bytes_} bytes, {entries} entries, {npools} pools, {n} pairs")
    rng = np.random.default_rng(n)
    pools = [R.bf16(rng, entries, bytes_ // 2) for _ in range(npools)]
    bufs = pool_buffers(pools)
    half = entries // 2
    src = np.repeat(rng.integers(-1, half + 1, n), rng.integers(1, 9, n))[:n].astype(np.int32)
    dst = rng.integers(half, entries + 2, n).astype(np.int32)
    src[-1], dst[-2] = entries, -3
    want = [p.copy() for p in pools]
    pairs = list(R.Table(entries, 1, 1, 16).pairs(src, dst, entries))
    assert len(pairs) > 3
    for s, d in pairs:
        for w, p in zip(want, pools):
            w[d] = p[s]
    a, b, ptrs = ints(src), ints(dst), pointers(bufs)
    hip.check(hip.api().cs1_kv_copy(ptrs, npools, bytes_, entries, a.at(0), b.at(0), n, stream().handle), "copy")
    for b, w in zip(bufs, want):
        np.testing.assert_array_equal(read_pool(b, w), w)


def test_forks_in_runs():
    """A block takes several pairs: of the same source, of others, of one without rows to copy, of one that is left out."""
    say("fork in runs")
    rng = np.random.default_rng(11)
    c = Cache(Table(90, 3, 200, 64), rng, 64, 1024)
    lens = [100, 64, 127, 65, 1, 129]
    assert c.reserve(range(6), np.cumsum([0] + lens).astype(np.int32)) == 0
    src = np.repeat([0, 1, 2, 3, 4, 5, 2, 0, -1, 4, 89], 7)[:74]
    dst = np.arange(6, 80)
    dst[[9, 20, 33]] = [6, 90, 2]  # twice, out of range, one that holds tokens (and so sequence 2 is no source)
    assert c.fork(src, dst) == 0
    c.free([0, 2, 5, 7, 8])
    c.compact()


@pytest.mark.parametrize("width", [1024, 1032, 1536, 2048, 8200])
def test_wide_rows(width):
    """Rows around and past the 128 packs that a wave holds at once, single tokens and prompts."""
    say(f"write rows of {width}")
    rng = np.random.default_rng(width)
    t = R.scattered(rng, 7, [5, 33, 0, 16, 48, 1, 17], 16)
    c = Cache(t, rng, 2, width)
    c.write([6, 1, -1, 3, 2, 0, 6], None, rng)
    c.write([4, 0, 7, 6, 1], np.array([0, 20, 25, 30, 31, 64], np.int32), rng, pad=(16, 0))


def test_prompts_of_more_sequences_than_a_launch_takes():
    """150 entries of host offsets, in launches of 64: empty ones, padding and repeats on both sides of their borders."""
    say("write 150 ragged entries")
    rng = np.random.default_rng(22)
    lens = rng.integers(1, 40, 140)
    t = R.scattered(rng, 140, lens.tolist(), 16)
    c = Cache(t, rng, 2, 72)
    seqs = rng.permutation(140)[:130].tolist() + [-1] * 20
    seqs = np.array(seqs)[rng.permutation(150)]
    seqs[63], seqs[64], seqs[65] = seqs[3], 140, seqs[64]
    seqs[127], seqs[128], seqs[149] = seqs[70], -7, seqs[66]
    rows = rng.integers(0, 12, 150)
    rows[[0, 62, 64, 126, 129, 148]] = 0
    rows[[63, 65, 127, 128, 149]] = 5
    cu = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    c.write(seqs, cu, rng)
    rows[:64] = 0  # a first launch without rows
    rows[64:] = 3
    c.write(seqs, np.concatenate([[0], np.cumsum(rows)]).astype(np.int32), rng, pad=(8, 16))
    c.write(seqs, np.concatenate([[0], np.cumsum(rng.integers(0, 60, 150))]).astype(np.int32), rng)


def test_repeats_far_into_a_list():
    """Sequences that entries past the 64th name, named again: the first has them, and their pages are given back once."""
    say("repeats past the first 64 entries")
    rng = np.random.default_rng(23)
    t = R.scattered(rng, 400, rng.integers(1, 40, 400).tolist(), 16)
    c = Cache(t, rng, 2, 8)
    seqs = rng.permutation(400)[:300]
    seqs[[130, 192, 260, 296, 297, 298, 299]] = seqs[[129, 64, 65, 64, 127, 128, 200]]
    c.write(seqs, None, rng)
    c.write(seqs, np.arange(301, dtype=np.int32) * 2, rng)
    c.free(seqs)
    assert (c.t.refs >= 0).all()
    src = rng.permutation(np.flatnonzero(c.t.lens > 0))[:90]
    dst = np.flatnonzero(c.t.lens == 0)[:90]
    dst[[80, 89]] = dst[[64, 70]]
    assert c.fork(src, dst) == 0
    c.free(np.concatenate([seqs, dst, dst[::-1], src]))


def test_two_tables_on_two_streams():
    """Calls on different tables run at the same time."""
    say("two tables on two streams")
    rng = np.random.default_rng(24)
    api, other = hip.api(), hip.Stream()
    sides = []
    for st, page in ((stream(), 16), (other, 48)):
        c = Cache(R.scattered(rng, 40, rng.integers(1, 90, 20).tolist(), page, max_pages=9, spare=150), rng, 2, 128)
        src, dst = rng.integers(0, 20, 20), np.arange(20, 40)
        k, v = R.bf16(rng, 20, 128), R.bf16(rng, 20, 128)
        sides.append((c, st, src, dst, k, v, [ints(src), ints(dst), dev(k), dev(v)], [ints([9]) for _ in range(3)]))
    stream().sync()
    for c, st, src, dst, k, v, (a, b, kb, vb), status in sides:
        hip.check(api.cs1_kv_fork(c.d.ref, a.at(0), b.at(0), 20, c.ptrs, 2, 256, c.ws.at(0), status[0].at(0), st.handle), "fork")
        hip.check(api.cs1_kv_reserve(c.d.ref, b.at(0), None, 20, status[1].at(0), st.handle), "reserve")
        hip.check(api.cs1_kv_write(c.d.ref, b.at(0), None, 20, kb.at(0), 128, vb.at(0), 128, c.bufs[0].at(0), c.bufs[1].at(0), 1,
                                   128, st.handle), "write")
        hip.check(api.cs1_kv_free(c.d.ref, a.at(0), 20, st.handle), "free")
        hip.check(api.cs1_kv_compact(c.d.ref, c.ptrs, 2, 256, c.ws.at(0), status[2].at(0), st.handle), "compact")
    other.sync()
    stream().sync()
    for c, _, src, dst, k, v, _, status in sides:
        want = [c.t.fork(src, dst, c.pools), c.t.reserve(dst)]
        c.t.write(dst, None, k, v, c.pools[0], c.pools[1])
        c.t.free(src)
        want.append(c.t.compact(c.pools))
        assert [int(get(s, np.int32, 1)[0]) for s in status] == want
        c.check("both")
    other.destroy()


def test_pages_in_a_graph():
    """Free, fork, reserve, write, compact and copy recorded once and replayed for other lists, with eager calls between."""
    say("the page calls in a graph")
    rng = np.random.default_rng(21)
    c = Cache(Table(12, 6, 60, 16), rng, 2, 64)
    assert c.reserve([0, 1, 2], np.array([0, 40, 56, 80], np.int32)) == 0
    gone, src, dst, new = (ints([-1] * 4) for _ in range(4))
    k, v = R.bf16(rng, 4, 64), R.bf16(rng, 4, 64)
    kb, vb, st, api = dev(k), dev(v), stream().handle, hip.api()
    entries = [R.bf16(rng, 12, 24)]
    ebufs = pool_buffers(entries)
    status, eptrs = [ints([77]) for _ in range(3)], pointers(ebufs)

    def record():
        hip.check(api.cs1_kv_free(c.d.ref, gone.at(0), 4, st), "free")
        hip.check(api.cs1_kv_fork(c.d.ref, src.at(0), dst.at(0), 4, c.ptrs, 2, 128, c.ws.at(0), status[0].at(0), st), "fork")
        hip.check(api.cs1_kv_copy(eptrs, 1, 48, 12, src.at(0), dst.at(0), 4, st), "copy")
        hip.check(api.cs1_kv_reserve(c.d.ref, new.at(0), None, 4, status[1].at(0), st), "reserve")
        hip.check(api.cs1_kv_write(c.d.ref, new.at(0), None, 4, kb.at(0), 64, vb.at(0), 64, c.bufs[0].at(0), c.bufs[1].at(0), 8, 8, st), "write")
        hip.check(api.cs1_kv_compact(c.d.ref, c.ptrs, 2, 128, c.ws.at(0), status[2].at(0), st), "compact")

    g = hip.Graph(stream(), record)
    c.check("recorded")  # and nothing has run
    lists = [([-1, -1, -1, -1], [0, 0, 2, 1], [3, 4, 5, 6], [0, 3, 4, 5]), ([1, 4, 1, 12], [3, 3, 0, -1], [1, 4, 7, 8], [1, 3, 7, 1]),
             ([0, 2, 3, 5], [7, 1, 6, 6], [8, 9, 10, 10], [10, 9, 8, -1]), ([9, 9, 9, 9], [8, 8, 8, 8], [0, 2, 3, 5], [5, 0, 2, 3])]
    for one in lists:
        for buf, x in zip((gone, src, dst, new), one):
            hip.upload(buf, np.array(x, np.int32), stream())
        g.launch(stream())
        t = c.t
        t.free(one[0])
        want = [t.fork(one[1], one[2], c.pools)]
        for s, d in list(t.pairs(one[1], one[2], 12)):
            entries[0][d] = entries[0][s]
        want.append(t.reserve(one[3]))
        t.write(one[3], None, k, v, c.pools[0], c.pools[1])
        want.append(t.compact(c.pools))
        assert [int(get(s, np.int32, 1)[0]) for s in status] == want
        c.check("replayed")
        np.testing.assert_array_equal(read_pool(ebufs[0], entries[0]), entries[0])
        assert c.reserve([6]) == 0  # an eager call between


def test_offsets_past_32_bits():
    """The last page of a pool of 5 GiB receives rows, is forked and moves to the front."""
    say("a pool of 5 GiB")
    page, width = 64, 1024
    npages = (5 << 30) // (page * width * 2)
    t = Table(3, 4, npages, page)
    t.table[0, 0], t.refs[npages - 1], t.lens[0] = npages - 1, 1, 37
    t.refs[npages - 2], t.table[1, 0], t.lens[1] = 1, npages - 2, 1
    t.refs[1:npages - 2] = 1  # held by nobody here: only pages 0 and 1 are of interest
    t.refs[1] = 0
    d = DeviceTable(t)
    pool_k, pool_v = empty(npages * page * width * 2), empty(npages * page * width * 2)
    rng = np.random.default_rng(2)
    k, v = R.bf16(rng, 37, width), R.bf16(rng, 37, width)
    kb, vb = dev(k), dev(v)
    cu = np.array([0, 37], np.int32)
    api, st, first, third = hip.api(), stream().handle, ints([0]), ints([2])
    hip.check(api.cs1_kv_write(d.ref, first.at(0), cu.ctypes.data, 1, kb.at(0), width, vb.at(0), width, pool_k.at(0),
                               pool_v.at(0), 8, 128, st), "write")
    last = (npages - 1) * page * width * 2
    np.testing.assert_array_equal(get(pool_k, np.uint16, 37 * width, last).reshape(37, width), k)
    ws, status, ptrs = empty(api.cs1_kv_workspace_bytes(npages, 1)), ints([1]), pointers([pool_k, pool_v])
    hip.check(api.cs1_kv_fork(d.ref, first.at(0), third.at(0), 1, ptrs, 2, width * 2, ws.at(0), status.at(0), st), "fork")
    assert get(status, np.int32, 1)[0] == 0
    np.testing.assert_array_equal(get(pool_v, np.uint16, 37 * width, 0).reshape(37, width), v)  # page 0 was the lowest free
    hip.check(api.cs1_kv_compact(d.ref, ptrs, 2, width * 2, ws.at(0), status.at(0), st), "compact")
    assert get(status, np.int32, 1)[0] == npages - 1
    table, _, refs = d.state()
    assert table[0, 0] == 1 and refs[npages - 1] == 0 and refs[1] == 1
    np.testing.assert_array_equal(get(pool_v, np.uint16, 37 * width, page * width * 2).reshape(37, width), v)
