"""A step of several new tokens for which there is no room, all of it in one graph: cs1_kv_rows_if_room goes by the status
that cs1_kv_extend has just left, so that no page, length or count changes; and the same graph once there is room."""
import ctypes

import numpy as np
import pytest

import decode_ref as R
import rows_ref as W
from decode_ref import DeviceTable, Table, ints
from gpu_helpers import dev, empty, get, say, stream
from qwen3_5_native import hip
from test_gpu_rows_step import Server

pytestmark = pytest.mark.gpu


class Careful(Server):
    """The server's step with the rows' places under the status."""

    def forward(self):
        api, b = hip.api(), self.b

        class Api:
            def __getattr__(self, name):
                return getattr(api, name)

            @staticmethod
            def cs1_kv_rows(pages, seqs, cu, n, rows, pos, slot, st):
                return api.cs1_kv_rows_if_room(pages, seqs, cu, n, rows, b["status"].at(0), pos, slot, st)

        real, hip.api = hip.api, Api
        try:
            super().forward()
        finally:
            hip.api = real

    def caches(self):
        return [get(y[x], np.uint8, y[x].nbytes) for y in self.layers for x in ("kp", "vp", "q", "g")] + list(self.d.state())


@pytest.mark.parametrize("n,rows,nseq", [(1, 1, 1), (5, 40, 7), (64, 1024, 64), (1025, 3000, 2000), (8192, 9000, 8192)])
def test_places_go_by_the_status(n, rows, nseq):
    say(f"rows if room: {rows} rows of {n}")
    rng = np.random.default_rng(n)
    t = Table(nseq, 4, 5 * nseq, 16)
    seqs = rng.integers(-1, nseq + 1, n) if n < nseq else rng.permutation(nseq)[:n]
    cu = np.concatenate([[0], np.cumsum(rng.integers(0, 3, n))])
    t.lens[:] = rng.integers(0, 64, nseq)
    t.table[:] = rng.integers(-1, t.npages + 1, t.table.shape)
    d, b, c, api = DeviceTable(t), ints(seqs), ints(cu), hip.api()
    for status in (0, 1, -1, 2 ** 31 - 1, -2 ** 31):
        out, st = dev(np.full(2 * (rows + 1), 99, np.int32)), ints([status])
        hip.check(api.cs1_kv_rows_if_room(d.ref, b.at(0), c.at(0), n, rows, st.at(0), out.at(0), out.at(4 * (rows + 1)),
                                          stream().handle), "rows if room")
        got = get(out, np.int32, 2 * (rows + 1)).reshape(2, -1)
        assert (got[:, rows] == 99).all() and get(st, np.int32, 1)[0] == status
        pos, slot = W.rows_of(t, seqs, cu, rows) if status == 0 else (np.full(rows, -1),) * 2
        np.testing.assert_array_equal(got[0, :rows], pos)
        np.testing.assert_array_equal(got[1, :rows], slot)


def test_a_step_without_room_changes_nothing():
    say("rows if room: a graph's steps with too few pages, beside a fork")
    rng = np.random.default_rng(4)
    n, rows = 5, 330
    stream()
    s = Careful(rng, 8, 2, 128, 128, 2, 1000, n, rows, 200, 4)
    api, t, d, st = hip.api(), s.t, s.d, stream().handle

    def upload(seqs, new):
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        xs = [R.bf16(rng, rows, s.ld) for _ in s.layers]
        targets = rng.integers(0, s.vocab, rows).astype(np.int32)
        for name, host in (("seqs", seqs), ("cu", cu), ("targets", targets)):
            hip.upload(s.b[name], np.asarray(host, np.int32), stream())
        for y, x in zip(s.layers, xs):
            hip.upload(y["x"], x, stream())
            for buf in ("q", "g", "out"):
                hip.upload(y[buf], np.zeros(rows * 8 * 128, np.uint16), stream())
        return seqs, cu, xs, targets

    try:
        # 48 of the 60 pages are two sequences' that take no part, then two prompts, and a fork of the first
        hogs, cu = ints([4, 5]), ints([0, 24 * 48, 48 * 48])
        hip.check(api.cs1_kv_extend(d.ref, hogs.at(0), cu.at(0), 2, s.b["status"].at(0), st), "extend")
        assert W.extend(t, [4, 5], [0, 24 * 48, 48 * 48]) == 0
        d.check()
        step = upload([0, 1, -1, -1, -1], [100, 100, 0, 0, 0])
        s.forward()
        s.check(*step)
        pools = [y[x] for y in s.layers for x in ("kp", "vp")]
        ptrs = (ctypes.c_void_p * 4)(*(p.at(0) for p in pools))
        src, dst, ws = ints([0]), ints([2]), empty(api.cs1_kv_workspace_bytes(t.npages, 1))
        hip.check(api.cs1_kv_fork(d.ref, src.at(0), dst.at(0), 1, ptrs, 4, 2 * 2 * 128, ws.at(0), s.b["status"].at(0), st), "fork")
        assert t.fork([0], [2], []) == 0
        d.check()
        graph = hip.Graph(stream(), s.forward)

        # three times 100 tokens want six pages, and there are five; then more than a sequence's row of the table
        for seqs, new, answer in (([0, 1, 2, -1, 9], [100, 100, 100, 4, 5], 1), ([2, 4, 0, 1, 3], [1, 1, 0, 2, 0], -1)):
            upload(seqs, new)
            before = s.caches()
            for run in (s.forward, lambda: graph.launch(stream()), lambda: graph.launch(stream())):
                run()
                assert get(s.b["status"], np.int32, 1)[0] == answer
                for x in ("pos", "slot"):
                    assert (get(s.b[x], np.int32, rows) == -1).all()
                for a, b in zip(before, s.caches()):
                    np.testing.assert_array_equal(a, b)
            d.check()

        # one of the two ends, and the same graph goes on where the sequences were
        gone = ints([5])
        hip.check(api.cs1_kv_free(d.ref, gone.at(0), 1, st), "free")
        t.free([5])
        step = upload([0, 1, 2, -1, 9], [100, 100, 100, 4, 5])
        s.forward()
        first = s.state()
        s.rewind()
        graph.launch(stream())
        for a, b in zip(first, s.state()):
            np.testing.assert_array_equal(a, b)
        s.check(*step)
    finally:
        s.close()
