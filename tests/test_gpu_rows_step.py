"""Several new tokens of cached sequences at once, the operations as a server runs them: room and places, attention inputs into
the pages, attention, the head's product, log-probabilities, and rejected tokens taken back.  One captured graph
serves every step, and each is checked part by part against float64 and bit by bit against the same calls without a graph."""
import ctypes

import numpy as np
import pytest

import decode_ref as R
import rows_ref as W
from decode_ref import DeviceTable, Table, ints
from gpu_helpers import dev, empty, get, get_bf16, say, stream
from qwen3_5_native import hip
from test_gpu_logprobs import reference as logprobs_reference

pytestmark = pytest.mark.gpu
EPS = 1e-6


class Server:
    """`layers` attention layers over one page table; a step's inputs are each layer's projected rows, as if from a model."""

    def __init__(self, rng, hq, hk, dh, dims, layers, vocab, n, rows, max_new, k, seqs=6, page=48):
        self.__dict__.update(hq=hq, hk=hk, dh=dh, dims=dims, vocab=vocab, n=n, rows=rows, max_new=max_new, k=k)
        self.t = Table(seqs, 24, 60, page)
        self.d = DeviceTable(self.t)
        self.ld = 2 * hq * dh + 2 * hk * dh
        self.w = [[R.bf16(rng, dh, std=0.2) for _ in range(2)] for _ in range(layers)]
        self.head = R.bf16(rng, vocab, hq * dh, std=0.05)
        freqs = (ctypes.c_double * (dims // 2))()
        hip.check(hip.api().cs1_rotary_freqs(freqs, dims, 1e6, 4.0, 1000.0, 1.0, 32.0), "rotary_freqs")
        self.freqs, self.magnitude = np.array(freqs), float(np.float32(0.1 * np.log(4) + 1))
        self.b = dict(head=dev(self.head), freqs=dev(self.freqs), status=ints([77]), seqs=ints([0] * n), cu=ints([0] * (n + 1)),
                      pos=ints([9] * rows), slot=ints([9] * rows), targets=ints([0] * rows), logits=empty(2 * rows * vocab),
                      lp=empty(4 * rows), ent=empty(4 * rows), ids=empty(4 * rows * k), top=empty(4 * rows * k), drop=ints([0] * n),
                      ws=empty(max(16, hip.api().cs1_token_logprobs_workspace_bytes(rows, vocab, k))))
        size = self.t.npages * page * hk * dh
        self.layers = [dict(x=empty(2 * rows * self.ld), qw=dev(w[0]), kw=dev(w[1]), kp=dev(np.zeros(size, np.uint16)),
                            vp=dev(np.zeros(size, np.uint16)), q=empty(2 * rows * hq * dh), g=empty(2 * rows * hq * dh),
                            out=empty(2 * rows * hq * dh), lse=empty(4 * rows * hq)) for w in self.w]
        self.attention, self.gemm = hip.api().cs1_attention_paged_create(), hip.api().cs1_gemm_create(1 << 25)
        assert self.attention and self.gemm

    def close(self):
        hip.api().cs1_attention_paged_destroy(self.attention)
        hip.api().cs1_gemm_destroy(self.gemm)

    def forward(self):
        api, st, b, d = hip.api(), stream().handle, self.b, self.d
        hq, hk, dh = self.hq, self.hk, self.dh
        at = lambda x: b[x].at(0)  # noqa: E731
        hip.check(api.cs1_kv_extend(d.ref, at("seqs"), at("cu"), self.n, at("status"), st), "extend")
        hip.check(api.cs1_kv_rows(d.ref, at("seqs"), at("cu"), self.n, self.rows, at("pos"), at("slot"), st), "rows")
        rot = hip.Rotary(at("freqs"), self.dims, 0, self.magnitude)
        for y in self.layers:
            p = lambda x: y[x].at(0)  # noqa: E731, B023
            hip.check(api.cs1_attn_prep_paged(p("x"), y["x"].at(4 * hq * dh), y["x"].at(4 * hq * dh + 2 * hk * dh), self.ld, p("qw"), p("kw"),
                                              EPS, ctypes.byref(rot), d.ref, at("pos"), at("slot"), p("q"), p("g"), p("kp"), p("vp"), self.rows,
                                              hq, hk, dh, st), "prep")
            hip.check(api.cs1_attention_paged_varlen(self.attention, p("q"), p("kp"), p("vp"), d.ref, at("seqs"), at("cu"), self.n,
                                                     self.max_new, p("g"), p("out"), p("lse"), self.rows, hq, hk, dh, dh ** -0.5, st), "attention")
        hip.check(api.cs1_gemm(self.gemm, self.layers[-1]["out"].at(0), at("head"), at("logits"), self.rows, self.vocab, hq * dh, self.vocab, st),
                  "head")
        hip.check(api.cs1_token_logprobs(at("logits"), 0, self.vocab, at("targets"), self.rows, self.vocab, self.k, at("lp"), at("ent"), at("ids"),
                                         at("top"), at("ws"), st), "logprobs")

    def state(self):
        """Everything that a step leaves, as bytes."""
        n = self.rows * self.hq * self.dh
        out = [get(self.b[x], np.uint8, self.b[x].nbytes) for x in ("status", "pos", "slot", "logits", "lp", "ent", "ids", "top")]
        for y in self.layers:
            out += [get_bf16(y["kp"], y["kp"].nbytes // 2), get_bf16(y["vp"], y["vp"].nbytes // 2), get_bf16(y["out"], n),
                    get(y["lse"], np.float32, self.rows * self.hq)]
        return out + list(self.d.state())

    def rewind(self):
        """The table as it was before the step."""
        for buf, host in zip((self.d.table, self.d.lens, self.d.refs), (self.t.table, self.t.lens, self.t.refs)):
            hip.upload(buf, host, stream())

    def check(self, seqs, cu, xs, targets):
        hq, hk, dh, rows = self.hq, self.hk, self.dh, self.rows
        assert W.extend(self.t, seqs, cu) == 0 and get(self.b["status"], np.int32, 1)[0] == 0
        self.d.check()
        pos, slot = W.rows_of(self.t, seqs, cu, rows)
        np.testing.assert_array_equal(get(self.b["pos"], np.int32, rows), pos)
        np.testing.assert_array_equal(get(self.b["slot"], np.int32, rows), slot)
        live, m = pos >= 0, self.t.npages * self.t.page
        for i, (x, w, y) in enumerate(zip(xs, self.w, self.layers)):
            x = x[live]
            raw, kv = x[:, :2 * hq * dh].reshape(-1, hq, 2 * dh), x[:, 2 * hq * dh:].reshape(-1, 2, hk, dh)
            turn = lambda a, b: W.turned(R.f64(np.ascontiguousarray(a)), R.f64(b), EPS, pos[live], self.freqs, self.dims, False,  # noqa: E731
                                         self.magnitude)
            q, g, out = (get_bf16(y[a], rows * hq * dh).reshape(rows, hq, dh) for a in ("q", "g", "out"))
            kp, vp = (get_bf16(y[a], m * hk * dh).reshape(m, hk, dh) for a in ("kp", "vp"))
            R.close(R.f64(q[live]), *turn(raw[..., :dh], w[0]), f"layer {i} q")
            R.close(R.f64(kp[slot[live]]), *turn(kv[:, 0], w[1]), f"layer {i} k")
            np.testing.assert_array_equal(vp[slot[live]], kv[:, 1])
            np.testing.assert_array_equal(g[live], raw[..., dh:])
            paged = lambda a: a.reshape(self.t.npages, self.t.page, hk, dh)  # noqa: E731
            want, wl, tol, ltol, ours = W.attention(self.t, seqs, cu, rows, self.max_new, q, paged(kp), paged(vp), g, hk, dh ** -0.5)
            R.close(R.f64(out[ours]), want[ours], tol[ours], f"layer {i} out")
            lse = get(y["lse"], np.float32, rows * hq).reshape(hq, rows)
            R.close(lse[:, ours].astype(np.float64), wl[:, ours], ltol[:, ours], f"layer {i} lse")
        x = R.f64(out[live]).reshape(-1, hq * dh)
        logits = R.f64(get_bf16(self.b["logits"], rows * self.vocab).reshape(rows, self.vocab)[live])
        head = R.f64(self.head)
        want = x @ head.T  # float32 sums of hq dh products in any order, and one rounding
        off = (hq * dh + 2) * R.E32 * (np.abs(x) @ np.abs(head).T)
        R.close(logits, want, off + R.E16 * (np.abs(want) + off), "logits")
        k = self.k
        (wl, tl), (we, te), wi, (wt, tt) = logprobs_reference(logits, targets[live], k)
        R.close(get(self.b["lp"], np.float32, rows)[live].astype(np.float64), wl, tl, "logprob")
        R.close(get(self.b["ent"], np.float32, rows)[live].astype(np.float64), we, te, "entropy")
        np.testing.assert_array_equal(get(self.b["ids"], np.int32, rows * k).reshape(rows, k)[live], wi)
        R.close(get(self.b["top"], np.float32, rows * k).reshape(rows, k)[live].astype(np.float64), wt, tt, "top")


@pytest.mark.parametrize("hq,hk,dh,dims", [(8, 2, 128, 128), (8, 2, 256, 64)])
def test_steps_in_one_graph(hq, hk, dh, dims):
    say(f"rows step: heads {hq}/{hk} Dh={dh}")
    rng = np.random.default_rng(dh)
    n, rows, max_new, k = 5, 330, 200, 4
    stream()
    s = Server(rng, hq, hk, dh, dims, 2, 1000, n, rows, max_new, k)
    try:
        graph = None
        # prompts; drafts behind them, most taken back; a prompt's next part beside single tokens; drafts alone; a second turn
        steps = [([0, 3, -1, 5, 1], [33, 200, 4, 1, 90], None), ([5, 0, 3, 1, -1], [4, 4, 4, 4, 0], [3, 0, 4, 2, 9]),
                 ([2, 0, 1, 3, 5], [150, 1, 1, 1, 1], [0, 0, 9, 0, 1]), ([0, 2, 3, 5, 1], [4, 3, 2, 1, 4], [4, 3, 2, 1, 4]),
                 ([0, 1, 3, 2, 9], [77, 100, 2, 100, 30], [100, 3, 0, 0, 5])]
        for i, (seqs, new, drop) in enumerate(steps):
            say(f"  step {i}")
            cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
            xs = [R.bf16(rng, rows, s.ld) for _ in s.layers]
            targets = rng.integers(0, s.vocab, rows).astype(np.int32)
            for name, host in (("seqs", seqs), ("cu", cu), ("targets", targets)):
                hip.upload(s.b[name], np.asarray(host, np.int32), stream())
            for y, x in zip(s.layers, xs):
                hip.upload(y["x"], x, stream())
                for buf in ("q", "g", "out"):  # rows of no one go through the head too: they are something
                    hip.upload(y[buf], np.zeros(rows * hq * dh, np.uint16), stream())
            s.forward()
            first = s.state()
            if graph is None:
                graph = hip.Graph(stream(), s.forward)
            for _ in range(2):
                s.rewind()
                graph.launch(stream())
                for a, b in zip(first, s.state()):
                    np.testing.assert_array_equal(a, b)
            s.check(seqs, cu, xs, targets)
            if drop is not None:
                hip.upload(s.b["drop"], np.asarray(drop, np.int32), stream())
                hip.check(hip.api().cs1_kv_trim(s.d.ref, s.b["seqs"].at(0), s.b["drop"].at(0), n, s.b["status"].at(0), stream().handle), "trim")
                assert W.trim(s.t, seqs, drop) == get(s.b["status"], np.int32, 1)[0]
                s.d.check()
    finally:
        s.close()
