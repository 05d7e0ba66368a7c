"""cs1_gdn_decode against the delta rule's step in float64 (decode_ref.gdn_step), within bounds that follow from
float32's roundings; against the prefill of the same tokens; padding, first tokens, repeats, graphs."""
import numpy as np
import pytest

import decode_ref as R
from decode_ref import D, ints
from gpu_helpers import dev, empty, get, get_bf16, say, stream
from qwen3_5_native import hip

pytestmark = pytest.mark.gpu
EPS = 1e-6


class Step:
    def __init__(self, rng, seqs, lens, H, HK, norm=True, pad=0):
        self.H, self.HK, self.norm = H, HK, norm
        self.seqs, self.lens = np.asarray(seqs, np.int32), np.asarray(lens, np.int32)
        B, n = len(seqs), len(lens)
        self.conv = (2 * HK + H) * D
        self.ld = self.conv + H * D + 2 * H + pad
        self.x = R.bf16(rng, B, self.ld)
        self.w = R.bf16(rng, self.conv, 4, std=0.3)
        self.a_log = R.O.f32_to_bf16(np.log(1 + 15 * rng.random(H)).astype(np.float32))
        self.dt = R.O.f32_to_bf16(np.log(np.expm1(np.exp(rng.uniform(np.log(1e-3), np.log(1e-1), H)))).astype(np.float32))
        self.gw = R.O.f32_to_bf16((1 + 0.1 * rng.standard_normal(D)).astype(np.float32)) if norm else None
        self.ring = R.bf16(rng, n, 4, self.conv)
        self.state = (rng.standard_normal((n, H, D, D)) * 0.1).astype(np.float32)

    def upload(self):
        self.bufs = {k: dev(getattr(self, k)) for k in ("seqs", "lens", "x", "w", "a_log", "dt", "ring", "state")}
        self.g = dev(self.gw) if self.norm else None
        self.n_out = len(self.seqs) * self.H * D
        self.out = dev(np.full(self.n_out + 8, 0x7fc1, np.uint16))

    def launch(self, null=False):
        b = {k: v.at(0) for k, v in self.bufs.items()}
        z = b["x"] + 2 * self.conv
        pb = z + 2 * self.H * D
        hip.check(hip.api().cs1_gdn_decode(
            b["x"], self.ld, b["w"], z if self.norm else None, pb, pb + 2 * self.H, b["a_log"], b["dt"],
            self.g.at(0) if self.norm else None, EPS, b["ring"], b["state"], None if null else b["seqs"], b["lens"],
            len(self.lens), self.out.at(0), len(self.seqs), self.H, self.HK, D ** -0.5, stream().handle), "gdn_decode")

    def results(self):
        out = get_bf16(self.out, self.n_out + 8)
        assert (out[self.n_out:] == 0x7fc1).all(), "written behind the last row"
        return (out[:self.n_out].reshape(len(self.seqs), self.H, D),
                get(self.bufs["state"], np.float32, self.state.size).reshape(self.state.shape),
                get_bf16(self.bufs["ring"], self.ring.size).reshape(self.ring.shape))

    def want(self, seqs=None):
        return R.gdn_step(self.x, self.w, self.a_log, self.dt, self.gw, self.ring, self.state,
                          self.seqs if seqs is None else seqs, self.lens, self.H, self.HK, D ** -0.5, EPS)

    def check(self, seqs=None):
        out, state, ring = self.results()
        want, S, ring2, tol, stol = self.want(seqs)
        R.close(R.f64(out), want, tol, "out")
        R.close(state.astype(np.float64), S, stol, "state")
        np.testing.assert_array_equal(ring, ring2)


@pytest.mark.parametrize("H,HK", [(16, 16), (32, 16), (48, 16), (1, 1), (6, 2), (5, 1), (33, 11)])
@pytest.mark.parametrize("norm", [True, False])
def test_heads(H, HK, norm):
    say(f"gdn decode heads {H}/{HK} norm={norm}")
    rng = np.random.default_rng(H)
    s = Step(rng, [2, 0, 3], [1, 9, 700, 2], H, HK, norm, pad=3)
    s.upload()
    s.launch()
    s.check()


def test_first_tokens_take_nothing_from_before():
    """Positions 0 to 5, with NaN where no earlier token is held."""
    say("gdn decode: first tokens")
    rng = np.random.default_rng(1)
    s = Step(rng, [5, 0, 4, 1, 3, 2], [1, 2, 3, 4, 5, 6], 4, 2)
    for q, n in enumerate(s.lens):
        for r in range(4):
            if r not in [i % 4 for i in range(max(0, n - 4), n - 1)]:
                s.ring[q, r] = 0x7fc0
    s.state[0] = np.nan
    s.upload()
    s.launch()
    s.check()


def test_padding_and_repeats():
    """Numbers out of range, sequences without tokens, a sequence named twice: zeros, and nothing else changes."""
    say("gdn decode: padding and repeats")
    rng = np.random.default_rng(2)
    s = Step(rng, [1, -1, 0, 4, 1, 2, 2 ** 31 - 1, 3, 0, -2 ** 31], [3, 9, 0, -5], 4, 4)
    s.x[[1, 3, 4, 5, 6, 7, 8, 9]] = 0x7fc0
    s.upload()
    s.launch()
    s.check()
    out = s.results()[0]
    assert (out[[1, 3, 4, 5, 6, 7, 8, 9]] == 0).all() and np.abs(R.f64(out[[0, 2]])).max() > 0


def test_no_list():
    say("gdn decode: no list")
    rng = np.random.default_rng(3)
    s = Step(rng, [-1] * 5, [7, 1, 30], 2, 2)
    s.upload()
    s.launch(null=True)
    s.check(seqs=[0, 1, 2, -1, -1])


def test_strong_and_weak_decays():
    """A state that is forgotten at once, one that stays, gates that are shut and wide open."""
    say("gdn decode: extreme gates")
    rng = np.random.default_rng(4)
    s = Step(rng, [0, 1, 2], [50, 51, 52], 4, 2)
    s.a_log = R.O.f32_to_bf16(np.array([2.77, -20.0, 2.77, 0.0], np.float32))
    s.dt = R.O.f32_to_bf16(np.array([60.0, 0.0, -40.0, 19.0], np.float32))
    b0 = s.conv + 4 * D
    s.x[:, b0:b0 + 4] = R.O.f32_to_bf16(np.array([[-90, 90, 0, 5], [30, -30, -4, 4], [0, 0, 100, -100]], np.float32).reshape(-1)).reshape(3, 4)
    s.upload()
    s.launch()
    s.check()


def test_many_rows():
    say("gdn decode: 300 rows of 320 sequences, the last row a repeat")
    rng = np.random.default_rng(5)
    seqs = rng.permutation(320)[:300]
    seqs[-1] = seqs[7]
    s = Step(rng, seqs, rng.integers(1, 9, 320), 2, 1)
    s.upload()
    s.launch()
    s.check()


def test_repeats_far_into_a_list():
    """Sequences that rows past the 64th name, named again: zeros there, and one block a head has the state."""
    say("gdn decode: repeats past the first 64 rows")
    rng = np.random.default_rng(18)
    seqs = rng.permutation(320)[:300]
    again = [130, 192, 260, 296, 297, 298, 299]
    seqs[again] = seqs[[129, 64, 65, 64, 127, 128, 200]]
    s = Step(rng, seqs, rng.integers(1, 9, 320), 2, 1)
    s.upload()
    s.launch()
    s.check()
    assert (s.results()[0][again] == 0).all()


def test_steps_follow_the_prefill():
    """Twenty tokens one at a time from what a prefill leaves, against a prefill of all of them."""
    say("gdn decode after a prefill")
    api, st = hip.api(), stream().handle
    H, HK, T, N = 4, 2, 77, 20
    rng = np.random.default_rng(6)
    s = Step(rng, [1], [0, T, 0], H, HK, norm=False)
    rows = R.bf16(rng, T + N, s.ld)
    xb, w, al, dt = dev(rows), dev(s.w), dev(s.a_log), dev(s.dt)
    pb = 2 * (s.conv + H * D)
    o = empty((T + N) * H * D * 2)

    def prefill(n, o, s_out):
        q, k, v = empty(n * HK * D * 2), empty(n * HK * D * 2), empty(n * H * D * 2)
        ws = empty(api.cs1_gdn_workspace_floats(n, H) * 4)
        hip.check(api.cs1_gdn_conv(xb.at(0), s.ld, w.at(0), q.at(0), k.at(0), v.at(0), n, HK * D, H * D, st), "conv")
        hip.check(api.cs1_gdn_prefill_gated_x(q.at(0), k.at(0), v.at(0), xb.at(pb), xb.at(pb + 2 * H), s.ld, al.at(0), dt.at(0),
                                              o.at(0), ws.at(0), n, H, HK, D ** -0.5, None, s_out, st), "prefill")
        stream().sync()

    final, first = empty(H * D * D * 4), empty(H * D * D * 4)
    prefill(T + N, o, final.at(0))
    whole = R.f64(get_bf16(o, (T + N) * H * D).reshape(T + N, H, D))
    prefill(T, empty(T * H * D * 2), first.at(0))
    s.state[1] = get(first, np.float32, H * D * D).reshape(H, D, D)
    for i in range(T - 3, T):
        s.ring[1, i % 4] = rows[i, :s.conv]
    s.upload()
    step = []
    for i in range(N):
        hip.upload(s.bufs["lens"], np.array([0, T + i + 1, 0], np.int32), stream())
        hip.upload(s.bufs["x"], rows[T + i], stream())
        s.launch()
        step.append(R.f64(s.results()[0][0]))
    # the prefill rounds q, k, v, beta and its chunks' operands to bfloat16, this does not: half a step each of
    # operands of size one, in sums over a few dozen tokens
    err, size = np.abs(np.array(step) - whole[T:]), np.sqrt((whole[T:] ** 2).mean())
    print(f"  largest difference {err.max() / size:.4f} of the rms", flush=True)
    assert err.max() <= 16 * R.E16 * max(size, np.abs(whole[T:]).max())
    want = get(final, np.float32, H * D * D).reshape(H, D, D)
    got = s.results()[1][1]
    assert np.linalg.norm(got - want) <= 4 * R.E16 * np.linalg.norm(want)


def test_the_same_bits_every_time_and_in_a_graph():
    say("gdn decode: repeats and graphs")
    rng = np.random.default_rng(7)
    s = Step(rng, [2, 0, -1, 1], [6, 1, 77], 8, 4)
    s.upload()
    s.launch()
    first = s.results()
    s.check()

    def reset():
        hip.upload(s.bufs["state"], s.state, stream())
        hip.upload(s.bufs["ring"], s.ring, stream())

    g = hip.Graph(stream(), s.launch)
    for _ in range(3):
        reset()
        g.launch(stream())
        for a, b in zip(s.results(), first):
            np.testing.assert_array_equal(a, b)
        reset()
        s.launch()
        for a, b in zip(s.results(), first):
            np.testing.assert_array_equal(a, b)
    # the graph reads the lists when it runs
    s.seqs[:] = [1, -1, 2, 0]
    hip.upload(s.bufs["seqs"], s.seqs, stream())
    reset()
    g.launch(stream())
    s.check()


def test_offsets_past_32_bits():
    """Sequences whose states lie behind 4 GiB."""
    say("gdn step: states of 4.4 GB")
    rng = np.random.default_rng(17)
    H, HK, many = 48, 16, 1400
    c = Step(rng, [2, 0, 1], [9, 1, 700], H, HK)
    want, S, ring2, tol, stol = c.want()
    c.upload()
    at = np.array([many - 1, 3, many - 30])  # where sequences 0, 1, 2 are
    lens = np.zeros(many, np.int32)
    lens[at] = c.lens
    size, rsize = H * D * D * 4, 4 * c.conv * 2
    state, ring = empty(many * size), empty(many * rsize)
    for i, s in enumerate(at):
        hip.upload(state, c.state[i], stream(), offset=int(s) * size)
        hip.upload(ring, c.ring[i], stream(), offset=int(s) * rsize)
    c.bufs.update(state=state, ring=ring, lens=dev(lens), seqs=ints(at[c.seqs]))
    c.lens = lens
    c.launch()
    out = get_bf16(c.out, c.n_out).reshape(3, H, D)
    R.close(R.f64(out), want, tol, "out")
    for i, s in enumerate(at):
        got = get(state, np.float32, H * D * D, int(s) * size).reshape(H, D, D)
        R.close(got.astype(np.float64), S[i], stol[i], f"state {i}")
        np.testing.assert_array_equal(get_bf16(ring, 4 * c.conv, int(s) * rsize).reshape(4, c.conv), ring2[i])
