"""Decoding as a program does it: a prompt is prefilled, its keys and values go to pages and its delta-rule
state to a slot, it is forked into continuations, and each takes tokens one at a time in a captured
graph of all the calls.  Every continuation's outputs are those of a prefill of its whole text."""
import numpy as np
import pytest

import decode_ref as R
from decode_ref import D, DeviceTable, Table, ints, pointers
from gpu_helpers import dev, empty, get, get_bf16, say, stream
from qwen3_5_native import hip

pytestmark = pytest.mark.gpu
EPS = 1e-6
HQ, HK, DH, HALF = 16, 4, 256, 32   # the attention layer
GH, GK = 4, 2                       # the delta-rule layer
PAGE, NSEQ = 16, 6


def test_prompt_fork_and_tokens_in_a_graph():
    say("decode: prompt, fork, tokens in a graph")
    api, s = hip.api(), stream()
    st = s.handle
    rng = np.random.default_rng(0)
    prompt, steps, kids = 75, 7, [4, 1, 5]
    scale = DH ** -0.5
    # attention layer rows: per q head (q | gate), k, v; delta-rule rows: q | k | v | z | b | a
    ald = 2 * HQ * DH + 2 * HK * DH
    conv = (2 * GK + GH) * D
    gld = conv + GH * D + 2 * GH
    n = prompt + steps
    arow = {c: R.bf16(rng, n, ald) for c in kids}
    grow = {c: R.bf16(rng, n, gld) for c in kids}
    for c in kids[1:]:
        arow[c][:prompt], grow[c][:prompt] = arow[kids[0]][:prompt], grow[kids[0]][:prompt]
    qw, kw = R.bf16(rng, DH, std=0.1), R.bf16(rng, DH, std=0.1)
    ang = np.arange(n)[:, None] / 1e7 ** (np.arange(HALF) / HALF)
    cos, sin = (R.O.f32_to_bf16(f(ang).astype(np.float32)).reshape(n, HALF) for f in (np.cos, np.sin))
    cw, gw = R.bf16(rng, conv, 4, std=0.3), R.O.f32_to_bf16((1 + 0.1 * rng.standard_normal(D)).astype(np.float32))
    al = R.O.f32_to_bf16(np.log(1 + 15 * rng.random(GH)).astype(np.float32))
    dt = R.O.f32_to_bf16(rng.uniform(-6, -2, GH).astype(np.float32))
    W = {k: dev(v) for k, v in dict(qw=qw, kw=kw, cw=cw, gw=gw, al=al, dt=dt).items()}

    def prep(x, rows, cb, sb):
        """q, gate, k of projected rows; V stays where it is."""
        q, g, k = empty(rows * HQ * DH * 2), empty(rows * HQ * DH * 2), empty(rows * HK * DH * 2)
        call = lambda: hip.check(api.cs1_attn_prep(  # noqa: E731
            x.at(0), x.at(4 * HQ * DH), ald, W["qw"].at(0), W["kw"].at(0), cb.at(0), sb.at(0), q.at(0), g.at(0), k.at(0), rows,
            HQ, HK, DH, HALF, EPS, st), "prep")
        call()
        return q, g, k, call

    def gdn_prefill(x, rows):
        q, k, v, o, ns = (empty(rows * w * D * 2) for w in (GK, GK, GH, GH, GH))
        ws, so = empty(api.cs1_gdn_workspace_floats(rows, GH) * 4), empty(GH * D * D * 4)
        hip.check(api.cs1_gdn_conv(x.at(0), gld, W["cw"].at(0), q.at(0), k.at(0), v.at(0), rows, GK * D, GH * D, st), "conv")
        zb = 2 * (conv + GH * D)
        hip.check(api.cs1_gdn_prefill_gated_x(q.at(0), k.at(0), v.at(0), x.at(zb), x.at(zb + 2 * GH), gld, W["al"].at(0),
                                              W["dt"].at(0), o.at(0), ws.at(0), rows, GH, GK, D ** -0.5, None, so.at(0), st), "prefill")
        hip.check(api.cs1_gated_rms_norm(o.at(0), x.at(2 * conv), gld, W["gw"].at(0), ns.at(0), rows, GH, D, EPS, st), "norm")
        s.sync()
        return get_bf16(ns, rows * GH * D).reshape(rows, GH, D), so

    # what a prefill of each whole text gives
    whole, gwhole = {}, {}
    for c in kids:
        x, cb, sb = dev(arow[c]), dev(cos), dev(sin)
        q, g, k, _ = prep(x, n, cb, sb)
        out = empty(n * HQ * DH * 2)
        hip.check(api.cs1_attention_gated(q.at(0), k.at(0), x.at(2 * (2 * HQ * DH + HK * DH)), ald, g.at(0), out.at(0), n, HQ, HK, DH,
                                          scale, st), "attention")
        whole[c] = R.f64(get_bf16(out, n * HQ * DH).reshape(n, HQ, DH))
        gwhole[c] = R.f64(gdn_prefill(dev(grow[c]), n)[0])

    # the cache, and the prompt as sequence 0
    t = Table(NSEQ, 8, 30, PAGE)
    d = DeviceTable(t)
    pools = [dev(np.full((t.npages, PAGE, HK * DH), 0x7fc0, np.uint16)) for _ in range(2)]
    states, rings = dev(np.full(NSEQ * GH * D * D, np.nan, np.float32)), dev(np.full(NSEQ * 4 * conv, 0x7fc0, np.uint16))
    status, ws = ints([9]), empty(api.cs1_kv_workspace_bytes(t.npages, NSEQ))
    zero, cu = ints([0]), np.array([0, prompt], np.int32)
    x, cb, sb = dev(arow[kids[0]][:prompt]), dev(cos[:prompt]), dev(sin[:prompt])
    q, g, k, _ = prep(x, prompt, cb, sb)
    hip.check(api.cs1_kv_reserve(d.ref, zero.at(0), cu.ctypes.data, 1, status.at(0), st), "reserve")
    hip.check(api.cs1_kv_write(d.ref, zero.at(0), cu.ctypes.data, 1, k.at(0), HK * DH, x.at(2 * (2 * HQ * DH + HK * DH)), ald,
                               pools[0].at(0), pools[1].at(0), HK, DH, st), "write")
    t.reserve([0], cu)
    _, so = gdn_prefill(dev(grow[kids[0]][:prompt]), prompt)
    hip.check(api.cs1_copy_dd(states.at(0), so.at(0), GH * D * D * 4, st), "state")
    for i in range(prompt - 3, prompt):
        hip.upload(rings, grow[kids[0]][i, :conv], s, offset=(i % 4) * conv * 2)

    # fork: pages by their counts, states and rings as entries
    src, dst = ints([0] * len(kids)), ints(kids)
    ptrs = pointers(pools)
    hip.check(api.cs1_kv_fork(d.ref, src.at(0), dst.at(0), len(kids), ptrs, 2, 2 * HK * DH, ws.at(0), status.at(0), st), "fork")
    for buf, size in ((states, GH * D * D * 4), (rings, 4 * conv * 2)):
        one = pointers([buf])
        hip.check(api.cs1_kv_copy(one, 1, size, NSEQ, src.at(0), dst.at(0), len(kids), st), "copy")
    t.fork([0] * len(kids), kids, [])
    d.check()

    # one step of the batch, two rows of it padding, recorded once
    rows = kids + [-1, NSEQ]
    B = len(rows)
    seqs, handle = ints(rows), api.cs1_attention_paged_create()
    ax, gx = dev(np.zeros((B, ald), np.uint16)), dev(np.zeros((B, gld), np.uint16))
    ac, asn = dev(np.zeros((B, HALF), np.uint16)), dev(np.zeros((B, HALF), np.uint16))
    q, g, k, prep_step = prep(ax, B, ac, asn)
    out, gout = empty(B * HQ * DH * 2), empty(B * GH * D * 2)

    def step():
        hip.check(api.cs1_kv_reserve(d.ref, seqs.at(0), None, B, status.at(0), st), "reserve")
        prep_step()
        hip.check(api.cs1_kv_write(d.ref, seqs.at(0), None, B, k.at(0), HK * DH, ax.at(2 * (2 * HQ * DH + HK * DH)), ald,
                                   pools[0].at(0), pools[1].at(0), HK, DH, st), "write")
        hip.check(api.cs1_attention_paged(handle, q.at(0), pools[0].at(0), pools[1].at(0), d.ref, seqs.at(0), g.at(0), out.at(0),
                                          None, B, HQ, HK, DH, scale, st), "attention")
        zb = 2 * (conv + GH * D)
        hip.check(api.cs1_gdn_decode(gx.at(0), gld, W["cw"].at(0), gx.at(2 * conv), gx.at(zb), gx.at(zb + 2 * GH), W["al"].at(0),
                                     W["dt"].at(0), W["gw"].at(0), EPS, rings.at(0), states.at(0), seqs.at(0), d.lens.at(0), NSEQ,
                                     gout.at(0), B, GH, GK, D ** -0.5, st), "gdn")

    graph = hip.Graph(s, step)
    worst = gworst = 0.0
    for i in range(prompt, n):
        for buf, rows_of, ld in ((ax, arow, ald), (gx, grow, gld)):
            a = np.zeros((B, ld), np.uint16)
            for r, c in enumerate(kids):
                a[r] = rows_of[c][i]
            hip.upload(buf, a, s)
        hip.upload(ac, np.repeat(cos[i:i + 1], B, 0), s)
        hip.upload(asn, np.repeat(sin[i:i + 1], B, 0), s)
        graph.launch(s)
        assert get(status, np.int32, 1)[0] == 0
        t.reserve(rows)
        d.check()
        o, go = get_bf16(out, B * HQ * DH).reshape(B, HQ, DH), get_bf16(gout, B * GH * D).reshape(B, GH, D)
        assert (o[len(kids):] == 0).all() and (go[len(kids):] == 0).all()
        for r, c in enumerate(kids):
            worst = max(worst, np.abs(R.f64(o[r]) - whole[c][i]).max() / np.abs(whole[c][i]).max())
            gworst = max(gworst, np.linalg.norm(R.f64(go[r]) - gwhole[c][i]) / np.linalg.norm(gwhole[c][i]))
    print(f"  attention {worst:.4f} of the largest value, delta rule {gworst:.4f}", flush=True)
    # the prefill rounds its probabilities, the attention and the gate: half a step each of values no larger than the largest
    assert worst <= 4 * R.E16
    # and q, k, v, beta, the chunks' operands (four products), o and two factors of the norm
    assert gworst <= 12 * R.E16

    # the continuations end, their pages are free again and the prompt's move to the front
    hip.check(api.cs1_kv_free(d.ref, seqs.at(0), B, st), "free")
    t.free(rows)
    hip.check(api.cs1_kv_compact(d.ref, ptrs, 2, 2 * HK * DH, ws.at(0), status.at(0), st), "compact")
    t.compact([])
    d.check()
    assert (t.refs > 0).sum() == R.cdiv(prompt, PAGE)
    api.cs1_attention_paged_destroy(handle)


def test_ragged_sequences_step_by_step():
    """Sequences of five lengths in one batch, each row with the rotary rows of its own position.  The room for a step is
    reserved before its graph is replayed and the status read, since a step without room must not run.  Every step is held
    against float64 on what the device held before it, within float32's bounds."""
    say("decode: ragged positions, reserve in front of the graph")
    api, s = hip.api(), stream()
    st = s.handle
    rng = np.random.default_rng(1)
    prompts, steps = {3: 75, 0: 1, 5: 16, 1: 130, 4: 33}, 6
    rows = [4, -1, 0, 5, NSEQ, 3, 1]
    B, scale = len(rows), DH ** -0.5
    ald = 2 * HQ * DH + 2 * HK * DH
    conv = (2 * GK + GH) * D
    gld = conv + GH * D + 2 * GH
    longest = max(prompts.values()) + steps
    arow = {c: R.bf16(rng, n + steps, ald) for c, n in prompts.items()}
    grow = {c: R.bf16(rng, n + steps, gld) for c, n in prompts.items()}
    qw, kw = R.bf16(rng, DH, std=0.1), R.bf16(rng, DH, std=0.1)
    ang = np.arange(longest)[:, None] / 1e7 ** (np.arange(HALF) / HALF)
    cos, sin = (R.O.f32_to_bf16(f(ang).astype(np.float32)).reshape(longest, HALF) for f in (np.cos, np.sin))
    cw, gw = R.bf16(rng, conv, 4, std=0.3), R.O.f32_to_bf16((1 + 0.1 * rng.standard_normal(D)).astype(np.float32))
    al = R.O.f32_to_bf16(np.log(1 + 15 * rng.random(GH)).astype(np.float32))
    dt = R.O.f32_to_bf16(rng.uniform(-6, -2, GH).astype(np.float32))
    W = {k: dev(v) for k, v in dict(qw=qw, kw=kw, cw=cw, gw=gw, al=al, dt=dt).items()}
    v_at = 2 * (2 * HQ * DH + HK * DH)

    def prep_call(x, n, cb, sb, q, g, k):
        hip.check(api.cs1_attn_prep(x.at(0), x.at(4 * HQ * DH), ald, W["qw"].at(0), W["kw"].at(0), cb.at(0), sb.at(0), q.at(0),
                                    g.at(0), k.at(0), n, HQ, HK, DH, HALF, EPS, st), "prep")

    t = Table(NSEQ, 12, 40, PAGE)
    d = DeviceTable(t)
    host = [np.full((t.npages, PAGE, HK * DH), 0x7fc0, np.uint16) for _ in range(2)]
    pools = [dev(x) for x in host]
    state, ring = np.full((NSEQ, GH, D, D), np.nan, np.float32), np.full((NSEQ, 4, conv), 0x7fc0, np.uint16)
    states, rings = dev(state), dev(ring)
    status = ints([9])
    qs, gs, ks = {}, {}, {}

    def reserved():
        s.sync()
        return int(get(status, np.int32, 1)[0])

    # the prompts: their keys and values into pages, their states and last rows into slots
    for c, n in prompts.items():
        x, cb, sb = dev(arow[c]), dev(cos[:n + steps]), dev(sin[:n + steps])
        m = n + steps
        q, g, k = empty(m * HQ * DH * 2), empty(m * HQ * DH * 2), empty(m * HK * DH * 2)
        prep_call(x, m, cb, sb, q, g, k)
        qs[c], gs[c] = (get_bf16(b, m * HQ * DH).reshape(m, HQ, DH) for b in (q, g))
        ks[c] = get_bf16(k, m * HK * DH).reshape(m, HK * DH)
        one, cu = ints([c]), np.array([0, n], np.int32)
        hip.check(api.cs1_kv_reserve(d.ref, one.at(0), cu.ctypes.data, 1, status.at(0), st), "reserve")
        assert reserved() == t.reserve([c], cu) == 0
        hip.check(api.cs1_kv_write(d.ref, one.at(0), cu.ctypes.data, 1, k.at(0), HK * DH, x.at(v_at), ald, pools[0].at(0),
                                   pools[1].at(0), HK, DH, st), "write")
        t.write([c], cu, ks[c][:n], arow[c][:n, v_at // 2:v_at // 2 + HK * DH], *host)
        gx = dev(grow[c][:n])
        gq, gk, gv, o = (empty(n * w * D * 2) for w in (GK, GK, GH, GH))
        ws = empty(api.cs1_gdn_workspace_floats(n, GH) * 4)
        zb = 2 * (conv + GH * D)
        hip.check(api.cs1_gdn_conv(gx.at(0), gld, W["cw"].at(0), gq.at(0), gk.at(0), gv.at(0), n, GK * D, GH * D, st), "conv")
        hip.check(api.cs1_gdn_prefill_gated_x(gq.at(0), gk.at(0), gv.at(0), gx.at(zb), gx.at(zb + 2 * GH), gld, W["al"].at(0),
                                              W["dt"].at(0), o.at(0), ws.at(0), n, GH, GK, D ** -0.5, None,
                                              states.at(c * GH * D * D * 4), st), "prefill")
        for i in range(max(0, n - 4), n):  # on the device, from the projection's rows
            hip.check(api.cs1_copy_dd(rings.at((c * 4 + i % 4) * conv * 2), gx.at(i * gld * 2), conv * 2, st), "ring")
        s.sync()
    d.check()

    seqs, handle = ints(rows), api.cs1_attention_paged_create()
    ax, gx = dev(np.zeros((B, ald), np.uint16)), dev(np.zeros((B, gld), np.uint16))
    ac, asn = dev(np.zeros((B, HALF), np.uint16)), dev(np.zeros((B, HALF), np.uint16))
    q, g, k = empty(B * HQ * DH * 2), empty(B * HQ * DH * 2), empty(B * HK * DH * 2)
    out, gout = empty(B * HQ * DH * 2), empty(B * GH * D * 2)
    lse = empty(HQ * B * 4)

    def step():
        prep_call(ax, B, ac, asn, q, g, k)
        hip.check(api.cs1_kv_write(d.ref, seqs.at(0), None, B, k.at(0), HK * DH, ax.at(v_at), ald, pools[0].at(0),
                                   pools[1].at(0), HK, DH, st), "write")
        hip.check(api.cs1_attention_paged(handle, q.at(0), pools[0].at(0), pools[1].at(0), d.ref, seqs.at(0), g.at(0), out.at(0),
                                          lse.at(0), B, HQ, HK, DH, scale, st), "attention")
        zb = 2 * (conv + GH * D)
        hip.check(api.cs1_gdn_decode(gx.at(0), gld, W["cw"].at(0), gx.at(2 * conv), gx.at(zb), gx.at(zb + 2 * GH), W["al"].at(0),
                                     W["dt"].at(0), W["gw"].at(0), EPS, rings.at(0), states.at(0), seqs.at(0), d.lens.at(0), NSEQ,
                                     gout.at(0), B, GH, GK, D ** -0.5, st), "gdn")

    graph = hip.Graph(s, step)
    for i in range(steps):
        if i == 3:  # one ends, and its row is padding from here on
            gone = ints([5])
            hip.check(api.cs1_kv_free(d.ref, gone.at(0), 1, st), "free")
            t.free([5])
            rows[rows.index(5)] = -1
            hip.upload(seqs, np.array(rows, np.int32), s)
        live = [(r, c, prompts[c] + i) for r, c in enumerate(rows) if 0 <= c < NSEQ]  # row, sequence, position
        a, x = np.full((B, ald), 0x7fc0, np.uint16), np.full((B, gld), 0x7fc0, np.uint16)
        cs, sn = np.zeros((B, HALF), np.uint16), np.zeros((B, HALF), np.uint16)
        for r, c, p in live:
            a[r], x[r], cs[r], sn[r] = arow[c][p], grow[c][p], cos[p], sin[p]
        for buf, arr in ((ax, a), (gx, x), (ac, cs), (asn, sn)):
            hip.upload(buf, arr, s)
        hip.check(api.cs1_kv_reserve(d.ref, seqs.at(0), None, B, status.at(0), st), "reserve")
        assert reserved() == t.reserve(rows) == 0
        state = get(states, np.float32, state.size).reshape(state.shape)
        ring = get_bf16(rings, ring.size).reshape(ring.shape)
        graph.launch(s)
        qi, gi, ki = np.zeros((B, HQ, DH), np.uint16), np.zeros((B, HQ, DH), np.uint16), np.zeros((B, HK * DH), np.uint16)
        for r, c, p in live:
            assert int(t.lens[c]) == p + 1
            qi[r], gi[r], ki[r] = qs[c][p], gs[c][p], ks[c][p]
        t.write(rows, None, ki, a[:, v_at // 2:v_at // 2 + HK * DH], *host)
        for buf, arr in zip(pools, host):
            np.testing.assert_array_equal(R.read_pool(buf, arr), arr)
        want, wl, tol, ltol = R.attention(t, rows, qi, *host, gi, HK, scale)
        R.close(R.f64(get_bf16(out, B * HQ * DH).reshape(B, HQ, DH)), want, tol, f"step {i} attention")
        R.close(get(lse, np.float32, HQ * B).reshape(HQ, B).astype(np.float64), wl, ltol, f"step {i} lse")
        want, S, ring2, tol, stol = R.gdn_step(x, cw, al, dt, gw, ring, state, rows, t.lens, GH, GK, D ** -0.5, EPS)
        R.close(R.f64(get_bf16(gout, B * GH * D).reshape(B, GH, D)), want, tol, f"step {i} delta rule")
        R.close(get(states, np.float32, state.size).reshape(state.shape).astype(np.float64), S, stol, f"step {i} state")
        np.testing.assert_array_equal(get_bf16(rings, ring.size).reshape(ring.shape), ring2)
    d.check()
    api.cs1_attention_paged_destroy(handle)
