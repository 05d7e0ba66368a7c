"""Plain implementations of the operations on several new tokens of a sequence, for their tests: room, positions and
slots, tokens taken back, attention inputs with rotary positions, attention of a batch's rows.  Nothing here comes from the library."""
import numpy as np

from decode_ref import E16, E32, cdiv, f64


def extend(t, seqs, cu):
    """Table.reserve where the offsets may fall: such an entry has no tokens."""
    return t.reserve(seqs, np.concatenate([[0], np.cumsum(np.maximum(np.diff(np.asarray(cu, np.int64)), 0))]))


def rows_of(t, seqs, cu, rows):
    """pos and slot of every row."""
    pos, slot = np.full(rows, -1, np.int64), np.full(rows, -1, np.int64)
    for i, s in t.listed(seqs):
        for r in range(int(cu[i]), min(rows, int(cu[i + 1]))):
            p = int(t.lens[s]) - (int(cu[i + 1]) - r)
            if 0 <= p < t.max_pages * t.page:
                pos[r] = p
                pg = int(t.table[s, p // t.page])
                if 0 <= pg < t.npages:
                    slot[r] = pg * t.page + p % t.page
    return pos.astype(np.int32), slot.astype(np.int32)


def trim(t, seqs, drop):
    """How many listed sequences stay as they are, since others hold the page that would be cut."""
    left, todo = 0, []
    for i, s in t.listed(seqs):
        n = int(t.lens[s])
        to = max(0, n - max(0, int(drop[i])))
        if to == n:
            continue
        p = int(t.table[s, to // t.page]) if to % t.page else -1
        if 0 <= p < t.npages and t.refs[p] > 1:
            left += 1
        else:
            todo.append((s, n, to))
    for s, n, to in todo:
        for j in range(cdiv(to, t.page), cdiv(n, t.page)):
            p = int(t.table[s, j])
            if 0 <= p < t.npages:
                t.refs[p] -= 1
            t.table[s, j] = -1
        t.lens[s] = to
    return left


def turned(x, w, eps, pos, freqs, dims, interleaved, magnitude):
    """Heads x [rows, heads, dh] (float64 of bfloat16) normed and turned, in float64, and the bound on a float32
    computation's error with one rounding to bfloat16.

    A sum of dh squares in any order is off by dh E32 of itself and a step each, the root halves that, and the root's
    reciprocal, the quotient, 1 + w and two products add a step of 2 E32 each: (dh / 2 + 12) E32 and another 2 E32.  An
    angle is its turns less the whole ones, exact but for float64's rounding of p f / 2 pi (2^-52 of it, in the test as in
    the kernel), rounded to float32 as up to one half turn's double (E32 of 1, that is pi E32 radians); a sine or cosine is
    good to two steps (4 E32), its product with the magnitude to one."""
    rows, heads, dh = x.shape
    y, rel = x, 0.0
    if w is not None:
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1 + w)
        rel = (dh / 2 + 14) * E32
    out, tol = y.copy(), rel * np.abs(y)
    if dims:
        h = dims // 2
        angle = pos.astype(np.float64)[:, None] * freqs[None, :]
        c, s = np.cos(angle)[:, None, :] * magnitude, np.sin(angle)[:, None, :] * magnitude
        off = ((np.pi + 8) * E32 + np.abs(angle)[:, None, :] * 2.0 ** -50) * magnitude
        a, b = (np.s_[..., 0:dims:2], np.s_[..., 1:dims:2]) if interleaved else (np.s_[..., :h], np.s_[..., h:dims])
        ya, yb = y[a], y[b]
        out[a], out[b] = ya * c - yb * s, yb * c + ya * s
        size = np.abs(ya) + np.abs(yb)
        tol[a] = tol[b] = size * (rel * magnitude + off + 4 * E32 * magnitude)
    return out, tol + E16 * (np.abs(out) + tol)


def attention(t, seqs, cu, rows, max_new, q, kp, vp, gate, hk, scale):
    """Float64 result, log-sum-exp, the bounds on the error of each, and which rows are someone's.

    As decode_ref.attention, but for the probabilities, which are rounded to bfloat16 for the second product (E16 of each
    weight there, and not in their sum)."""
    _, hq, dh = q.shape
    rep = hq // hk
    out, lse = np.zeros((rows, hq, dh)), np.full((hq, rows), -np.inf)
    tol, ltol = np.zeros((rows, hq, dh)), np.zeros((hq, rows))
    ours = np.zeros(rows, bool)
    for i, s in enumerate(seqs):
        lo, hi = int(cu[i]), int(cu[i + 1])
        L = min(hi - lo, max_new)
        ours[lo:lo + L] = True
        n = min(int(t.lens[s]), t.max_pages * t.page) if 0 <= s < t.nseq else 0
        if L <= 0 or n == 0:
            continue
        j = np.arange(n)
        pg = t.table[s, j // t.page]
        there = (pg >= 0) & (pg < t.npages)
        j = j[there]
        if not len(j):
            continue
        K, V = f64(kp[pg[there], j % t.page]), f64(vp[pg[there], j % t.page])
        sees = j[None, :] <= (n - (hi - lo) + np.arange(L))[:, None]
        some = sees.any(1)
        for h in range(hq):
            k, v, x = K[:, h // rep], V[:, h // rep], f64(np.ascontiguousarray(q[lo:lo + L, h]))
            sc = np.where(sees, (x @ k.T) * scale, -np.inf)
            top = np.where(some, np.max(sc, 1, initial=-np.inf), 0.0)[:, None]
            off = (dh + 2) * E32 * (np.abs(x) @ np.abs(k).T) * abs(scale) + 4 * E32 * np.abs(np.where(sees, sc, 0))
            w = np.exp(sc - top)
            z = w.sum(1, keepdims=True)
            p = w / np.where(z > 0, z, 1)
            o = p @ v
            rel = 2 * (off + np.where(sees, off, 0).max(1, keepdims=True)) + 4 * E32 + 2 * n * E32
            f = 1.0
            if gate is not None:
                f = 1 / (1 + np.exp(-f64(np.ascontiguousarray(gate[lo:lo + L, h]))))
            mean = (p * rel).sum(1, keepdims=True)
            err = (p * (rel + E16)) @ np.abs(v) + np.abs(o) * mean + 16 * E32 * np.abs(o)
            out[lo:lo + L, h] = o * f
            tol[lo:lo + L, h] = err * f + E16 * (np.abs(o * f) + err * f)
            with np.errstate(divide="ignore"):
                lse[h, lo:lo + L] = np.where(some, top[:, 0] + np.log(z[:, 0]), -np.inf)
            size = np.where(some, np.abs(np.where(some, lse[h, lo:lo + L], 0)), 0)
            ltol[h, lo:lo + L] = mean[:, 0] + 8 * E32 * (1 + size + np.log(max(n, 2)))
    return out, lse, tol, ltol, ours
