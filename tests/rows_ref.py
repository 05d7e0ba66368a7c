"""Plain implementations of the operations on several new tokens of a sequence, for their tests: room, positions and
slots, tokens taken back, attention inputs with rotary positions.  Nothing here comes from the library."""
import numpy as np

from decode_ref import E16, E32, cdiv


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
