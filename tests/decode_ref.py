"""Plain implementations of the decode operations for their tests: the page table as lists of whole
numbers, attention of one token and the delta rule's step in float64 with bounds on what float32 arithmetic
may be off by.  Nothing here comes from the library."""
import ctypes

import numpy as np

import oracle as O
from gpu_helpers import dev, empty, get, stream
from qwen3_5_native import hip

E32 = 2.0 ** -24  # half a step of float32, relative to the value
E16 = 2.0 ** -8   # of bfloat16
D = 128


def bf16(rng, *shape, std=1.0):
    """Normal values as bfloat16 patterns (uint16)."""
    return O.f32_to_bf16((rng.standard_normal(int(np.prod(shape))) * std).astype(np.float32)).reshape(shape)


def f64(u16):
    return O.bf16_to_f32(np.ascontiguousarray(u16).reshape(-1)).astype(np.float64).reshape(u16.shape)


def cdiv(a, b):
    return -(-a // b)


# ---------------------------------------------------------------- the page table

class Table:
    """The bookkeeping of Cs1PageTable, step by step as the header says it."""

    def __init__(self, nseq, max_pages, npages, page):
        self.nseq, self.max_pages, self.npages, self.page = nseq, max_pages, npages, page
        self.table = np.full((nseq, max_pages), -1, np.int32)
        self.lens = np.zeros(nseq, np.int32)
        self.refs = np.zeros(npages, np.int32)

    def listed(self, seqs):
        """(entry, sequence) of the entries that are no padding; the first that names a sequence has it."""
        seen = set()
        for i, s in enumerate(seqs):
            if 0 <= s < self.nseq and s not in seen:
                seen.add(s)
                yield i, int(s)

    def free_pages(self):
        return [p for p in range(self.npages) if self.refs[p] == 0]

    def reserve(self, seqs, cu=None):
        add = [1] * len(seqs) if cu is None else np.diff(cu).tolist()
        todo = [(s, int(self.lens[s]), add[i]) for i, s in self.listed(seqs)]
        if any(n + k > self.max_pages * self.page for _, n, k in todo):
            return -1
        need = [cdiv(n + k, self.page) - cdiv(n, self.page) for _, n, k in todo]
        free = self.free_pages()
        if sum(need) > len(free):
            return sum(need) - len(free)
        for (s, n, k), m in zip(todo, need):
            for j in range(m):
                p = free.pop(0)
                self.table[s, cdiv(n, self.page) + j] = p
                self.refs[p] = 1
            self.lens[s] += k
        return 0

    def write(self, seqs, cu, k, v, kp, vp):
        """k, v: rows; kp, vp: [npages, page, width] arrays that receive them."""
        for i, s in self.listed(seqs):
            lo, hi = (i, i + 1) if cu is None else (int(cu[i]), int(cu[i + 1]))
            for r in range(lo, hi):
                pos = int(self.lens[s]) - (hi - r)
                if pos < 0:
                    continue
                p = int(self.table[s, pos // self.page])
                if 0 <= p < self.npages:
                    kp[p, pos % self.page], vp[p, pos % self.page] = k[r], v[r]

    def pairs(self, src, dst, n):
        """The pairs of entries below n that are carried out."""
        named = [int(d) for d in dst if 0 <= d < n]
        seen = set()
        for s, d in zip(src, dst):
            s, d = int(s), int(d)
            first = d not in seen
            if 0 <= d < n:
                seen.add(d)
            if 0 <= s < n and 0 <= d < n and first and s not in named:
                yield s, d

    def fork(self, src, dst, pools):
        todo = [(s, d) for s, d in self.pairs(src, dst, self.nseq) if self.lens[d] == 0 and self.lens[s] > 0]
        free = self.free_pages()
        need = sum(int(self.lens[s]) % self.page > 0 for s, _ in todo)
        if need > len(free):
            return need - len(free)
        for s, d in todo:
            full, part = divmod(int(self.lens[s]), self.page)
            self.table[d, :full] = self.table[s, :full]
            for p in self.table[s, :full]:
                self.refs[p] += 1
            if part:
                p, old = free.pop(0), self.table[s, full]
                self.table[d, full] = p
                self.refs[p] = 1
                for pool in pools:
                    pool[p, :part] = pool[old, :part]
            self.lens[d] = self.lens[s]
        return 0

    def free(self, seqs):
        for _, s in self.listed(seqs):
            for p in self.table[s, :cdiv(int(self.lens[s]), self.page)]:
                self.refs[p] -= 1
            self.table[s] = -1
            self.lens[s] = 0

    def compact(self, pools):
        held = np.flatnonzero(self.refs)
        L = len(held)
        moves = dict(zip(held[held >= L].tolist(), np.flatnonzero(self.refs[:L] == 0).tolist()))
        for a, b in moves.items():
            for pool in pools:
                pool[b] = pool[a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        for s in range(self.nseq):
            for j in range(cdiv(int(self.lens[s]), self.page)):
                self.table[s, j] = moves.get(int(self.table[s, j]), self.table[s, j])
        return L


class DeviceTable:
    """A Table's arrays on the device and the struct that names them."""

    def __init__(self, t):
        self.t = t
        self.table, self.lens, self.refs = dev(t.table), dev(t.lens), dev(t.refs)
        self.struct = hip.PageTable(self.table.at(0), self.lens.at(0), self.refs.at(0), t.nseq, t.max_pages, t.npages,
                                    t.page)
        self.ref = ctypes.byref(self.struct)

    def state(self):
        t = self.t
        return (get(self.table, np.int32, t.nseq * t.max_pages).reshape(t.nseq, t.max_pages),
                get(self.lens, np.int32, t.nseq), get(self.refs, np.int32, t.npages))

    def check(self):
        for name, got, want in zip(("table", "lens", "refs"), self.state(), (self.t.table, self.t.lens, self.t.refs)):
            np.testing.assert_array_equal(got, want, err_msg=name)


def ints(values):
    return dev(np.asarray(values, np.int32))


def pointers(bufs):
    return (ctypes.c_void_p * max(1, len(bufs)))(*[b.at(0) for b in bufs])


def scattered(rng, nseq, lens, page, max_pages=None, spare=3):
    """A Table whose sequences 0 .. len(lens) - 1 hold lens tokens on pages in random order."""
    need = [cdiv(n, page) for n in lens]
    t = Table(nseq, max_pages or max(need + [1]) + 1, sum(need) + spare, page)
    order = rng.permutation(t.npages)
    at = 0
    for s, (n, k) in enumerate(zip(lens, need)):
        t.table[s, :k] = order[at:at + k]
        t.refs[order[at:at + k]] = 1
        t.lens[s] = n
        at += k
    return t


# ---------------------------------------------------------------- attention of one token

def attention(t, seqs, q, kp, vp, gate, hk, scale):
    """Float64 result, log-sum-exp, and the bounds on a float32 computation's error of each.

    A score is a sum of Dh products of bfloat16 values, each exact in float32, so a float32 sum in any order is
    off by at most Dh E32 sum |q k|; it is scaled (E32) and taken to an exponential of base 2, whose argument
    carries two more roundings of |S| and whose value one of a step (2 E32).  The probability's weight goes to the product in two
    bfloat16 parts: eight bits cut off, which leaves less than 2 E16 of it, and that rest rounded: 2 E16^2 of the weight.  The sums over n keys add n E32 each at most."""
    B, hq, dh = q.shape
    out, lse = np.zeros((B, hq, dh)), np.full((hq, B), -np.inf)
    tol, ltol = np.zeros((B, hq, dh)), np.zeros((hq, B))
    for r, s in enumerate(seqs):
        n = int(t.lens[s]) if 0 <= s < t.nseq else 0
        at = [(int(t.table[s, j // t.page]), j % t.page) for j in range(n)]
        at = [(p, j) for p, j in at if 0 <= p < t.npages]
        if not at:
            continue
        pg, sl = np.array([p for p, _ in at]), np.array([j for _, j in at])
        n = len(at)
        K, V = f64(kp[pg, sl].reshape(n, hk, dh)), f64(vp[pg, sl].reshape(n, hk, dh))
        for h in range(hq):
            x, k, v = f64(q[r, h]), K[:, h // (hq // hk)], V[:, h // (hq // hk)]
            sc = (k @ x) * scale
            off = (dh + 2) * E32 * (np.abs(k) @ np.abs(x)) * abs(scale) + 4 * E32 * np.abs(sc)
            w = np.exp(sc - sc.max())
            z = w.sum()
            p = w / z
            o = p @ v
            rel = 2 * (off + off.max()) + 4 * E32 + 2 * E16 * E16 + 2 * n * E32  # of each weight, and of their sum
            f = 1.0
            if gate is not None:
                f = 1 / (1 + np.exp(-f64(gate[r, h])))
            err = (p * rel) @ np.abs(v) + np.abs(o) * (p @ rel) + 16 * E32 * np.abs(o)
            out[r, h] = o * f
            lse[h, r] = sc.max() + np.log(z)
            tol[r, h] = err * f + E16 * (np.abs(o * f) + err * f)
            ltol[h, r] = p @ rel + 8 * E32 * (1 + abs(lse[h, r]) + np.log(max(n, 2)))
    return out, lse, tol, ltol


# ---------------------------------------------------------------- the delta rule's step

def gdn_step(x, w, a_log, dt_bias, gw, ring, state, seqs, lens, H, HK, scale, eps):
    """Float64 out, state, ring and the bounds on a float32 computation's error of out and state.

    Relative errors are counted in units u = 2^-23 of float32: a conv output has four products and sums and
    a SiLU (an exponential, a division: 16 u of sum |w x| with its slope at most 1.1), the norms of q and k 128 sums of
    squares (64 u after the root), a decay exp(g) the error of g times |g| (g: two exponentials and a logarithm, 16 u).
    What is under float32's normal range, 2^-126, may come out as zero: beta = 1 / (1 + e^-b) where e^-b passes the
    largest float32, 2^128, and then beta itself is under 2^-128; and products and outputs of that size."""
    u, tiny = 2 * E32, 2.0 ** -126
    conv = (2 * HK + H) * D
    B, grp = x.shape[0], H // HK
    nseq = len(lens)
    out, tol = np.zeros((B, H, D)), np.zeros((B, H, D))
    S2, ring2 = state.astype(np.float64), ring.copy()
    stol = np.zeros_like(S2)
    seen = set()
    W, dt, al = f64(w), f64(dt_bias), f64(a_log)
    for r in range(B):
        s = int(seqs[r])
        if not 0 <= s < nseq or s in seen:
            continue
        seen.add(s)
        p = int(lens[s]) - 1
        if p < 0:
            continue
        X = f64(x[r])
        y, mag = W[:, 3] * X[:conv], np.abs(W[:, 3] * X[:conv])
        for i in range(1, min(3, p) + 1):
            old = f64(ring[s, (p - i) % 4])
            y, mag = y + W[:, 3 - i] * old, mag + np.abs(W[:, 3 - i] * old)
        ey = 16 * u * mag
        y = y / (1 + np.exp(-y))
        qy, ky, v = y[:HK * D].reshape(HK, D), y[HK * D:2 * HK * D].reshape(HK, D), y[2 * HK * D:].reshape(H, D)
        eq, ek, ev = ey[:HK * D].reshape(HK, D), ey[HK * D:2 * HK * D].reshape(HK, D), ey[2 * HK * D:].reshape(H, D)

        def unit(a, e):
            n = np.sqrt((a * a).sum(-1, keepdims=True) + 1e-6)
            return a / n, e / n + np.abs(a) / n * (64 * u + (np.abs(a) * e).sum(-1, keepdims=True) / n ** 2)

        q, eq = unit(qy, eq)
        k, ek = unit(ky, ek)
        q, eq = q * scale, eq * abs(scale) + 2 * u * np.abs(q) * abs(scale)
        z = X[conv:conv + H * D].reshape(H, D)
        b, a = X[conv + H * D:conv + H * D + H], X[conv + H * D + H:conv + H * D + 2 * H]
        g = -np.exp(al) * np.logaddexp(0, a + dt)
        beta = 1 / (1 + np.exp(-b))
        for h in range(H):
            kk, qq, ekk, eqq = k[h // grp], q[h // grp], ek[h // grp], eq[h // grp]
            d = np.exp(g[h]) if p > 0 else 0.0
            ed = d * (16 * abs(g[h]) + 4) * u
            S = S2[s, h] if p > 0 else np.zeros((D, D))
            A = np.abs(S)
            kS = kk @ S * d
            ekS = (np.abs(kk) * (140 * u * d + ed) + ekk * d) @ A
            un = beta[h] * (v[h] - kS)
            eu = beta[h] * (ev[h] + ekS + 8 * u * (np.abs(v[h]) + np.abs(kS)))
            eu = eu + tiny * (np.abs(v[h]) + np.abs(kS) + 1)
            S1 = d * S + np.outer(kk, un)
            e1 = (ed + 2 * u * d) * A + np.outer(ekk, np.abs(un)) + np.outer(np.abs(kk), eu) + 2 * u * np.abs(np.outer(kk, un))
            qk, eqk = abs(qq @ kk), (eqq @ np.abs(kk) + np.abs(qq) @ ekk) + 140 * u * (np.abs(qq) @ np.abs(kk))
            o = qq @ S1
            eo = ((np.abs(qq) * (140 * u * d + ed) + eqq * d) @ A) + qk * eu + eqk * np.abs(un) + 4 * u * np.abs(o)
            if gw is not None:
                inv = 1 / np.sqrt((o * o).mean() + eps)
                f = f64(gw) * z[h] / (1 + np.exp(-z[h]))
                en = inv * (eo + np.abs(o) * ((np.abs(o) * eo).mean() * inv ** 2 + 80 * u))
                o, eo = o * inv * f, en * np.abs(f) + 8 * u * np.abs(o * inv * f)
            out[r, h], tol[r, h] = o, eo + E16 * (np.abs(o) + eo) + tiny
            S2[s, h], stol[s, h] = S1, e1 + 2 * u * np.abs(S1) + tiny
        ring2[s, p % 4] = x[r, :conv]
    return out, S2, ring2, tol, stol


def close(got, want, tol, what):
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        off = np.where(same, 0.0, np.abs(got - want))
    bad = ~(off <= tol)
    worst = np.max(off / np.where(tol > 0, tol, 1), initial=0.0)
    print(f"  {what}: worst {worst:.3f} of the bound", flush=True)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {worst:.3f} of the bound"


def pool_buffers(arrays):
    return [dev(a) for a in arrays]


def read_pool(buf, like):
    return get(buf, np.uint16, like.size).reshape(like.shape)


__all__ = [n for n in dir() if not n.startswith("_")] + ["empty", "stream"]
