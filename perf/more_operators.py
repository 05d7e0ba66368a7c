"""Several new tokens of cached sequences at once, as measurable cases: the second turn of a chat, drafted
tokens to be verified, a long prompt taken in parts, candidates behind one prompt.  A step of such a
program makes room in the pages and maps its rows to places in them (slots), prepares queries, keys and
values with rotary positions and stores them there (prep), attends over the pages (chunk), and reads the
log-probabilities of the given tokens, the entropy and the best alternatives from the logits (logprobs).

Each case runs in a plain form made of elementary torch operations in 32 bits, or, where `own` is
true, through the library's operations as a serving program calls them.  Sizes are the repository's
own: 16 query over 4 key-value heads with head dim 128 or 256 (4B class) and 24 over 4 (27B class),
rotary positions on 64 of 256 dims with base 1e7, vocabularies of 151936 and 248320 tokens, contexts of
the prompt lengths up to 8192 and on to 32768 tokens.
"""
import ctypes
import math
import os
import sys

import numpy as np
import torch

own = False

BF = torch.bfloat16
F32 = torch.float32
F64 = torch.float64
EPS = 1e-6
BASE = 1e7  # of the rotary frequencies


def listed():
    return [
        # four drafted tokens of one user's chat are verified: the smallest call, latency counts
        {"name": "chunk-4-at-700", "kind": "chunk", "n": 1, "ctx_lo": 700, "ctx_hi": 700, "new_lo": 4, "new_hi": 4, "last": 0, "lens": 1,
         "hq": 16, "hk": 4, "dh": 128, "page": 16, "gate": True, "lse": True, "pad": 0},
        # drafted tokens of a server's whole batch in the 4B class, 43 ragged chats, the batch's last rows padding
        {"name": "chunk-43x4k", "kind": "chunk", "n": 43, "ctx_lo": 1, "ctx_hi": 4096, "new_lo": 1, "new_hi": 4, "last": 0, "lens": 2,
         "hq": 16, "hk": 4, "dh": 256, "page": 64, "gate": True, "lse": False, "pad": 11},
        # the second turn of a chat: 333 tokens behind 936
        {"name": "chunk-333-at-936", "kind": "chunk", "n": 1, "ctx_lo": 936, "ctx_hi": 936, "new_lo": 333, "new_hi": 333, "last": 0,
         "lens": 3, "hq": 16, "hk": 4, "dh": 256, "page": 64, "gate": True, "lse": False, "pad": 0},
        # a part of a long document's prompt rides along with the next tokens of 29 other users, heads of 128
        {"name": "chunk-mixed-29", "kind": "chunk", "n": 30, "ctx_lo": 100, "ctx_hi": 4096, "new_lo": 1, "new_hi": 1, "last": 1021,
         "lens": 4, "hq": 16, "hk": 4, "dh": 128, "page": 48, "gate": True, "lse": True, "pad": 0},
        # the last part of a long document in the 27B class, six query heads to a key-value head
        {"name": "chunk-2048-at-30k", "kind": "chunk", "n": 1, "ctx_lo": 30720, "ctx_hi": 30720, "new_lo": 2048, "new_hi": 2048, "last": 0,
         "lens": 5, "hq": 24, "hk": 4, "dh": 256, "page": 208, "gate": True, "lse": True, "pad": 0},
        # drafted tokens of one user: room in the pages, where the rows go, and all taken back
        {"name": "slots-1x4", "kind": "slots", "n": 1, "ctx_lo": 700, "ctx_hi": 700, "new_lo": 4, "new_hi": 4, "last": 0,
         "lens": 6, "page": 64, "pad": 0},
        # the rows of a large step: parts of prompts and drafts of 200 users
        {"name": "slots-200", "kind": "slots", "n": 200, "ctx_lo": 1, "ctx_hi": 8192, "new_lo": 1, "new_hi": 80, "last": 0,
         "lens": 7, "page": 16, "pad": 37},
        # a few drafted tokens through the 4B class's attention layer
        {"name": "prep-4", "kind": "prep", "rows": 4, "pad": 0, "at": 700, "hq": 16, "hk": 4, "dh": 256, "dims": 64, "inter": False,
         "factor": 1.0, "gate": True, "norm": True, "page": 64},
        # a prompt of 4096 tokens through it
        {"name": "prep-4096", "kind": "prep", "rows": 4096, "pad": 0, "at": 0, "hq": 16, "hk": 4, "dh": 256, "dims": 64,
         "inter": False, "factor": 1.0, "gate": True, "norm": True, "page": 64},
        # a layer without norms and gate that turns whole heads in neighbouring pairs, far into a context four times
        # as long as the one that its frequencies were made for
        {"name": "prep-1021-far", "kind": "prep", "rows": 1021, "pad": 3, "at": 120000, "hq": 32, "hk": 8, "dh": 128, "dims": 128,
         "inter": True, "factor": 4.0, "gate": False, "norm": False, "page": 16},
        # a user's next token with what else it could have been, in the 4B class
        {"name": "logprobs-1", "kind": "logprobs", "rows": 1, "vocab": 151936, "pad": 0, "k": 20, "f32": False, "std": 3.0},
        # candidate scoring in the 27B class: 1217 tokens of eight candidates
        {"name": "logprobs-1217", "kind": "logprobs", "rows": 1217, "vocab": 248320, "pad": 0, "k": 5, "f32": False, "std": 2.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["chunk", "chunk", "chunk", "slots", "prep", "prep", "logprobs", "logprobs"])
    c = {"kind": kind}
    if kind == "chunk":
        hq, hk, dh = rng.choice([(16, 4, 128), (16, 4, 256), (24, 4, 256), (8, 4, 128), (32, 8, 128), (16, 1, 256), (6, 2, 128)])
        n = rng.choice([1, 1, 2, _log_int(rng, 1, 48)])
        ctx = _log_int(rng, 1, min(30000, 120000 // n))
        new = _log_int(rng, 1, min(2048, 8192 // n))
        c.update(n=n, ctx_lo=rng.choice([0, 1 + ctx // 2, ctx]), ctx_hi=ctx, new_lo=rng.choice([1, new]), new_hi=new,
                 last=rng.choice([0, 0, 0, _log_int(rng, 1, 2048)]), lens=rng.randint(0, 1 << 20), hq=hq, hk=hk, dh=dh,
                 page=rng.choice([16, 32, 48, 64, 128, 208, 256]), gate=rng.random() < 0.7, lse=rng.random() < 0.5,
                 pad=rng.choice([0, 0, 1, 13]))
    elif kind == "slots":
        n = _log_int(rng, 1, 512)
        c.update(n=n, ctx_lo=0, ctx_hi=_log_int(rng, 1, 8192), new_lo=1, new_hi=_log_int(rng, 1, min(2048, 16384 // n)), last=0,
                 lens=rng.randint(0, 1 << 20), page=rng.choice([16, 48, 64, 128]), pad=rng.choice([0, 5]))
    elif kind == "prep":
        hq, hk, dh = rng.choice([(16, 4, 128), (16, 4, 256), (24, 4, 256), (32, 8, 128), (6, 2, 128)])
        c.update(rows=_log_int(rng, 1, 4096), pad=rng.choice([0, 0, 3]), at=_log_int(rng, 1, 500000), hq=hq, hk=hk, dh=dh,
                 dims=rng.choice([dh // 4, dh // 2, dh, 32]), inter=rng.random() < 0.5, factor=rng.choice([1.0, 1.0, 4.0, 16.0]),
                 gate=rng.random() < 0.6, norm=rng.random() < 0.6, page=rng.choice([16, 48, 64]))
    else:
        vocab = rng.choice([151936, 248320, _log_int(rng, 500, 250000)])
        f32 = rng.random() < 0.4
        c.update(rows=_log_int(rng, 1, min(2000, (150000000 if f32 else 300000000) // vocab)), vocab=vocab,
                 pad=rng.choice([0, 0, 1, 24]), k=rng.choice([0, 1, 5, 20, 32]), f32=f32, std=rng.choice([0.5, 2.0, 4.0]))
    return c


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=F32).mul_(std).to(BF)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _lengths(c):
    """Tokens that each sequence holds already and new ones, the same for every seed of the case (they are its work);
    `last`: new tokens of the last sequence, where it is not like the others."""
    rng = np.random.default_rng(c["lens"])
    ctx, new = (rng.integers(c[k + "_lo"], c[k + "_hi"] + 1, c["n"]) for k in ("ctx", "new"))
    if c["last"]:
        new[-1] = c["last"]
    return ctx, new


def _pages(n, page):
    return -(-n // page)


def _table(rng, nseq, lens, page, max_pages, spare):
    """lens {sequence: tokens} on pages in a random order; `spare` pages are free."""
    held = sum(_pages(int(n), page) for n in lens.values())
    order = rng.permutation(held + spare)
    table, n_of, refs = np.full((nseq, max_pages), -1, np.int32), np.zeros(nseq, np.int32), np.zeros(held + spare, np.int32)
    at = 0
    for s, n in lens.items():
        k = _pages(int(n), page)
        table[s, :k] = order[at:at + k]
        refs[order[at:at + k]] = 1
        n_of[s] = n
        at += k
    return table, n_of, refs


def _batch(c, seed, taken):
    """A batch's sequences in a random order with their offsets; `taken`: its new tokens are in the pages already."""
    rng = np.random.default_rng(seed)
    ctx, new = _lengths(c)
    n, page = len(ctx), c["page"]
    ids = rng.permutation(n + 3)[:n]
    most = int((ctx + new).max())
    table, lens, refs = _table(rng, n + 3, dict(zip(ids.tolist(), ctx + new if taken else ctx)), page, _pages(most, page) + 1,
                               2 + (0 if taken else int(sum(_pages(int(x), page) + 1 for x in new))))
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return {"seqs": _ints(ids), "cu": _ints(cu), "new": _ints(new), "table": _ints(table), "lens": _ints(lens),
            "refs": _ints(refs), "rows": int(cu[-1]) + c["pad"], "host_cu": cu, "host_seqs": ids, "host_len": ctx + new,
            "host_table": table}


def _chunk_inputs(c, seed):
    g = _gen(seed)
    s = _batch(c, seed, True)
    s["q"] = _randn(g, s["rows"], c["hq"], c["dh"])
    s["gate"] = _randn(g, s["rows"], c["hq"], c["dh"]) if c["gate"] else None
    s["kp"] = _randn(g, s["refs"].numel(), c["page"], c["hk"], c["dh"])
    s["vp"] = _randn(g, s["refs"].numel(), c["page"], c["hk"], c["dh"])
    return s


def _slots_inputs(c, seed):
    return _batch(c, seed, False)


def _freqs(dims, factor):
    """Turns of each pair of dims by one token, in radians.  With a factor, pairs that turn less than once in the 32768
    tokens that the frequencies were made for are slowed down by it, those that turn 32 times are left as they are, and
    those between are in between."""
    f = BASE ** (-np.arange(0, dims, 2, dtype=np.float64) / dims)
    if factor == 1.0:
        return f
    keep = np.clip((32768 * f / (2 * math.pi) - 1.0) / (32.0 - 1.0), 0.0, 1.0)
    return f * keep + f / factor * (1 - keep)


def _prep_inputs(c, seed):
    # a row is what the layer's input projection writes: q and gate head by head, then k, then v
    g = _gen(seed)
    rng = np.random.default_rng(seed)
    hq, hk, dh, page = c["hq"], c["hk"], c["dh"], c["page"]
    T = c["rows"] + c["pad"]
    npages = _pages(c["rows"], page) + 2
    s = {"x": _randn(g, T, (hq * (2 if c["gate"] else 1) + 2 * hk) * dh)}
    s["qw"], s["kw"] = (_randn(g, dh, std=0.1) if c["norm"] else None for _ in range(2))
    # two sequences share the rows: their last rows are at positions at + 1, at + 2, ..; pages in a random order
    half = c["rows"] // 2
    pos = np.full(T, -1, np.int32)
    pos[:half] = c["at"] + np.arange(half)
    pos[half:c["rows"]] = c["at"] // 3 + np.arange(c["rows"] - half)
    slot = np.full(T, -1, np.int32)
    order = rng.permutation(npages)
    at = np.arange(c["rows"])
    slot[:c["rows"]] = order[at // page] * page + at % page
    s["pos"], s["slot"] = _ints(pos), _ints(slot)
    s["freqs"] = torch.from_numpy(_freqs(c["dims"], c["factor"])).cuda()
    s["magnitude"] = float(np.float32(0.1 * math.log(c["factor"]) + 1.0))
    s["kp"], s["vp"] = (torch.zeros(npages, page, hk, dh, dtype=BF, device="cuda") for _ in range(2))
    return s


def _logprobs_inputs(c, seed):
    # rows of logits as an LM head leaves them, behind each other in rows of the vocabulary and some padding; the given
    # token is the best or a good one in half of the rows, any one in the others
    g = _gen(seed)
    R, V = c["rows"], c["vocab"]
    dt = F32 if c["f32"] else BF
    logits = torch.empty(R, V + c["pad"], dtype=dt, device="cuda")
    for i in range(0, R, 256):
        logits[i:i + 256] = torch.randn(min(256, R - i), V + c["pad"], generator=g, device="cuda").mul_(c["std"])
    targets = torch.randint(0, V, (R,), generator=g, device="cuda", dtype=torch.int32)
    if R > 1:
        logits[torch.arange(0, R, 2, device="cuda"), targets[::2].long()] = 6.0 * c["std"]
    return {"logits": logits, "targets": targets}


_INPUTS = {"chunk": _chunk_inputs, "slots": _slots_inputs, "prep": _prep_inputs, "logprobs": _logprobs_inputs}


def prepare(case, seed):
    c = dict(case)
    s = _INPUTS[c["kind"]](c, seed)
    s["case"] = c
    if c["kind"] == "chunk":
        s["out"] = torch.zeros(s["rows"], c["hq"], c["dh"], dtype=BF, device="cuda")
        s["lse"] = torch.zeros(c["hq"], s["rows"], dtype=F32, device="cuda") if c["lse"] else None
    elif c["kind"] == "slots":
        s["pos"], s["slot"] = (torch.zeros(s["rows"], dtype=torch.int32, device="cuda") for _ in range(2))
        s["status"] = torch.zeros(2, dtype=torch.int32, device="cuda")
    elif c["kind"] == "prep":
        T = c["rows"] + c["pad"]
        s["q"] = torch.zeros(T, c["hq"], c["dh"], dtype=BF, device="cuda")
        s["gate"] = torch.zeros(T, c["hq"], c["dh"], dtype=BF, device="cuda") if c["gate"] else None
    else:
        s["lp"], s["ent"] = (torch.zeros(c["rows"], dtype=F32, device="cuda") for _ in range(2))
        s["ids"] = torch.zeros(c["rows"], c["k"], dtype=torch.int32, device="cuda")
        s["top"] = torch.zeros(c["rows"], c["k"], dtype=F32, device="cuda")
        if own:
            need = _hip().api().cs1_token_logprobs_workspace_bytes(c["rows"], c["vocab"], c["k"])
            s["ws"] = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------- one pass, plain

def _plain_chunk(s, c):
    # sequence by sequence, all heads at once; a row at position p sees the keys 0 to p
    page, hk, dh, rep = c["page"], c["hk"], c["dh"], c["hq"] // c["hk"]
    cu, table = s["host_cu"], s["table"]
    for i, seq in enumerate(s["host_seqs"].tolist()):
        n, a, b = int(s["host_len"][i]), int(cu[i]), int(cu[i + 1])
        pg = table[seq, :_pages(n, page)].long()
        k = s["kp"][pg].flatten(0, 1)[:n].float().permute(1, 2, 0).contiguous()
        v = s["vp"][pg].flatten(0, 1)[:n].float().permute(1, 0, 2).contiguous()
        q = s["q"][a:b].float().view(b - a, hk, rep, dh).permute(1, 2, 0, 3).reshape(hk, rep * (b - a), dh)
        sc = (torch.matmul(q, k) * dh ** -0.5).view(hk, rep, b - a, n)
        late = torch.arange(n, device="cuda")[None, :] > torch.arange(n - (b - a), n, device="cuda")[:, None]
        sc.masked_fill_(late, -math.inf)
        m = sc.amax(-1, keepdim=True)
        p = sc.sub_(m).exp_()
        z = p.sum(-1, keepdim=True)
        o = torch.matmul(p.view(hk, rep * (b - a), n), v).view(hk, rep, b - a, dh) / z
        o = o.permute(2, 0, 1, 3).reshape(b - a, c["hq"], dh)
        if c["gate"]:
            o = o / (1 + torch.exp(-s["gate"][a:b].float()))
        s["out"][a:b] = o
        if c["lse"]:
            s["lse"][:, a:b] = (m + torch.log(z)).reshape(c["hq"], b - a)
    return [s["out"], s["lse"]] if c["lse"] else [s["out"]]


def _plain_slots(s, c):
    page = c["page"]
    table, lens, refs, cu = s["table"], s["lens"], s["refs"], s["cu"].long()
    seqs, new = s["seqs"].long(), s["new"]
    width = table.shape[1]
    # room: the lowest free pages in the list's order
    held = lens[seqs]
    begin = -(-held // page)
    need = -(-(held + new) // page) - begin
    j = torch.arange(width, device="cuda")[None, :]
    rank = ((torch.cumsum(need, 0) - need)[:, None] + j)
    takes = j < need[:, None]
    got = torch.searchsorted(torch.cumsum((refs == 0).int(), 0), (rank + 1).contiguous()).clamp(max=refs.numel() - 1)
    rows = torch.cat([table[seqs], table[seqs][:, :1]], 1)
    rows.scatter_(1, torch.where(takes, begin[:, None] + j, width).long(), got.int())
    table[seqs] = rows[:, :-1]
    refs.index_add_(0, got.reshape(-1), takes.int().reshape(-1))
    lens[seqs] = held + new
    # the rows' positions and places
    at = torch.arange(s["rows"], device="cuda")
    entry = torch.searchsorted(cu, at, right=True) - 1
    live = at < cu[-1]
    entry = entry.clamp(max=len(seqs) - 1)
    pos = torch.where(live, held[entry] + at - cu[entry], 0).long()
    place = table[seqs[entry], pos // page] * page + pos % page
    s["pos"].copy_(torch.where(live, pos, -1))
    s["slot"].copy_(torch.where(live, place, -1))
    # none of the drafted tokens is kept
    lens[seqs] = held
    j = torch.arange(width, device="cuda")[None, :]
    gone = (j >= begin[:, None]) & (j < (begin + need)[:, None])
    pages = table[seqs]
    refs.index_add_(0, pages.clamp(min=0).reshape(-1).long(), -gone.int().reshape(-1))
    table[seqs] = torch.where(gone, -1, pages)
    s["status"].zero_()
    return [s["pos"], s["slot"], table, lens, refs, s["status"]]


def _turn(x, cos, sin, c):
    """x [rows, heads, dh], its first `dims` dims turned; cos and sin [rows, dims / 2]."""
    d = c["dims"]
    a, b = (x[..., 0:d:2], x[..., 1:d:2]) if c["inter"] else (x[..., :d // 2], x[..., d // 2:d])
    cos, sin = cos[:, None, :], sin[:, None, :]
    ra, rb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([ra, rb], -1).flatten(-2) if c["inter"] else torch.cat([ra, rb], -1)
    return torch.cat([turned, x[..., d:]], -1)


def _prep(s, c, dt):
    """q, gate, k and v of the live rows in type dt."""
    hq, hk, dh, n = c["hq"], c["hk"], c["dh"], c["rows"]
    x = s["x"][:n].to(dt)
    w = hq * dh * (2 if c["gate"] else 1)
    qg = x[:, :w].view(n, hq, -1)
    q, gate = qg[..., :dh], qg[..., dh:]
    k, v = x[:, w:w + hk * dh].view(n, hk, dh), x[:, w + hk * dh:].view(n, hk, dh)
    if c["norm"]:
        q = q / torch.sqrt((q * q).mean(-1, keepdim=True) + EPS) * (1 + s["qw"].to(dt))
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + EPS) * (1 + s["kw"].to(dt))
    turn = s["pos"][:n].double()[:, None] * s["freqs"][None, :]  # 32 bits lose the angles of far positions
    cos, sin = torch.cos(turn).to(dt) * s["magnitude"], torch.sin(turn).to(dt) * s["magnitude"]
    return _turn(q, cos, sin, c), gate, _turn(k, cos, sin, c), v


def _plain_prep(s, c):
    n, place = c["rows"], s["slot"][:c["rows"]].long()
    q, gate, k, v = _prep(s, c, F32)
    s["q"][:n] = q
    if c["gate"]:
        s["gate"][:n] = gate
    s["kp"].flatten(0, 1)[place] = k.to(BF)
    s["vp"].flatten(0, 1)[place] = v.to(BF)
    return _prep_outputs(s, c)


def _prep_outputs(s, c):
    return [s["q"], s["kp"], s["vp"]] + ([s["gate"]] if c["gate"] else [])


def _plain_logprobs(s, c):
    R, V = c["rows"], c["vocab"]
    index = torch.arange(V, device="cuda", dtype=torch.int32)[None, :]
    for a in range(0, R, 256):  # what 256 rows take in 32 bits fits the card several times over
        x = s["logits"][a:a + 256, :V].to(F32, copy=True)  # (the alternatives are taken out of it below)
        m = x.amax(-1, keepdim=True)
        e = torch.exp(x - m)
        z = e.sum(-1, keepdim=True)
        lse = m + torch.log(z)
        s["lp"][a:a + 256] = (x.gather(1, s["targets"][a:a + 256].long()[:, None]) - lse)[:, 0]
        s["ent"][a:a + 256] = (torch.log(z) - (e * (x - m)).sum(-1, keepdim=True) / z)[:, 0]
        # the best alternatives one after another, the lowest index among equals
        for i in range(c["k"]):
            best = x.amax(-1, keepdim=True)
            at = torch.where(x == best, index, V).amin(-1, keepdim=True)
            s["ids"][a:a + 256, i:i + 1] = at
            s["top"][a:a + 256, i:i + 1] = best - lse
            x.scatter_(1, at.long(), -math.inf)
    return [s["lp"], s["ent"], s["ids"], s["top"]]


_PLAIN = {"chunk": _plain_chunk, "slots": _plain_slots, "prep": _plain_prep, "logprobs": _plain_logprobs}


# ---------------------------------------------------------------- one pass, the library's operations

_LIB = []  # the loaded library and the attention handle that a program keeps


def _hip():
    if not _LIB:
        pkg = os.path.join(os.getcwd(), "system1-omni_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from qwen3_5_native import hip

        hip.load()
        handle = hip.api().cs1_attention_paged_create()
        if not handle:
            raise RuntimeError("cs1_attention_paged_create")
        _LIB.extend([hip, handle])
    return _LIB[0]


def _p(t):
    return None if t is None else t.data_ptr()


def _calls(s, c):
    """The calls of one pass, as a program holds them ready: (function, arguments before the stream)."""
    hip = _hip()
    api, kind = hip.api(), c["kind"]
    if kind == "logprobs":
        return [(api.cs1_token_logprobs, (_p(s["logits"]), int(c["f32"]), c["vocab"] + c["pad"], _p(s["targets"]), c["rows"],
                                          c["vocab"], c["k"], _p(s["lp"]), _p(s["ent"]), _p(s["ids"]) if c["k"] else None,
                                          _p(s["top"]) if c["k"] else None, _p(s["ws"])))]
    if kind == "prep":
        hq, hk, dh = c["hq"], c["hk"], c["dh"]
        x, wq = s["x"].data_ptr(), hq * dh * (2 if c["gate"] else 1)
        s["rotary"] = hip.Rotary(_p(s["freqs"]), c["dims"], int(c["inter"]), s["magnitude"])
        s["pt"] = hip.PageTable(None, None, None, 1, 1, s["kp"].shape[0], c["page"])
        return [(api.cs1_attn_prep_paged, (x, x + 2 * wq, x + 2 * (wq + hk * dh), s["x"].shape[1], _p(s["qw"]), _p(s["kw"]), EPS,
                                           ctypes.byref(s["rotary"]), ctypes.byref(s["pt"]), _p(s["pos"]), _p(s["slot"]),
                                           _p(s["q"]), _p(s["gate"]), _p(s["kp"]), _p(s["vp"]), c["rows"] + c["pad"], hq, hk,
                                           dh))]
    nseq, max_pages = s["table"].shape
    s["pt"] = hip.PageTable(_p(s["table"]), _p(s["lens"]), _p(s["refs"]), nseq, max_pages, s["refs"].numel(), c["page"])
    pt, n = ctypes.byref(s["pt"]), len(s["host_seqs"])
    if kind == "chunk":
        most = int(np.diff(s["host_cu"]).max())
        return [(api.cs1_attention_paged_varlen, (_LIB[1], _p(s["q"]), _p(s["kp"]), _p(s["vp"]), pt, _p(s["seqs"]), _p(s["cu"]), n,
                                                  most, _p(s["gate"]), _p(s["out"]), _p(s["lse"]), s["rows"], c["hq"], c["hk"],
                                                  c["dh"], c["dh"] ** -0.5))]
    return [(api.cs1_kv_extend, (pt, _p(s["seqs"]), _p(s["cu"]), n, _p(s["status"]))),
            (api.cs1_kv_rows, (pt, _p(s["seqs"]), _p(s["cu"]), n, s["rows"], _p(s["pos"]), _p(s["slot"]))),
            (api.cs1_kv_trim, (pt, _p(s["seqs"]), _p(s["new"]), n, _p(s["status"]) + 4))]


def _outputs(s, c):
    if c["kind"] == "chunk":
        return [s["out"], s["lse"]] if c["lse"] else [s["out"]]
    if c["kind"] == "slots":
        return [s["pos"], s["slot"], s["table"], s["lens"], s["refs"], s["status"]]
    return _prep_outputs(s, c) if c["kind"] == "prep" else [s["lp"], s["ent"], s["ids"], s["top"]]


def run(s):
    c = s["case"]
    if own:
        if "calls" not in s:
            s["calls"] = _calls(s, c)
            s["outputs"] = _outputs(s, c)
        stream = torch.cuda.current_stream().cuda_stream
        for fn, args in s["calls"]:
            code = fn(*args, stream)
            if code:
                _hip().check(code, fn.__name__)
        return s["outputs"]
    return _PLAIN[c["kind"]](s, c)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    kind = c["kind"]
    if kind == "chunk":
        ctx, new = (x.astype(np.float64) for x in _lengths(c))
        row = c["hq"] * c["dh"]
        pairs = float((ctx * new + new * (new + 1) / 2).sum())  # (row, key)
        return {"bytes": 4.0 * float((ctx + new).sum()) * c["hk"] * c["dh"] + float(new.sum()) *
                (2.0 * row * (3 if c["gate"] else 2) + (4.0 * c["hq"] if c["lse"] else 0.0)), "flops": 4.0 * pairs * row}
    if kind == "slots":
        ctx, new = _lengths(c)
        taken = float(sum(_pages(int(a + b), c["page"]) - _pages(int(a), c["page"]) for a, b in zip(ctx, new)))
        # positions and slots out; offsets, numbers and lengths in and out; the pages that come and go
        return {"bytes": 8.0 * (float(new.sum()) + c["pad"]) + 20.0 * len(ctx) + 16.0 * taken, "flops": 0.0}
    if kind == "prep":
        row = (c["hq"] * (2 if c["gate"] else 1) + 2 * c["hk"]) * c["dh"]
        return {"bytes": c["rows"] * (4.0 * row + 8.0) + 4.0 * c["dims"], "flops": c["rows"] * 8.0 * (c["hq"] + c["hk"]) * c["dh"]}
    size = 4.0 if c["f32"] else 2.0
    return {"bytes": c["rows"] * (size * c["vocab"] + 12.0 + 8.0 * c["k"]), "flops": 5.0 * c["rows"] * c["vocab"]}


# ---------------------------------------------------------------- the same in 64 bits

def _exact_chunk(s, c):
    """Row by row in blocks: softmax over the keys up to the row's own."""
    rows, hq, dh, page = s["rows"], c["hq"], c["dh"], c["page"]
    out = torch.zeros(rows, hq, dh, dtype=F64, device="cuda")
    lse = torch.zeros(hq, rows, dtype=F64, device="cuda")
    for i, seq in enumerate(s["host_seqs"]):
        n, a, b = int(s["host_len"][i]), int(s["host_cu"][i]), int(s["host_cu"][i + 1])
        place = torch.tensor([int(s["host_table"][seq, j // page]) * page + j % page for j in range(n)], device="cuda")
        for h in range(hq):
            k = s["kp"].flatten(0, 1)[place, h // (hq // c["hk"])].to(F64)
            v = s["vp"].flatten(0, 1)[place, h // (hq // c["hk"])].to(F64)
            for r in range(a, b, 512):
                e = min(b, r + 512)
                sc = s["q"][r:e, h].to(F64) @ k.t() / math.sqrt(dh)
                pos = n - b + torch.arange(r, e, device="cuda")
                sc = sc.masked_fill(torch.arange(n, device="cuda")[None, :] > pos[:, None], -math.inf)
                lse[h, r:e] = torch.logsumexp(sc, -1)
                out[r:e, h] = torch.softmax(sc, -1) @ v
    n = int(s["host_cu"][-1])
    if c["gate"]:
        out[:n] *= torch.sigmoid(s["gate"][:n].to(F64))
    return [out, lse] if c["lse"] else [out]


def _exact_prep(s, c):
    hk, dh, n = c["hk"], c["dh"], c["rows"]
    x = s["x"][:n].to(F64)
    half = c["dims"] // 2
    angle = torch.outer(s["pos"][:n].to(F64), s["freqs"])
    unit = torch.polar(torch.full_like(angle, s["magnitude"]), angle)  # a pair of dims is a complex number, turned by this

    def head(h, width, at, w):
        y = x[:, at + h * width:at + h * width + dh].clone()
        if w is not None:
            y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / dh + EPS) * (1 + w.to(F64))
        lo, hi = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if c["inter"] else (slice(0, half), slice(half, 2 * half))
        z = torch.complex(y[:, lo], y[:, hi]) * unit
        y[:, lo], y[:, hi] = z.real, z.imag
        return y

    wide = dh * (2 if c["gate"] else 1)
    k0 = c["hq"] * wide
    q = torch.zeros(n + c["pad"], c["hq"], dh, dtype=F64, device="cuda")
    gate = torch.zeros_like(q)
    kp = torch.zeros(s["kp"].shape[0] * c["page"], hk, dh, dtype=F64, device="cuda")
    vp = torch.zeros_like(kp)
    place = s["slot"][:n].long()
    for h in range(c["hq"]):
        q[:n, h] = head(h, wide, 0, s["qw"])
        gate[:n, h] = x[:, h * wide + wide - dh:(h + 1) * wide]
    for h in range(hk):
        kp[place, h] = head(h, dh, k0, s["kw"])
        vp[place, h] = x[:, k0 + (hk + h) * dh:k0 + (hk + h + 1) * dh]
    shape = s["kp"].shape
    return [q, kp.view(shape), vp.view(shape)] + ([gate] if c["gate"] else [])


def _exact_logprobs(s, c):
    R, V, k = c["rows"], c["vocab"], c["k"]
    lp, ent = (torch.zeros(R, dtype=F64, device="cuda") for _ in range(2))
    top = torch.zeros(R, k, dtype=F64, device="cuda")
    ids = torch.zeros(R, k, dtype=torch.int32, device="cuda")
    for r in range(0, R, 64):
        x = s["logits"][r:r + 64, :V].to(F64)
        logp = torch.log_softmax(x, -1)
        lp[r:r + 64] = logp.gather(1, s["targets"][r:r + 64].long()[:, None])[:, 0]
        ent[r:r + 64] = -(logp.exp() * logp).sum(-1)
        if k:
            order = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :k]
            ids[r:r + 64] = order.int()
            top[r:r + 64] = logp.gather(1, order)
    return [lp, ent, ids, top]


def exact(case, seed):
    """The operators' definition; None where a pass gives whole numbers only."""
    c = dict(case)
    if c["kind"] == "slots":
        return None
    s = _INPUTS[c["kind"]](c, seed)
    return {"chunk": _exact_chunk, "prep": _exact_prep, "logprobs": _exact_logprobs}[c["kind"]](s, c)
