"""The decode side of the hybrid decoder, as measurable cases: attention of one new token over a paged
key-value cache, one token of the gated delta rule on its stored states, and what a program does to
the cache's pages (fork, reserve, write, free, compact, copy).

Each case runs in a plain form made of elementary torch operations in 32 bits, or, where `own` is
true, through the library's operations as a serving program calls them.  Sizes are the repository's
own: 16 query over 4 key-value heads with head dim 128 or 256 (4B class) and 24 over 4 (27B class), 16
key heads over 16, 32 or 48 value heads of dim 128 in the delta rule, 8 and 16 attention layers, 24 and 48
delta-rule layers, prefixes and contexts of the prompt lengths up to 8192 and, for decoding, on to
32768 tokens.
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
D = 128  # head dim of the delta rule


def listed():
    return [
        # a chat turn in progress, one user: the smallest call, latency counts
        {"name": "paged-1x700", "kind": "paged", "rows": 1, "live": 1, "nseq": 4, "lo": 700, "hi": 700, "hq": 16, "hk": 4,
         "dh": 128, "page": 16, "gate": True, "lse": True, "lens": 1},
        # one long document, one user: few rows, all of the chip has to share one sequence
        {"name": "paged-1x32768", "kind": "paged", "rows": 1, "live": 1, "nseq": 2, "lo": 32768, "hi": 32768, "hq": 16,
         "hk": 4, "dh": 256, "page": 64, "gate": True, "lse": False, "lens": 2},
        # a server's batch of ragged chats in the 4B-class decoder, its last rows padding
        {"name": "paged-48x4k", "kind": "paged", "rows": 48, "live": 43, "nseq": 64, "lo": 1, "hi": 4096, "hq": 16, "hk": 4,
         "dh": 256, "page": 64, "gate": True, "lse": False, "lens": 3},
        # long contexts in the 27B-class decoder, six query heads to a key-value head, large pages of an odd size
        {"name": "paged-9x32k", "kind": "paged", "rows": 9, "live": 9, "nseq": 9, "lo": 9000, "hi": 32768, "hq": 24, "hk": 4,
         "dh": 256, "page": 208, "gate": True, "lse": True, "lens": 4},
        # one user's next token through a delta-rule layer of the 4B-class decoder
        {"name": "gdnstep-1", "kind": "gdnstep", "rows": 1, "live": 1, "nseq": 4, "hk": 16, "h": 32, "norm": True, "lens": 5},
        # a batch with padding in the 27B-class decoder
        {"name": "gdnstep-61-27b", "kind": "gdnstep", "rows": 64, "live": 61, "nseq": 72, "hk": 16, "h": 48, "norm": True,
         "lens": 6},
        # a middling batch of the smallest layer, whose output goes on without gate and norm
        {"name": "gdnstep-13-raw", "kind": "gdnstep", "rows": 13, "live": 13, "nseq": 16, "hk": 16, "h": 16, "norm": False,
         "lens": 7},
        # two continuations of a short prompt, a few tokens each: latency
        {"name": "branch-2", "kind": "branch", "n": 2, "prefix": 107, "lo": 1, "hi": 9, "page": 16, "layers": 1, "hk": 4,
         "dh": 128, "lens": 8},
        # candidate scoring over one cached 2048-token prompt: eight candidates in the 4B-class decoder
        {"name": "branch-8", "kind": "branch", "n": 8, "prefix": 2077, "lo": 64, "hi": 256, "page": 64, "layers": 8, "hk": 4,
         "dh": 256, "lens": 9},
        # many samples of one prompt in the 27B-class decoder, one token each so far
        {"name": "branch-64", "kind": "branch", "n": 64, "prefix": 936, "lo": 1, "hi": 1, "page": 64, "layers": 16, "hk": 4,
         "dh": 256, "lens": 10},
        # a pool of the 4B-class decoder after chats have ended in it: the pages that are held move to its start
        {"name": "compact-4b", "kind": "compact", "nseq": 48, "lo": 1, "hi": 1800, "page": 64, "layers": 8, "hk": 4, "dh": 256,
         "free": 0.5, "lens": 11},
        # the delta-rule states of eight candidates start as copies of their prompt's, in every layer of the 4B class
        {"name": "copy-8", "kind": "copy", "n": 8, "nseq": 16, "layers": 24, "h": 32, "sources": 1, "lens": 12},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["paged", "paged", "paged", "gdnstep", "gdnstep", "branch", "branch", "compact", "copy"])
    c = {"kind": kind}
    if kind == "paged":
        hq, hk, dh = rng.choice([(16, 4, 128), (16, 4, 256), (24, 4, 256), (8, 4, 128), (32, 8, 128), (16, 1, 256)])
        live = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, min(32768, 180000 // live))
        c.update(rows=live + rng.choice([0, 0, 1, 5]), live=live, nseq=live + rng.randint(0, 9), lo=rng.choice([1, hi, 1 + hi // 2]),
                 hi=hi, hq=hq, hk=hk, dh=dh, page=rng.choice([16, 32, 48, 64, 128, 208, 256]), gate=rng.random() < 0.7,
                 lse=rng.random() < 0.5)
    elif kind == "gdnstep":
        live = _log_int(rng, 1, 64)
        c.update(rows=live + rng.choice([0, 0, 1, 5]), live=live, nseq=live + 5 + rng.randint(0, 9), hk=16,
                 h=rng.choice([16, 32, 48]), norm=rng.random() < 0.7)
    elif kind == "branch":
        hi = rng.choice([1, 9, 64, 256])
        c.update(n=_log_int(rng, 1, 64), prefix=_log_int(rng, 1, 8192), lo=rng.choice([1, hi]), hi=hi,
                 page=rng.choice([16, 32, 48, 64, 128]), layers=rng.choice([1, 2, 8]), hk=4, dh=rng.choice([128, 256]))
    elif kind == "compact":
        c.update(nseq=_log_int(rng, 2, 32), lo=rng.choice([0, 1, 500]), hi=_log_int(rng, 501, 1800),
                 page=rng.choice([16, 48, 64, 128]), layers=rng.choice([1, 2, 8]), hk=4, dh=rng.choice([128, 256]),
                 free=round(rng.uniform(0.1, 0.6), 2))
    else:
        n = _log_int(rng, 1, 24)
        c.update(n=n, nseq=2 * n + rng.randint(1, 4), layers=rng.choice([1, 3, 24 if n <= 8 else 6]),
                 h=rng.choice([16, 32]), sources=rng.randint(1, n))
    c["lens"] = rng.randint(0, 1 << 20)
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


def _lens(c, n):
    """n lengths, uniform on [lo, hi], the same for every seed (the work is the case's)."""
    return np.random.default_rng(c["lens"]).integers(c["lo"], c["hi"] + 1, n)


def _pages(n, page):
    return -(-n // page)


def _page_table(seed, nseq, lens_of, page, spare, max_pages):
    """Sequences lens_of {sequence: tokens} on pages in a random order; `spare` pages are free."""
    rng = np.random.default_rng(seed)
    held = sum(_pages(int(n), page) for n in lens_of.values())
    order = rng.permutation(held + spare)
    table, lens = np.full((nseq, max_pages), -1, np.int32), np.zeros(nseq, np.int32)
    refs = np.zeros(held + spare, np.int32)
    at = 0
    for s, n in lens_of.items():
        k = _pages(int(n), page)
        table[s, :k] = order[at:at + k]
        refs[order[at:at + k]] = 1
        lens[s] = n
        at += k
    return table, lens, refs


def _paged_inputs(c, seed):
    rng = np.random.default_rng(seed)
    g = _gen(seed)
    n, page = _lens(c, c["live"]), c["page"]
    seqs = np.full(c["rows"], -1, np.int32)
    seqs[:c["live"]] = rng.permutation(c["nseq"])[:c["live"]]
    table, lens, refs = _page_table(seed, c["nseq"], dict(zip(seqs[:c["live"]].tolist(), n)), page, 3, _pages(c["hi"], page) + 1)
    s = {"table": _ints(table), "lens": _ints(lens), "refs": _ints(refs), "seqs": _ints(seqs)}
    s["q"] = _randn(g, c["rows"], c["hq"], c["dh"])
    s["gate"] = _randn(g, c["rows"], c["hq"], c["dh"]) if c["gate"] else None
    s["kp"] = _randn(g, len(refs), page, c["hk"], c["dh"])
    s["vp"] = _randn(g, len(refs), page, c["hk"], c["dh"])
    return s


def _gdnstep_inputs(c, seed):
    # a row is what the layer's input projection writes: q | k | v | z | b | a.  The gates' decay is spread as the
    # layer's parameters are set up: softplus(dt_bias) log-uniform on [1e-3, 1e-1], A on [1, 16].
    rng = np.random.default_rng(seed)
    g = _gen(seed)
    hk, h, nseq = c["hk"], c["h"], c["nseq"]
    conv = (2 * hk + h) * D
    u = torch.rand(h, generator=g, device="cuda")
    dt = torch.exp(math.log(1e-3) + u * (math.log(1e-1) - math.log(1e-3)))
    seqs = np.full(c["rows"], -1, np.int32)
    seqs[:c["live"]] = rng.permutation(nseq)[:c["live"]]
    # tokens held with the new one: mostly far into a text, some sequences at their first tokens
    lens = rng.integers(5, 5000, nseq)
    lens[rng.permutation(nseq)[:nseq // 4]] = rng.integers(1, 5, nseq // 4)
    s = {"seqs": _ints(seqs), "lens": _ints(lens), "x": _randn(g, c["rows"], conv + h * D + 2 * h),
         "cw": (torch.rand(conv, 4, generator=g, device="cuda") - 0.5).to(BF),
         "a_log": torch.log(1 + 15 * torch.rand(h, generator=g, device="cuda")).to(BF),
         "dt_bias": torch.log(torch.expm1(dt)).to(BF), "gw": (1 + _randn(g, D, std=0.1).float()).to(BF),
         "ring": _randn(g, nseq, 4, conv), "state": torch.randn(nseq, h, D, D, generator=g, device="cuda").mul_(0.1)}
    s["x"][:, -h:] *= 0.5
    return s


def _branch_inputs(c, seed):
    rng = np.random.default_rng(seed)
    g = _gen(seed)
    n, page, hk, dh = c["n"], c["page"], c["hk"], c["dh"]
    new = _lens(c, n)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    longest = _pages(c["prefix"] + c["hi"], page)
    spare = n * (_pages(c["hi"], page) + 1) + 2
    # two sequences besides: the prefix and another that is left alone
    ids = rng.permutation(n + 3)
    table, lens, refs = _page_table(seed, n + 3, {int(ids[0]): c["prefix"], int(ids[1]): 2 * page + 1}, page, spare,
                                    max(longest, 3))
    rows = np.repeat(np.arange(n), new)
    return {"table": _ints(table), "lens": _ints(lens), "refs": _ints(refs), "src": _ints(np.full(n, ids[0])),
            "dst": _ints(ids[2:2 + n]), "cu": cu, "add": _ints(new), "row_child": _ints(rows),
            "row_at": _ints(np.arange(cu[-1]) - cu[rows]), "status": torch.zeros(2, dtype=torch.int32, device="cuda"),
            # what the layers' projections leave of the new tokens: the prepared keys, and raw rows k | v
            "k": _randn(g, c["layers"], int(cu[-1]), hk * dh), "kv": _randn(g, c["layers"], int(cu[-1]), 2 * hk * dh),
            "pools": _randn(g, 2 * c["layers"], len(refs), page, hk * dh).view(torch.int16)}


def _compact_inputs(c, seed):
    g = _gen(seed)
    n = _lens(c, c["nseq"])
    held = int(sum(_pages(int(x), c["page"]) for x in n))
    spare = max(1, int(held * c["free"] / (1 - c["free"])))
    table, lens, refs = _page_table(seed, c["nseq"], dict(enumerate(n)), c["page"], spare, _pages(c["hi"], c["page"]) + 1)
    # one block of whole numbers, so that one copy brings the server's table of the moment
    meta = _ints(np.concatenate([table.reshape(-1), lens, refs]))
    here = torch.empty_like(meta)
    a, b = table.size, table.size + lens.size
    return {"meta0": meta, "meta": here, "table": here[:a].view(table.shape), "lens": here[a:b], "refs": here[b:],
            "status": torch.zeros(1, dtype=torch.int32, device="cuda"),
            "pools": _randn(g, 2 * c["layers"], len(refs), c["page"], c["hk"] * c["dh"]).view(torch.int16)}


def _copy_inputs(c, seed):
    rng = np.random.default_rng(seed)
    g = _gen(seed)
    ids = rng.permutation(c["nseq"])
    n, k = c["n"], c["sources"]
    src = ids[rng.integers(0, k, n)]
    return {"src": _ints(src), "dst": _ints(ids[k:k + n]),
            "pools": torch.randn(c["layers"], c["nseq"], c["h"] * D * D, generator=g, device="cuda").view(torch.int32)}


_INPUTS = {"paged": _paged_inputs, "gdnstep": _gdnstep_inputs, "branch": _branch_inputs, "compact": _compact_inputs,
           "copy": _copy_inputs}


def prepare(case, seed):
    c = dict(case)
    s = _INPUTS[c["kind"]](c, seed)
    s["case"] = c
    if c["kind"] == "paged":
        s["out"] = torch.empty(c["rows"], c["hq"], c["dh"], dtype=BF, device="cuda")
        s["lse"] = torch.empty(c["hq"], c["rows"], dtype=F32, device="cuda") if c["lse"] else None
    elif c["kind"] == "gdnstep":
        s["out"] = torch.empty(c["rows"], c["h"], D, dtype=BF, device="cuda")
    elif c["kind"] in ("branch", "compact"):
        s["ws"] = torch.empty(2 * s["refs"].numel() + 4 * c.get("n", 0) + 64, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------- one pass, plain

def _plain_paged(s, c):
    # every sequence padded to the longest; a padding row sees nothing: zeros, and a log-sum-exp of -inf
    page, hk, dh = c["page"], c["hk"], c["dh"]
    rows, longest = c["rows"], c["hi"]
    live = s["seqs"] >= 0
    seq = s["seqs"].clamp(min=0).long()
    n = torch.where(live, s["lens"][seq], 0)
    at = torch.arange(longest, device="cuda")
    see = at[None, :] < n[:, None]
    pg = s["table"][seq][:, at // page].clamp(min=0).long()
    k = s["kp"][pg, at % page].float()
    v = s["vp"][pg, at % page].float().masked_fill_(~see[:, :, None, None], 0.0)
    q = s["q"].float().view(rows, hk, -1, dh)
    sc = torch.matmul(q, k.permute(0, 2, 3, 1)) * dh ** -0.5
    sc = sc.masked_fill(~see[:, None, None, :], -math.inf)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(torch.isfinite(m), m, 0.0)
    p = torch.exp(sc - m)
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(z > 0, z, 1.0)
    o = o.reshape(rows, c["hq"], dh)
    if c["gate"]:
        o = o / (1 + torch.exp(-s["gate"].float()))
    s["out"].copy_(o)
    if not c["lse"]:
        return [s["out"]]
    s["lse"].copy_((m + torch.log(z)).reshape(rows, c["hq"]).t())
    return [s["out"], s["lse"]]


def _plain_gdnstep(s, c):
    hk, h, rows = c["hk"], c["h"], c["rows"]
    conv = (2 * hk + h) * D
    live = s["seqs"] >= 0
    seq = s["seqs"].clamp(min=0).long()
    pos = (s["lens"][seq] - 1).long()
    x = s["x"].float()
    # the last four inputs of the conv, the new one last; those before position 0 are zero
    back = pos[:, None] + torch.arange(-3, 0, device="cuda")[None, :]
    past = s["ring"][seq[:, None], back % 4].float() * (back >= 0)[:, :, None]
    win = torch.cat([past, x[:, None, :conv]], 1)
    y = (win * s["cw"].float().t()[None]).sum(1)
    y = y / (1 + torch.exp(-y))
    q = y[:, :hk * D].view(rows, hk, D)
    k = y[:, hk * D:2 * hk * D].view(rows, hk, D)
    v = y[:, 2 * hk * D:].view(rows, h, D)
    q = (q * torch.rsqrt((q * q).sum(-1, keepdim=True) + 1e-6) * D ** -0.5).repeat_interleave(h // hk, 1)
    k = (k * torch.rsqrt((k * k).sum(-1, keepdim=True) + 1e-6)).repeat_interleave(h // hk, 1)
    z, b, a = x[:, conv:conv + h * D].view(rows, h, D), x[:, conv + h * D:conv + h * D + h], x[:, conv + h * D + h:]
    beta = 1 / (1 + torch.exp(-b))
    decay = torch.exp(-torch.exp(s["a_log"].float()) * torch.log1p(torch.exp(a + s["dt_bias"].float())))
    # S' = decay S + k (beta (v - (decay S)^T k))^T, o = S'^T q; a sequence's first token starts from zero
    S = s["state"][seq] * (decay * (pos > 0)[:, None])[:, :, None, None]
    u = beta[:, :, None] * (v - (S * k[:, :, :, None]).sum(2))
    S = S + k[:, :, :, None] * u[:, :, None, :]
    o = (S * q[:, :, :, None]).sum(2)
    if c["norm"]:
        o = s["gw"].float() * (o * torch.rsqrt((o * o).mean(-1, keepdim=True) + EPS)) * (z / (1 + torch.exp(-z)))
    s["out"].copy_(o * live[:, None, None])
    n = c["live"]  # the padding rows are the last ones
    s["state"][seq[:n]] = S[:n]
    s["ring"][seq[:n], pos[:n] % 4] = s["x"][:n, :conv]
    return [s["out"], s["state"], s["ring"]]


def _lowest_free(refs, rank):
    """The page that is free as number `rank` (from 0), counted from page 0."""
    return torch.searchsorted(torch.cumsum((refs == 0).int(), 0), (rank + 1).contiguous())


def _plain_branch(s, c):
    page, n = c["page"], c["n"]
    table, lens, refs, pools = s["table"], s["lens"], s["refs"], s["pools"]
    src, dst, add = s["src"].long(), s["dst"].long(), s["add"]
    npages = refs.numel()
    # fork: whole pages are shared; what the last one holds of an unfinished page goes to a page of its own
    held, full = lens[src], lens[src] // page
    part = held % page
    need = (part > 0).int()
    fresh = _lowest_free(refs, torch.cumsum(need, 0) - need).clamp(max=npages - 1)
    rows = table[src]
    last = full.long().clamp(max=table.shape[1] - 1)[:, None]
    old = rows.gather(1, last)[:, 0].clamp(min=0).long()
    shared = torch.arange(table.shape[1], device="cuda")[None, :] < full[:, None]
    refs.index_add_(0, rows.clamp(min=0).reshape(-1).long(), shared.int().reshape(-1))
    refs.index_add_(0, fresh, need)
    rows.scatter_(1, last, torch.where(need > 0, fresh.int(), rows.gather(1, last)[:, 0])[:, None])
    table[dst] = rows
    lens[dst] = held
    if c["prefix"] % page:
        kept = (torch.arange(page, device="cuda")[None, :] < part[:, None])[None, :, :, None]
        pools[:, fresh] = torch.where(kept, pools[:, old], pools[:, fresh])
    # reserve: the lowest free pages in the sequences' order
    begin = -(-held // page)
    need = -(-(held + add) // page) - begin
    j = torch.arange(_pages(c["hi"], page), device="cuda")[None, :]
    got = _lowest_free(refs, (torch.cumsum(need, 0) - need)[:, None] + j).clamp(max=npages - 1)
    takes = j < need[:, None]
    to = (begin[:, None] + j).clamp(max=table.shape[1] - 1)
    rows = torch.cat([table[dst], table[dst][:, :1]], 1)  # a last column for what is not taken
    rows.scatter_(1, torch.where(takes, to, table.shape[1]).long(), got.int())
    table[dst] = rows[:, :-1]
    refs.index_add_(0, got.reshape(-1), takes.int().reshape(-1))
    lens[dst] = held + add
    # write: the new tokens' keys and values in every layer
    child = s["row_child"].long()
    pos = held[child] + s["row_at"]
    flat = table[dst[child], (pos // page).long()].long() * page + pos % page
    L, width = c["layers"], c["hk"] * c["dh"]
    slots = pools.view(2 * L, npages * page, width)
    slots[:L, flat] = s["k"].view(torch.int16)
    slots[L:, flat] = s["kv"][:, :, width:].view(torch.int16)
    # free: the continuations are scored
    held_pages = torch.arange(table.shape[1], device="cuda")[None, :] < (-(-lens[dst] // page))[:, None]
    refs.index_add_(0, table[dst].clamp(min=0).reshape(-1).long(), -held_pages.int().reshape(-1))
    table[dst] = -1
    lens[dst] = 0
    s["status"].zero_()
    return [pools, table, lens, refs, s["status"]]


def _plain_compact(s, c):
    s["meta"].copy_(s["meta0"])
    table, refs, pools = s["table"], s["refs"], s["pools"]
    held = refs > 0
    n = held.sum()
    at = torch.arange(refs.numel(), device="cuda")
    moved = torch.nonzero(held & (at >= n))[:, 0]
    holes = torch.nonzero(~held & (at < n))[:, 0]
    to = at.int()
    to[moved] = holes.int()
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    refs[holes] = refs[moved]
    refs[moved] = 0
    pools[:, holes] = pools[:, moved]
    s["status"].copy_(n.reshape(1))
    # the pages that are held; those behind them are free, whatever they hold
    return [table, s["lens"], refs, pools, s["status"]]


def _plain_copy(s, c):
    s["pools"][:, s["dst"].long()] = s["pools"][:, s["src"].long()]
    return [s["pools"]]


_PLAIN = {"paged": _plain_paged, "gdnstep": _plain_gdnstep, "branch": _plain_branch, "compact": _plain_compact,
          "copy": _plain_copy}


# ---------------------------------------------------------------- one pass, the library's operations

_LIB = []  # the loaded library and the attention handle that a program keeps


def _lib():
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
    return _LIB


def _p(t):
    return None if t is None else t.data_ptr()


def _calls(s, c):
    """The calls of one pass, as a program holds them ready: (function, arguments before the stream)."""
    hip, handle = _lib()
    api = hip.api()
    kind = c["kind"]
    if kind == "gdnstep":
        conv, h = (2 * c["hk"] + c["h"]) * D, c["h"]
        x = s["x"].data_ptr()
        z, b = x + 2 * conv, x + 2 * (conv + h * D)
        return [(api.cs1_gdn_decode, (x, s["x"].shape[1], _p(s["cw"]), z if c["norm"] else None, b, b + 2 * h,
                                      _p(s["a_log"]), _p(s["dt_bias"]), _p(s["gw"]) if c["norm"] else None, EPS,
                                      _p(s["ring"]), _p(s["state"]), _p(s["seqs"]), _p(s["lens"]), c["nseq"], _p(s["out"]),
                                      c["rows"], h, c["hk"], D ** -0.5))]
    if kind == "copy":
        width = s["pools"].shape[2] * 4
        s["ptrs"] = (ctypes.c_void_p * c["layers"])(*[s["pools"][i].data_ptr() for i in range(c["layers"])])
        return [(api.cs1_kv_copy, (s["ptrs"], c["layers"], width, c["nseq"], _p(s["src"]), _p(s["dst"]), c["n"]))]
    nseq, max_pages = s["table"].shape
    s["pt"] = hip.PageTable(_p(s["table"]), _p(s["lens"]), _p(s["refs"]), nseq, max_pages, s["refs"].numel(), c["page"])
    pt = ctypes.byref(s["pt"])
    if kind == "paged":
        return [(api.cs1_attention_paged, (handle, _p(s["q"]), _p(s["kp"]), _p(s["vp"]), pt, _p(s["seqs"]), _p(s["gate"]),
                                           _p(s["out"]), _p(s["lse"]), c["rows"], c["hq"], c["hk"], c["dh"],
                                           c["dh"] ** -0.5))]
    L, row = c["layers"], 2 * c["hk"] * c["dh"]
    s["ptrs"] = (ctypes.c_void_p * (2 * L))(*[s["pools"][i].data_ptr() for i in range(2 * L)])
    assert api.cs1_kv_workspace_bytes(s["refs"].numel(), c.get("n", 0)) <= 4 * s["ws"].numel()
    if kind == "compact":
        return [(api.cs1_copy_dd, (_p(s["meta"]), _p(s["meta0"]), 4 * s["meta"].numel())),
                (api.cs1_kv_compact, (pt, s["ptrs"], 2 * L, row, _p(s["ws"]), _p(s["status"])))]
    n, cu, width = c["n"], s["cu"].ctypes.data, c["hk"] * c["dh"]
    calls = [(api.cs1_kv_fork, (pt, _p(s["src"]), _p(s["dst"]), n, s["ptrs"], 2 * L, row, _p(s["ws"]), _p(s["status"]))),
             (api.cs1_kv_reserve, (pt, _p(s["dst"]), cu, n, _p(s["status"]) + 4))]
    calls += [(api.cs1_kv_write, (pt, _p(s["dst"]), cu, n, _p(s["k"][i]), width, _p(s["kv"][i]) + 2 * width, 2 * width,
                                  s["ptrs"][i], s["ptrs"][L + i], c["hk"], c["dh"])) for i in range(L)]
    return calls + [(api.cs1_kv_free, (pt, _p(s["dst"]), n))]


def _outputs(s, c):
    kind = c["kind"]
    if kind == "paged":
        return [s["out"], s["lse"]] if c["lse"] else [s["out"]]
    if kind == "gdnstep":
        return [s["out"], s["state"], s["ring"]]
    if kind == "branch":
        return [s["pools"], s["table"], s["lens"], s["refs"], s["status"]]
    return [s["table"], s["lens"], s["refs"], s["pools"], s["status"]] if kind == "compact" else [s["pools"]]


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
                _lib()[0].check(code, fn.__name__)
        return s["outputs"]
    return _PLAIN[c["kind"]](s, c)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    kind = c["kind"]
    if kind == "paged":
        n = float(_lens(c, c["live"]).sum())
        return {"bytes": 4.0 * n * c["hk"] * c["dh"] + 2.0 * c["live"] * c["hq"] * c["dh"] * (3 if c["gate"] else 2),
                "flops": 4.0 * n * c["hq"] * c["dh"]}
    if kind == "gdnstep":
        hk, h, B = c["hk"], c["h"], c["live"]
        conv = (2 * hk + h) * D
        row = conv * 5 + 2 * h + h * D * (2 if c["norm"] else 1)  # the new row in, three old ones in, one out
        return {"bytes": B * (8.0 * h * D * D + 2.0 * row) + 8.0 * conv, "flops": B * h * 8.0 * D * D}
    if kind == "branch":
        row = 2.0 * c["hk"] * c["dh"] * 2 * c["layers"]
        n, new = c["n"], float(_lens(c, c["n"]).sum())
        return {"bytes": 2 * row * (n * (c["prefix"] % c["page"]) + new) + 8.0 * n * _pages(c["prefix"], c["page"]), "flops": 0.0}
    if kind == "compact":
        # of the pages that are held, a share of `free` lies behind the held ones' count
        held = sum(_pages(int(x), c["page"]) for x in _lens(c, c["nseq"]))
        page = 2.0 * c["hk"] * c["dh"] * c["page"] * 2 * c["layers"]
        return {"bytes": 2 * page * max(1.0, held * c["free"]) + 4.0 * held / (1 - c["free"]), "flops": 0.0}
    return {"bytes": 2.0 * c["n"] * c["layers"] * c["h"] * D * D * 4, "flops": 0.0}


# ---------------------------------------------------------------- the same in 64 bits

def _exact_paged(s, c):
    out = torch.zeros(c["rows"], c["hq"], c["dh"], dtype=F64, device="cuda")
    lse = torch.full((c["hq"], c["rows"]), -math.inf, dtype=F64, device="cuda")
    rep = c["hq"] // c["hk"]
    table, lens = s["table"].tolist(), s["lens"].tolist()
    for r, seq in enumerate(s["seqs"].tolist()):
        if seq < 0 or lens[seq] == 0:
            continue
        n = lens[seq]
        pages = torch.tensor(table[seq][:_pages(n, c["page"])], device="cuda")
        k = s["kp"][pages].flatten(0, 1)[:n].to(F64)
        v = s["vp"][pages].flatten(0, 1)[:n].to(F64)
        for h in range(c["hq"]):
            sc = (k[:, h // rep] * s["q"][r, h].to(F64)).sum(-1) / math.sqrt(c["dh"])
            lse[h, r] = torch.logsumexp(sc, 0)
            out[r, h] = (torch.softmax(sc, 0)[:, None] * v[:, h // rep]).sum(0)
    if c["gate"]:
        out *= torch.sigmoid(s["gate"].to(F64))
    return [out, lse] if c["lse"] else [out]


def _exact_gdnstep(s, c):
    hk, h = c["hk"], c["h"]
    conv = (2 * hk + h) * D
    out = torch.zeros(c["rows"], h, D, dtype=F64, device="cuda")
    state, ring = s["state"].to(F64), s["ring"].to(F64)
    w, lens = s["cw"].to(F64), s["lens"].tolist()
    silu = torch.nn.functional.silu
    for r, seq in enumerate(s["seqs"].tolist()):
        if seq < 0:
            continue
        pos = lens[seq] - 1
        x = s["x"][r].to(F64)
        y = w[:, 3] * x[:conv]
        for i in range(1, min(3, pos) + 1):
            y = y + w[:, 3 - i] * ring[seq, (pos - i) % 4]
        y = silu(y)
        q, k, v = y[:hk * D].view(hk, D), y[hk * D:2 * hk * D].view(hk, D), y[2 * hk * D:].view(h, D)
        q = q / torch.sqrt((q ** 2).sum(-1, keepdim=True) + 1e-6) / math.sqrt(D)
        k = k / torch.sqrt((k ** 2).sum(-1, keepdim=True) + 1e-6)
        rest = x[conv:]
        z, b, a = rest[:h * D].view(h, D), rest[h * D:h * D + h], rest[h * D + h:]
        g = -torch.exp(s["a_log"].to(F64)) * torch.nn.functional.softplus(a + s["dt_bias"].to(F64))
        for i in range(h):
            S = state[seq, i] * torch.exp(g[i]) if pos > 0 else torch.zeros(D, D, dtype=F64, device="cuda")
            kk, qq = k[i // (h // hk)], q[i // (h // hk)]
            S = S + torch.outer(kk, torch.sigmoid(b[i]) * (v[i] - kk @ S))
            state[seq, i] = S
            o = qq @ S
            if c["norm"]:
                o = s["gw"].to(F64) * o / torch.sqrt((o ** 2).mean() + EPS) * silu(z[i])
            out[r, i] = o
        ring[seq, pos % 4] = x[:conv]
    return [out, state, ring]


def exact(case, seed):
    """The operators' definition, sequence by sequence and head by head; None where a pass only moves whole values."""
    c = dict(case)
    if c["kind"] == "paged":
        return _exact_paged(_paged_inputs(c, seed), c)
    if c["kind"] == "gdnstep":
        return _exact_gdnstep(_gdnstep_inputs(c, seed), c)
    return None
