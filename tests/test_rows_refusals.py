"""The operations on several new tokens of a sequence refuse what they cannot do before any device work, and accept
empty work; the rotary frequencies, which need no device, against their formula."""
import ctypes
import math

import numpy as np
import pytest

from qwen3_5_native import hip
from test_decode_refusals import BAD_TABLES, table

INVALID = hip.HIP_ERROR_INVALID_VALUE
N = None
A = 1 << 20  # an aligned address that is never followed: every call here returns before a launch


@pytest.fixture(scope="module")
def api():
    return hip.load()


@pytest.mark.parametrize("bad", BAD_TABLES + [dict(npages=(1 << 30) + 1)], ids=str)
def test_bad_tables(api, bad):
    t = table(**bad)
    assert api.cs1_kv_extend(t, N, A, 0, A, N) == INVALID
    assert api.cs1_kv_rows(t, N, A, 0, 0, A, A, N) == INVALID
    assert api.cs1_kv_trim(t, N, A, 0, A, N) == INVALID


def test_extend_rows_trim(api):
    for n in (-1, 8193):
        assert api.cs1_kv_extend(table(), N, A, n, A, N) == INVALID
        assert api.cs1_kv_rows(table(), N, A, n, 4, A, A, N) == INVALID
        assert api.cs1_kv_trim(table(), N, A, n, A, N) == INVALID
    assert api.cs1_kv_extend(N, N, A, 1, A, N) == INVALID
    assert api.cs1_kv_extend(table(), N, N, 1, A, N) == INVALID  # no offsets
    assert api.cs1_kv_extend(table(), N, A, 1, N, N) == INVALID  # no status
    assert api.cs1_kv_rows(table(), N, N, 1, 4, A, A, N) == INVALID
    assert api.cs1_kv_rows(table(), N, A, 1, -1, A, A, N) == INVALID
    assert api.cs1_kv_rows(table(), N, A, 1, 4, N, A, N) == INVALID
    assert api.cs1_kv_rows(table(), N, A, 1, 4, A, N, N) == INVALID
    assert api.cs1_kv_rows(table(npages=1 << 27), N, A, 1, 4, A, A, N) == INVALID  # 2^31 slots
    assert api.cs1_kv_rows(table(), N, N, 1, 0, N, N, N) == 0
    assert api.cs1_kv_trim(table(), N, N, 1, A, N) == INVALID
    assert api.cs1_kv_trim(table(), N, A, 1, N, N) == INVALID


def test_prep(api):
    def call(qg=A, kr=A, v=A, ld=8192 + 2048, qw=A, kw=A, freqs=A, dims=64, pages=None, pos=A, slot=A, q=A, gate=A, kp=A, vp=A,
             T=1, hq=16, hk=4, dh=256):
        rot = hip.Rotary(freqs, dims, 0, 1.0)
        return api.cs1_attn_prep_paged(qg, kr, v, ld, qw, kw, 1e-6, ctypes.byref(rot), pages or table(), pos, slot, q, gate, kp, vp,
                                       T, hq, hk, dh, N)

    assert call(T=-1) == INVALID and call(hq=0) == INVALID and call(hk=0) == INVALID and call(dh=64) == INVALID
    assert call(ld=8191) == INVALID and call(ld=8184) == INVALID and call(ld=4096) == INVALID
    assert call(ld=4088, gate=N) == INVALID
    assert call(dims=8) == INVALID and call(dims=-16) == INVALID and call(dims=272) == INVALID and call(dims=40) == INVALID
    assert call(freqs=N) == INVALID and call(freqs=A + 4) == INVALID
    assert call(pages=table(npages=0)) == INVALID and call(pages=table(npages=1 << 27)) == INVALID
    assert call(hk=1 << 17, dh=256, ld=1 << 26) == INVALID
    for name in ("qg", "kr", "v", "q", "kp", "vp"):
        assert call(**{name: N}) == INVALID and call(**{name: A + 8}) == INVALID, name
    for name in ("qw", "kw", "gate"):
        assert call(**{name: A + 8}) == INVALID, name
    assert call(pos=N) == INVALID and call(slot=N) == INVALID
    assert api.cs1_attn_prep_paged(A, A, A, 8192, A, A, 1e-6, N, table(), A, A, A, A, A, A, 1, 16, 4, 256, N) == INVALID
    assert call(T=0, qg=N, q=N) == 0


def freqs_of(api, dims, *args):
    f = np.full(dims // 2 + 1, 7.0)
    assert api.cs1_rotary_freqs(f.ctypes.data, dims, *args) == 0
    assert f[-1] == 7.0
    return f[:-1]


def test_rotary_freqs(api):
    f = freqs_of(api, 64, 1e7, 1.0, 32768.0, 1.0, 32.0)
    plain = 1e7 ** (-np.arange(0, 64, 2) / 64)
    np.testing.assert_allclose(f, plain, rtol=1e-14)
    np.testing.assert_allclose(freqs_of(api, 64, 1e7, 8.0, 32768.0, 1.0, math.inf), plain / 8, rtol=1e-14)
    f = freqs_of(api, 128, 1e4, 4.0, 4096.0, 1.0, 32.0)
    plain = 1e4 ** (-np.arange(0, 128, 2) / 128)
    turns = 4096 * plain / (2 * math.pi)
    ramp = np.clip((turns - 1) / 31, 0, 1)
    np.testing.assert_allclose(f, plain * (ramp + (1 - ramp) / 4), rtol=1e-13)
    same = freqs_of(api, 128, 1e4, 1.0, 4096.0, 1.0, 32.0)
    assert (f[turns >= 32] == same[turns >= 32]).all() and (turns <= 1).any() and (turns >= 32).any()
    # an edge without a slope: all or nothing
    f = freqs_of(api, 128, 1e4, 4.0, 4096.0, 5.0, 5.0)
    np.testing.assert_allclose(f, np.where(turns >= 5, plain, plain / 4), rtol=1e-14)


def test_rotary_refusals(api):
    f = np.zeros(64)
    ok = (f.ctypes.data, 64, 1e4, 2.0, 4096.0, 1.0, 32.0)
    assert api.cs1_rotary_freqs(*ok) == 0
    for i, bad in ((0, N), (1, 0), (1, -2), (1, 63), (2, 0.0), (2, math.nan), (3, 0.5), (3, math.nan), (4, 0.0), (5, -1.0), (6, 0.5),
                   (6, math.nan)):
        args = list(ok)
        args[i] = bad
        assert api.cs1_rotary_freqs(*args) == INVALID, (i, bad)


def test_logprobs(api):
    def call(x=A, f32=0, ld=1000, targets=A, rows=2, V=1000, k=5, lp=A, ent=A, ids=A, top=A, ws=A):
        return api.cs1_token_logprobs(x, f32, ld, targets, rows, V, k, lp, ent, ids, top, ws, N)

    assert call(rows=-1) == INVALID and call(V=0) == INVALID and call(V=(1 << 28) + 1, ld=1 << 29) == INVALID
    assert call(ld=999) == INVALID and call(k=-1) == INVALID and call(k=33) == INVALID
    assert call(x=N) == INVALID and call(x=A + 1) == INVALID and call(x=A + 2, f32=1) == INVALID
    assert call(targets=N) == INVALID and call(lp=N) == INVALID  # both or neither
    assert call(ids=N) == INVALID and call(top=N) == INVALID
    assert call(V=100000, ld=100000, ws=N) == INVALID and call(V=100000, ld=100000, ws=A + 8) == INVALID
    assert call(rows=0, x=N) == 0
    size = api.cs1_token_logprobs_workspace_bytes
    assert size(0, 1000, 5) == 0 and size(2, 0, 5) == 0 and size(2, 1000, 33) == 0 and size(2, 1000, 5) == 0
    assert size(1, 248320, 20) > 0 and size(5000, 248320, 20) == 0


def test_attention(api):
    def call(h=N, q=A, kp=A, vp=A, t=None, cu=A, n=1, most=4, gate=A, out=A, rows=4, hq=16, hk=4, dh=128, scale=0.1):
        return api.cs1_attention_paged_varlen(h, q, kp, vp, t or table(), N, cu, n, most, gate, out, N, rows, hq, hk, dh, scale, N)

    assert call() == INVALID  # no handle
    # a handle is looked into last: for work that there is, on operands that are right
    for bad in BAD_TABLES:
        assert call(h=A, t=table(**bad)) == INVALID, bad
    for kw in (dict(dh=64), dict(hk=0), dict(hq=0), dict(hq=15), dict(hq=516), dict(n=-1), dict(n=8193), dict(rows=-1), dict(most=-1),
               dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(rows=(1 << 20) + 1),
               dict(hq=1 << 18, hk=1 << 18, rows=1, dh=128), dict(t=table(npages=1 << 27))):
        assert call(h=A, **kw) == INVALID, kw
    for name in ("q", "kp", "vp", "out"):
        assert call(h=A, **{name: N}) == INVALID and call(h=A, **{name: A + 8}) == INVALID, name
    assert call(h=A, gate=A + 8) == INVALID and call(h=A, cu=N) == INVALID
    assert call(h=A, rows=0, q=N) == 0 and call(h=A, n=0, cu=N) == 0 and call(h=A, most=0) == 0
