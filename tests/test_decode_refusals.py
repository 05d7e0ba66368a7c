"""The decode operations refuse what they cannot do before any device work, and accept empty work."""
import ctypes

import pytest

from qwen3_5_native import hip

INVALID = hip.HIP_ERROR_INVALID_VALUE
N = None
A = 1 << 20  # an aligned address that is never followed: every call here returns before a launch


@pytest.fixture(scope="module")
def api():
    return hip.load()


def table(**kw):
    f = dict(table=A, lens=A, refs=A, nseq=4, max_pages=8, npages=16, page=16)
    f.update(kw)
    return ctypes.byref(hip.PageTable(*[f[n] for n, _ in hip.PageTable._fields_]))


BAD_TABLES = [dict(table=N), dict(lens=N), dict(refs=N), dict(nseq=0), dict(nseq=8193), dict(max_pages=0), dict(npages=0),
              dict(page=0), dict(page=8), dict(page=24), dict(page=1 << 16, max_pages=1 << 15), dict(npages=-1)]


@pytest.mark.parametrize("bad", BAD_TABLES, ids=str)
def test_bad_tables(api, bad):
    t = table(**bad)
    pools = (ctypes.c_void_p * 1)(A)
    assert api.cs1_kv_reserve(t, N, N, 0, A, N) == INVALID
    assert api.cs1_kv_write(t, N, N, 0, N, 512, N, 512, N, N, 4, 128, N) == INVALID
    assert api.cs1_kv_fork(t, A, A, 1, pools, 1, 16, A, A, N) == INVALID
    assert api.cs1_kv_free(t, N, 0, N) == INVALID
    assert api.cs1_kv_compact(t, pools, 1, 16, A, A, N) == INVALID
    assert api.cs1_attention_paged(A, N, N, N, t, N, N, N, N, 0, 16, 4, 128, 1.0, N) == INVALID


def test_no_table(api):
    assert api.cs1_kv_reserve(N, N, N, 0, A, N) == INVALID
    assert api.cs1_kv_free(N, N, 0, N) == INVALID


def test_reserve(api):
    cu = (ctypes.c_int32 * 66)(*range(66))
    assert api.cs1_kv_reserve(table(), N, N, -1, A, N) == INVALID
    assert api.cs1_kv_reserve(table(), N, N, 8193, A, N) == INVALID
    assert api.cs1_kv_reserve(table(), N, N, 1, N, N) == INVALID  # no status
    assert api.cs1_kv_reserve(table(), N, cu, 65, A, N) == INVALID  # offsets of at most 64
    assert api.cs1_kv_reserve(table(), N, (ctypes.c_int32 * 3)(0, 3, 2), 2, A, N) == INVALID
    assert api.cs1_kv_reserve(table(), N, (ctypes.c_int32 * 3)(1, 3, 4), 2, A, N) == INVALID


def test_write(api):
    def call(t=None, cu=N, n=1, k=A, ldk=512, v=A, ldv=512, kp=A, vp=A, hk=4, dh=128):
        return api.cs1_kv_write(t or table(), N, cu, n, k, ldk, v, ldv, kp, vp, hk, dh, N)

    assert call(n=-1) == INVALID and call(n=8193) == INVALID
    assert call(hk=0) == INVALID and call(dh=0) == INVALID and call(hk=1, dh=4, ldk=8, ldv=8) == INVALID
    assert call(ldk=511) == INVALID and call(ldk=504) == INVALID and call(ldv=504) == INVALID and call(ldv=516) == INVALID
    for name in ("k", "v", "kp", "vp"):
        assert call(**{name: N}) == INVALID and call(**{name: A + 8}) == INVALID, name
    assert call(cu=(ctypes.c_int32 * 3)(0, 3, 2), n=2) == INVALID
    assert call(cu=(ctypes.c_int32 * 2)(0, 1 << 24), n=1) == INVALID  # more rows than a launch takes
    assert call(n=0, k=N, v=N, kp=N, vp=N) == 0
    assert call(cu=(ctypes.c_int32 * 3)(0, 0, 0), n=2, k=N) == 0


def test_fork(api):
    pools = (ctypes.c_void_p * 2)(A, A)

    def call(src=A, dst=A, n=1, pools=pools, npools=2, row=1024, ws=A, status=A):
        return api.cs1_kv_fork(table(), src, dst, n, pools, npools, row, ws, status, N)

    assert call(n=-1) == INVALID and call(n=8193) == INVALID and call(src=N) == INVALID and call(dst=N) == INVALID
    assert call(row=0) == INVALID and call(row=1000) == INVALID and call(npools=-1) == INVALID
    assert call(pools=N) == INVALID and call(ws=N) == INVALID and call(ws=A + 4) == INVALID and call(status=N) == INVALID
    assert call(pools=(ctypes.c_void_p * 2)(A, N)) == INVALID
    assert call(pools=(ctypes.c_void_p * 2)(A, A + 4)) == INVALID
    assert call(row=1 << 33) == INVALID


def test_free_and_compact(api):
    pools = (ctypes.c_void_p * 1)(A)
    assert api.cs1_kv_free(table(), N, -1, N) == INVALID
    assert api.cs1_kv_free(table(), N, 8193, N) == INVALID
    assert api.cs1_kv_free(table(), N, 0, N) == 0
    assert api.cs1_kv_compact(table(), pools, 1, 1000, A, A, N) == INVALID
    assert api.cs1_kv_compact(table(), pools, 1, 1024, N, A, N) == INVALID
    assert api.cs1_kv_compact(table(), pools, 1, 1024, A, N, N) == INVALID
    assert api.cs1_kv_compact(table(), N, 1, 1024, A, A, N) == INVALID


def test_copy(api):
    pools = (ctypes.c_void_p * 1)(A)
    assert api.cs1_kv_copy(pools, 1, 24, 4, A, A, 1, N) == INVALID
    assert api.cs1_kv_copy(pools, 1, 16, -1, A, A, 1, N) == INVALID
    assert api.cs1_kv_copy(pools, 1, 16, 4, A, A, -1, N) == INVALID
    assert api.cs1_kv_copy(pools, 1, 16, 4, A, A, 8193, N) == INVALID
    assert api.cs1_kv_copy(pools, 1, 16, 4, N, A, 1, N) == INVALID
    assert api.cs1_kv_copy(pools, 1, 16, 4, A, N, 1, N) == INVALID
    assert api.cs1_kv_copy((ctypes.c_void_p * 1)(A + 8), 1, 16, 4, A, A, 1, N) == INVALID
    assert api.cs1_kv_copy(pools, 1, 16, 4, N, N, 0, N) == 0
    assert api.cs1_kv_copy(N, 0, 16, 4, A, A, 1, N) == 0
    assert api.cs1_kv_copy(pools, 1, 16, 0, A, A, 1, N) == 0


def test_workspace(api):
    assert api.cs1_kv_workspace_bytes(100, 10) >= 4 * (200 + 40)
    assert api.cs1_kv_workspace_bytes(0, 0) > 0
    assert api.cs1_kv_workspace_bytes(-1, 0) == 0


def test_attention_without_a_handle(api):
    assert api.cs1_attention_paged(N, A, A, A, table(), N, N, A, N, 1, 16, 4, 128, 1.0, N) == INVALID
    api.cs1_attention_paged_destroy(N)


def test_gdn_decode(api):
    def call(x=A, ld=8256, w=A, z=A, b=A, a=A, al=A, dt=A, gw=A, ring=A, state=A, lens=A, nseq=4, out=A, B=1, H=32, HK=16):
        return api.cs1_gdn_decode(x, ld, w, z, b, a, al, dt, gw, 1e-6, ring, state, N, lens, nseq, out, B, H, HK, 0.1, N)

    assert call(B=-1) == INVALID and call(B=8193) == INVALID and call(H=0) == INVALID and call(HK=0) == INVALID
    assert call(H=24) == INVALID and call(nseq=0) == INVALID and call(ld=8191) == INVALID
    assert call(z=N) == INVALID and call(gw=N) == INVALID  # both or neither
    for name in ("x", "w", "b", "a", "al", "dt", "ring", "state", "lens", "out"):
        assert call(**{name: N}) == INVALID, name
    assert call(state=A + 4) == INVALID and call(w=A + 2) == INVALID and call(out=A + 4) == INVALID
    assert call(B=0, x=N, out=N) == 0


@pytest.mark.parametrize("npages", [(1 << 30) + 1, 2 ** 31 - 4096, 2 ** 31 - 1])
def test_more_pages_than_are_counted_in_32_bits(api, npages):
    """The scans over the counts step past the last page, and compaction's plan has half as many entries again behind it."""
    t = table(npages=npages)
    assert api.cs1_kv_reserve(t, N, N, 0, A, N) == INVALID
    assert api.cs1_kv_write(t, N, N, 0, N, 512, N, 512, N, N, 4, 128, N) == INVALID
    assert api.cs1_kv_fork(t, N, N, 0, N, 0, 16, N, A, N) == INVALID
    assert api.cs1_kv_free(t, N, 0, N) == INVALID
    assert api.cs1_kv_compact(t, N, 0, 16, A, A, N) == INVALID
    assert api.cs1_attention_paged(A, N, N, N, t, N, N, N, N, 0, 16, 4, 128, 1.0, N) == INVALID


def test_as_many_pages_as_are_counted(api):
    assert api.cs1_kv_write(table(npages=1 << 30), N, N, 0, N, 512, N, 512, N, N, 4, 128, N) == 0
    assert api.cs1_kv_free(table(npages=1 << 30), N, 0, N) == 0
