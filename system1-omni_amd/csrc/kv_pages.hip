// The pages of a key-value cache on the device (cs1_kv_*): room for new tokens, their keys and values,
// forks that share whole pages, the end of sequences, compaction, and copies of whole entries.
//
// All bookkeeping is whole numbers in device memory and every result is a function of the arguments: the
// pages that a list of sequences receives are the lowest-numbered free ones in the list's order.
// With need_i new pages for entry i and off_i the sum of the needs before it, the free page with k
// free pages below it goes to the entry with off_i <= k < off_i + need_i.  One block of 1024 threads does
// that: a scan over the needs, then scans over 4096 counts at a time until enough pages are found.
// What moves keys and values is a kernel of its own that fills the chip: 16-byte accesses, a page's
// filled rows being one run of bytes in each pool.
#include "common.h"
#include "paged.h"

namespace q35 {
namespace {

constexpr int PLAN_THREADS = 1024, PLAN_WAVES = PLAN_THREADS / 64;
constexpr int PER = MAX_LISTED / PLAN_THREADS;  // list entries a thread has at most
constexpr int SEQS_MAX = 64, POOLS_MAX = 64;    // offsets and pools that travel with a launch
constexpr int MOVE_THREADS = 256;

struct Offsets {
    int32_t at[SEQS_MAX + 1];
    int n;  // 0: every entry has one row
};

struct Pools {
    char* p[POOLS_MAX];
};

// Sum of x over the threads before this one; total: over all. red: PLAN_WAVES + 1 ints of LDS, free before
// the call and after the next barrier.
__device__ __forceinline__ int block_scan(int x, int* red, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int sum = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int below = __shfl_up(sum, o, 64);
        if (lane >= o) sum += below;
    }
    __syncthreads();
    if (lane == 63) red[wave] = sum;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < PLAN_WAVES; w++) {
        const int r = red[w];
        if (w < wave) before += r;
        total += r;
    }
    return before + sum - x;
}

__device__ __forceinline__ int pages_of(int64_t tokens, int page) { return (int)((tokens + page - 1) / page); }

// The entry with off[i] <= k < off[i] + need: the last one with off[i] <= k.
__device__ __forceinline__ int entry_of(const int* off, int n, int k) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (off[mid] <= k)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

// Calls take(k, page) for the `total` lowest free pages, k = 0 .., or for all there are; returns their number.
template <typename Take>
__device__ __forceinline__ int take_free(const int32_t* refs, int npages, int total, int* red, Take take) {
    int found = 0;
    for (int base = 0; base < npages && found < total; base += 4 * PLAN_THREADS) {
        const int p = base + 4 * threadIdx.x;
        bool free[4];
        int mine = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            free[e] = p + e < npages && refs[p + e] == 0;
            mine += free[e];
        }
        int all, k = found + block_scan(mine, red, all);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (free[e]) {
                if (k < total) take(k, p + e);
                k++;
            }
        found = min(total, found + all);
    }
    return found;
}

__global__ void __launch_bounds__(PLAN_THREADS)
    kv_reserve_kernel(const Cs1PageTable t, const int32_t* __restrict__ seqs, const Offsets cu, int n, int32_t* status) {
    __shared__ int work[MAX_LISTED];  // first entry that names a sequence, then the offsets off_i
    __shared__ int red[PLAN_WAVES];
    const int tid = threadIdx.x;
    for (int s = tid; s < t.nseq; s += PLAN_THREADS) work[s] = n;
    __syncthreads();
    for (int i = tid; i < n; i += PLAN_THREADS) {
        const int s = listed_seq(seqs, i, t.nseq);
        if (s >= 0) atomicMin(&work[s], i);
    }
    __syncthreads();
    const int per = (n + PLAN_THREADS - 1) / PLAN_THREADS, i0 = tid * per;
    int need[PER], mine = 0;
    uint32_t has = 0;  // the entries that have their sequence
    bool wide = false;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int i = i0 + e;
        need[e] = 0;
        if (e >= per || i >= n) continue;
        const int s = listed_seq(seqs, i, t.nseq);
        if (s < 0 || work[s] != i) continue;
        has |= 1u << e;
        const int64_t len = max(t.lens[s], 0), to = len + (cu.n ? cu.at[i + 1] - cu.at[i] : 1);
        if (to > (int64_t)t.max_pages * t.page) {
            wide = true;
            continue;
        }
        need[e] = pages_of(to, t.page) - pages_of(len, t.page);
        mine += need[e];
    }
    if (__syncthreads_or(wide)) {
        if (tid == 0) *status = -1;
        return;
    }
    int total, off = block_scan(mine, red, total);
#pragma unroll
    for (int e = 0; e < PER; e++) {
        if (e < per && i0 + e < n) work[i0 + e] = off;
        off += need[e];
    }
    __syncthreads();
    auto slot = [&](int k) {  // the table entry for new page k
        const int i = entry_of(work, n, k), s = listed_seq(seqs, i, t.nseq);
        return t.table + (size_t)s * t.max_pages + pages_of(max(t.lens[s], 0), t.page) + (k - work[i]);
    };
    const int found = take_free(t.refs, t.npages, total, red, [&](int k, int p) {
        *slot(k) = p;
        t.refs[p] = 1;
    });
    if (found < total) {  // give back what was taken
        __syncthreads();
        for (int k = tid; k < found; k += PLAN_THREADS) {
            int32_t* const e = slot(k);
            t.refs[*e] = 0;
            *e = -1;
        }
    } else {
        __syncthreads();  // slot() has read the lengths
#pragma unroll
        for (int e = 0; e < PER; e++)
            if (has >> e & 1) {
                const int i = i0 + e;
                int32_t* const len = t.lens + listed_seq(seqs, i, t.nseq);
                *len = max(*len, 0) + (cu.n ? cu.at[i + 1] - cu.at[i] : 1);
            }
    }
    if (tid == 0) *status = total - found;
}

// One block a row: its keys by the first half of the threads, its values by the second.
__global__ void __launch_bounds__(MOVE_THREADS)
    kv_write_kernel(const Cs1PageTable t, const int32_t* __restrict__ seqs, const Offsets cu, int first,
                    const bf16* __restrict__ k, int ldk, const bf16* __restrict__ v, int ldv, char* kp, char* vp,
                    int width) {
    const int r = blockIdx.x;
    int i = r, back = 1;  // list entry, and how far from the end of its sequence the row is
    if (cu.n) {
        i = 0;
        while (i + 1 < cu.n && r >= cu.at[i + 1] - cu.at[0]) i++;
        back = cu.at[i + 1] - cu.at[0] - r;
        i += first;
    }
    const int s = listed_seq(seqs, i, t.nseq);
    if (s < 0) return;
    const bool again = named_before(seqs, i, s);
    const int pos = t.lens[s] - back;
    if (__syncthreads_or(again) || pos < 0 || pos / t.page >= t.max_pages) return;
    const int pg = t.table[(size_t)s * t.max_pages + pos / t.page];
    if (pg < 0 || pg >= t.npages) return;
    const size_t row = cu.n ? (size_t)cu.at[0] + r : (size_t)r;
    const size_t to = ((size_t)pg * t.page + pos % t.page) * width * 2;
    const bool value = threadIdx.x >= MOVE_THREADS / 2;
    const char* const from = reinterpret_cast<const char*>(value ? v + row * ldv : k + row * ldk);
    char* const at = (value ? vp : kp) + to;
    for (int e = (threadIdx.x % (MOVE_THREADS / 2)) * 16; e < width * 2; e += MOVE_THREADS / 2 * 16)
        *reinterpret_cast<u32x4*>(at + e) = *reinterpret_cast<const u32x4*>(from + e);
}

// What a fork does for one pair: the last page that is not full (rows of it, 0: none), copied from `from` to `to`.
struct Pair {
    int32_t on, from, to, rows;
};

__global__ void __launch_bounds__(PLAN_THREADS)
    kv_fork_plan_kernel(const Cs1PageTable t, const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int n,
                        Pair* __restrict__ plan, int32_t* status) {
    __shared__ int work[MAX_LISTED];
    __shared__ int red[PLAN_WAVES];
    const int tid = threadIdx.x;
    for (int s = tid; s < t.nseq; s += PLAN_THREADS) work[s] = n;
    __syncthreads();
    for (int i = tid; i < n; i += PLAN_THREADS) {
        const int d = listed_seq(dst, i, t.nseq);
        if (d >= 0) atomicMin(&work[d], i);
    }
    __syncthreads();
    const int per = (n + PLAN_THREADS - 1) / PLAN_THREADS, i0 = tid * per;
    Pair mine[PER];
    int need = 0;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int i = i0 + e;
        mine[e] = Pair{0, -1, -1, 0};
        if (e >= per || i >= n) continue;
        const int s = listed_seq(src, i, t.nseq), d = listed_seq(dst, i, t.nseq);
        if (s < 0 || d < 0 || work[d] != i || work[s] != n || t.lens[d] > 0) continue;
        const int len = t.lens[s];
        if (len <= 0 || pages_of(len, t.page) > t.max_pages) continue;
        mine[e].on = 1;
        mine[e].rows = len % t.page;
        if (mine[e].rows) mine[e].from = t.table[(size_t)s * t.max_pages + len / t.page];
        need += mine[e].rows > 0;
    }
    int total, off = block_scan(need, red, total);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; e++) {
        if (e < per && i0 + e < n) {
            work[i0 + e] = off;
            plan[i0 + e] = mine[e];
        }
        off += mine[e].rows > 0;
    }
    __syncthreads();
    const int found = take_free(t.refs, t.npages, total, red, [&](int k, int p) {
        plan[entry_of(work, n, k)].to = p;
        t.refs[p] = 1;
    });
    if (found < total) {
        __syncthreads();
        for (int i = tid; i < n; i += PLAN_THREADS) {
            if (plan[i].to >= 0) t.refs[plan[i].to] = 0;
            plan[i].on = plan[i].rows = 0;
        }
    }
    if (tid == 0) *status = total - found;
}

// Blocks y = 0 of the first launch: the pair's row of the table, the shared pages' counts, the length. The others: the
// filled rows of the unfinished page, in pool y - 1, CHUNK bytes a block.
constexpr int FORK_CHUNK = MOVE_THREADS * 16 * 4;

__global__ void __launch_bounds__(MOVE_THREADS)
    kv_fork_kernel(const Cs1PageTable t, const int32_t* __restrict__ src, const int32_t* __restrict__ dst,
                   const Pair* __restrict__ plan, const Pools pools, size_t row_bytes, int tables) {
    const Pair pr = plan[blockIdx.z];
    if (!pr.on) return;
    const int pool = (int)blockIdx.y - tables;
    if (pool < 0) {
        if (blockIdx.x > 0) return;
        const int s = src[blockIdx.z], d = dst[blockIdx.z], len = t.lens[s], full = len / t.page;
        for (int j = threadIdx.x; j < full; j += MOVE_THREADS) {
            const int p = t.table[(size_t)s * t.max_pages + j];
            t.table[(size_t)d * t.max_pages + j] = p;
            if (p >= 0 && p < t.npages) atomicAdd(&t.refs[p], 1);
        }
        if (threadIdx.x == 0) {
            if (pr.rows) t.table[(size_t)d * t.max_pages + full] = pr.to;
            t.lens[d] = len;
        }
        return;
    }
    if (pr.from < 0 || pr.from >= t.npages) return;
    const size_t bytes = pr.rows * row_bytes, page_bytes = t.page * row_bytes;
    const size_t end = min(bytes, ((size_t)blockIdx.x + 1) * FORK_CHUNK);
    const char* const from = pools.p[pool] + pr.from * page_bytes;
    char* const to = pools.p[pool] + pr.to * page_bytes;
    for (size_t e = (size_t)blockIdx.x * FORK_CHUNK + threadIdx.x * 16; e < end; e += MOVE_THREADS * 16)
        *reinterpret_cast<u32x4*>(to + e) = *reinterpret_cast<const u32x4*>(from + e);
}

__global__ void __launch_bounds__(MOVE_THREADS)
    kv_free_kernel(const Cs1PageTable t, const int32_t* __restrict__ seqs) {
    const int i = blockIdx.x, s = listed_seq(seqs, i, t.nseq);
    if (s < 0) return;
    if (__syncthreads_or(named_before(seqs, i, s))) return;
    int32_t* const row = t.table + (size_t)s * t.max_pages;
    const int held = min(pages_of(max(t.lens[s], 0), t.page), t.max_pages);
    for (int j = threadIdx.x; j < held; j += MOVE_THREADS) {
        const int p = row[j];
        if (p >= 0 && p < t.npages) atomicSub(&t.refs[p], 1);
    }
    __syncthreads();
    for (int j = threadIdx.x; j < t.max_pages; j += MOVE_THREADS) row[j] = -1;
    if (threadIdx.x == 0) t.lens[s] = 0;
}

// Compaction's plan: ws[0] the number of moves, ws[1] the held pages L, ws[2] .. the held pages from L on in
// ascending order, ws[2 + npages] .. the free pages before L.
__global__ void __launch_bounds__(PLAN_THREADS)
    kv_compact_plan_kernel(const Cs1PageTable t, int32_t* __restrict__ ws, int32_t* status) {
    __shared__ int red[PLAN_WAVES];
    int mine = 0;
    for (int p = threadIdx.x; p < t.npages; p += PLAN_THREADS) mine += t.refs[p] != 0;
    int held;
    (void)block_scan(mine, red, held);
    int moved = 0, holes = 0;
    for (int base = 0; base < t.npages; base += 4 * PLAN_THREADS) {
        const int p = base + 4 * threadIdx.x;
        bool live[4];
        int count = 0;  // pages to move in the upper half, free ones before L in the lower
#pragma unroll
        for (int e = 0; e < 4; e++) {
            live[e] = p + e < t.npages && t.refs[p + e] != 0;
            if (p + e < held)
                count += !live[e];
            else
                count += live[e] ? 1 << 16 : 0;
        }
        int all;
        const int before = block_scan(count, red, all);
        int m = moved + (before >> 16), f = holes + (before & 0xffff);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (p + e < held) {
                if (!live[e]) ws[2 + t.npages + f++] = p + e;
            } else if (live[e]) {
                ws[2 + m++] = p + e;
            }
        }
        moved += all >> 16;
        holes += all & 0xffff;
    }
    if (threadIdx.x == 0) {
        ws[0] = moved;
        ws[1] = held;
        *status = held;
    }
}

constexpr int COMPACT_CHUNK = MOVE_THREADS * 16 * 4;

// Blocks before `tables`: a sequence's row of the table each. The others move pages, a chunk at a time.
__global__ void __launch_bounds__(MOVE_THREADS)
    kv_compact_kernel(const Cs1PageTable t, const int32_t* __restrict__ ws, const Pools pools, int npools,
                      size_t page_bytes, int tables) {
    const int moves = ws[0], held = ws[1];
    const int32_t* const from = ws + 2;
    const int32_t* const to = ws + 2 + t.npages;
    if ((int)blockIdx.x < tables) {
        const int s = blockIdx.x;
        int32_t* const row = t.table + (size_t)s * t.max_pages;
        const int n = min(pages_of(max(t.lens[s], 0), t.page), t.max_pages);
        for (int j = threadIdx.x; j < n; j += MOVE_THREADS) {
            const int p = row[j];
            if (p < held || p >= t.npages) continue;
            const int k = entry_of(from, moves, p);
            if (moves > 0 && from[k] == p) row[j] = to[k];
        }
        return;
    }
    const int block = (int)blockIdx.x - tables, blocks = (int)gridDim.x - tables;
    if (tables > 0)  // the first launch of a call
        for (int k = block * MOVE_THREADS + threadIdx.x; k < moves; k += blocks * MOVE_THREADS) {
            t.refs[to[k]] = t.refs[from[k]];
            t.refs[from[k]] = 0;
        }
    const int chunks = (int)((page_bytes + COMPACT_CHUNK - 1) / COMPACT_CHUNK);
    const int64_t items = (int64_t)moves * npools * chunks;
    for (int64_t it = block; it < items; it += blocks) {
        const int chunk = (int)(it % chunks), pool = (int)(it / chunks % npools), k = (int)(it / chunks / npools);
        const char* const a = pools.p[pool] + from[k] * page_bytes;
        char* const b = pools.p[pool] + to[k] * page_bytes;
        const size_t end = min(page_bytes, ((size_t)chunk + 1) * COMPACT_CHUNK);
        for (size_t e = (size_t)chunk * COMPACT_CHUNK + threadIdx.x * 16; e < end; e += MOVE_THREADS * 16)
            *reinterpret_cast<u32x4*>(b + e) = *reinterpret_cast<const u32x4*>(a + e);
    }
}

constexpr int COPY_CHUNK = MOVE_THREADS * 16 * 4;

// Block: a chunk (x) of pair z's entry in pool y.
__global__ void __launch_bounds__(MOVE_THREADS)
    kv_copy_kernel(const Pools pools, size_t bytes, int entries, const int32_t* __restrict__ src,
                   const int32_t* __restrict__ dst, int n) {
    const int i = blockIdx.z, s = src[i], d = dst[i];
    if (s < 0 || s >= entries || d < 0 || d >= entries) return;
    bool out = false;
    for (int j = threadIdx.x; j < n; j += MOVE_THREADS) {
        const int other = dst[j];
        out |= other == s || (j < i && other == d);
    }
    if (__syncthreads_or(out)) return;
    const char* const a = pools.p[blockIdx.y] + s * bytes;
    char* const b = pools.p[blockIdx.y] + d * bytes;
    const size_t end = min(bytes, ((size_t)blockIdx.x + 1) * COPY_CHUNK);
    for (size_t e = (size_t)blockIdx.x * COPY_CHUNK + threadIdx.x * 16; e < end; e += MOVE_THREADS * 16)
        *reinterpret_cast<u32x4*>(b + e) = *reinterpret_cast<const u32x4*>(a + e);
}

// Nondecreasing HOST offsets from 0.
bool offsets_ok(const int32_t* cu, int n) {
    if (!cu) return true;
    if (cu[0] != 0) return false;
    for (int i = 0; i < n; i++)
        if (cu[i + 1] < cu[i]) return false;
    return true;
}

bool pools_ok(void* const* pools, int npools) {
    if (npools < 0 || (npools > 0 && !pools)) return false;
    for (int i = 0; i < npools; i++)
        if (!pools[i] || !on16(pools[i])) return false;
    return true;
}

// Up to POOLS_MAX of them from number `first` on; their count.
int some_pools(void* const* pools, int npools, int first, Pools& out) {
    const int n = npools - first < POOLS_MAX ? npools - first : POOLS_MAX;
    for (int i = 0; i < n; i++) out.p[i] = static_cast<char*>(pools[first + i]);
    return n;
}

constexpr size_t CHUNKS_MAX = 1u << 22;  // of an entry, a grid's x
constexpr int ROWS_MAX = 1 << 23;         // of one launch

}  // namespace
}  // namespace q35

using namespace q35;

extern "C" int cs1_kv_reserve(const Cs1PageTable* pages, const int32_t* seqs, const int32_t* cu_seqlens, int n,
                              int32_t* status, void* stream) {
    if (!table_ok(pages) || n < 0 || n > MAX_LISTED || !status) return hipErrorInvalidValue;
    if (cu_seqlens && (n > SEQS_MAX || !offsets_ok(cu_seqlens, n))) return hipErrorInvalidValue;
    Offsets cu;
    cu.n = cu_seqlens ? n : 0;
    if (cu_seqlens)
        for (int i = 0; i <= n; i++) cu.at[i] = cu_seqlens[i];
    kv_reserve_kernel<<<1, PLAN_THREADS, 0, static_cast<hipStream_t>(stream)>>>(*pages, seqs, cu, n, status);
    return hipGetLastError();
}

extern "C" int cs1_kv_write(const Cs1PageTable* pages, const int32_t* seqs, const int32_t* cu_seqlens, int n,
                            const void* k, int ldk, const void* v, int ldv, void* kp, void* vp, int Hk, int Dh,
                            void* stream) {
    if (!table_ok(pages) || n < 0 || n > MAX_LISTED || Hk <= 0 || Dh <= 0 || !offsets_ok(cu_seqlens, n))
        return hipErrorInvalidValue;
    const int64_t width = (int64_t)Hk * Dh;
    if (width % 8 != 0 || width > (1 << 24) || ldk % 8 != 0 || ldv % 8 != 0 || ldk < width || ldv < width)
        return hipErrorInvalidValue;
    if (n == 0 || (cu_seqlens && cu_seqlens[n] == 0)) return hipSuccess;
    if (cu_seqlens && cu_seqlens[n] > ROWS_MAX) return hipErrorInvalidValue;
    if (!all_set({k, v, kp, vp}) || !on16(k) || !on16(v) || !on16(kp) || !on16(vp)) return hipErrorInvalidValue;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    auto launch = [&](const Offsets& cu, int first, int rows) {
        kv_write_kernel<<<rows, MOVE_THREADS, 0, st>>>(*pages, seqs, cu, first, static_cast<const bf16*>(k), ldk,
                                                       static_cast<const bf16*>(v), ldv, static_cast<char*>(kp),
                                                       static_cast<char*>(vp), (int)width);
        return hipGetLastError();
    };
    Offsets cu;
    cu.n = 0;
    if (!cu_seqlens) return launch(cu, 0, n);
    for (int s0 = 0; s0 < n; s0 += SEQS_MAX) {
        cu.n = n - s0 < SEQS_MAX ? n - s0 : SEQS_MAX;
        for (int i = 0; i <= cu.n; i++) cu.at[i] = cu_seqlens[s0 + i];
        const int rows = cu.at[cu.n] - cu.at[0];
        if (rows == 0) continue;
        const hipError_t e = launch(cu, s0, rows);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

extern "C" size_t cs1_kv_workspace_bytes(int npages, int n) {
    if (npages < 0 || n < 0) return 0;
    return 4 * (2 * (size_t)npages + 4 * (size_t)n + 64);
}

extern "C" int cs1_kv_fork(const Cs1PageTable* pages, const int32_t* src, const int32_t* dst, int n, void* const* pools,
                           int npools, size_t row_bytes, void* workspace, int32_t* status, void* stream) {
    if (!table_ok(pages) || n < 0 || n > MAX_LISTED || !pools_ok(pools, npools) || !status) return hipErrorInvalidValue;
    if (npools > 0 && (row_bytes == 0 || row_bytes % 16 != 0 || row_bytes > ((size_t)1 << 32))) return hipErrorInvalidValue;
    const size_t chunks = npools > 0 ? ((pages->page - 1) * row_bytes + FORK_CHUNK - 1) / FORK_CHUNK : 1;
    if (chunks > CHUNKS_MAX) return hipErrorInvalidValue;
    if (n > 0 && (!all_set({src, dst, workspace}) || !on16(workspace))) return hipErrorInvalidValue;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    Pair* const plan = static_cast<Pair*>(workspace);
    kv_fork_plan_kernel<<<1, PLAN_THREADS, 0, st>>>(*pages, src, dst, n, plan, status);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || n == 0) return e;
    int first = 0;
    do {
        Pools some = {};
        const int k = some_pools(pools, npools, first, some), tables = first == 0;
        kv_fork_kernel<<<dim3((unsigned)chunks, k + tables, n), MOVE_THREADS, 0, st>>>(*pages, src, dst, plan, some,
                                                                                      row_bytes, tables);
        e = hipGetLastError();
        first += k;
    } while (first < npools && e == hipSuccess);
    return e;
}

extern "C" int cs1_kv_free(const Cs1PageTable* pages, const int32_t* seqs, int n, void* stream) {
    if (!table_ok(pages) || n < 0 || n > MAX_LISTED) return hipErrorInvalidValue;
    if (n == 0) return hipSuccess;
    kv_free_kernel<<<n, MOVE_THREADS, 0, static_cast<hipStream_t>(stream)>>>(*pages, seqs);
    return hipGetLastError();
}

extern "C" int cs1_kv_compact(const Cs1PageTable* pages, void* const* pools, int npools, size_t row_bytes,
                              void* workspace, int32_t* status, void* stream) {
    if (!table_ok(pages) || !pools_ok(pools, npools) || !status || !workspace || !on16(workspace))
        return hipErrorInvalidValue;
    if (npools > 0 && (row_bytes == 0 || row_bytes % 16 != 0 || row_bytes > ((size_t)1 << 32))) return hipErrorInvalidValue;
    const size_t page_bytes = pages->page * row_bytes;
    if (npools > 0 && page_bytes / COMPACT_CHUNK > CHUNKS_MAX) return hipErrorInvalidValue;
    const int cus = device_cus();
    if (cus == 0) return hipErrorInvalidDevice;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    int32_t* const ws = static_cast<int32_t*>(workspace);
    kv_compact_plan_kernel<<<1, PLAN_THREADS, 0, st>>>(*pages, ws, status);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    int first = 0;
    do {
        Pools some = {};
        const int k = some_pools(pools, npools, first, some), tables = first == 0 ? pages->nseq : 0;
        kv_compact_kernel<<<tables + 8 * cus, MOVE_THREADS, 0, st>>>(*pages, ws, some, k, npools > 0 ? page_bytes : 0,
                                                                    tables);
        e = hipGetLastError();
        first += k;
    } while (first < npools && e == hipSuccess);
    return e;
}

extern "C" int cs1_kv_copy(void* const* pools, int npools, size_t entry_bytes, int entries, const int32_t* src,
                           const int32_t* dst, int n, void* stream) {
    if (!pools_ok(pools, npools) || n < 0 || n > MAX_LISTED || entries < 0 || entry_bytes % 16 != 0)
        return hipErrorInvalidValue;
    const size_t chunks = (entry_bytes + COPY_CHUNK - 1) / COPY_CHUNK;
    if (chunks > CHUNKS_MAX) return hipErrorInvalidValue;
    if (npools == 0 || n == 0 || entries == 0 || entry_bytes == 0) return hipSuccess;
    if (!all_set({src, dst})) return hipErrorInvalidValue;
    for (int first = 0; first < npools; first += POOLS_MAX) {
        Pools some = {};
        const int k = some_pools(pools, npools, first, some);
        kv_copy_kernel<<<dim3((unsigned)chunks, k, n), MOVE_THREADS, 0, static_cast<hipStream_t>(stream)>>>(
            some, entry_bytes, entries, src, dst, n);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
