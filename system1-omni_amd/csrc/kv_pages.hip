// The pages of a key-value cache on the device (cs1_kv_*): room for new tokens, their keys and values,
// forks that share whole pages, the end of sequences, compaction, and copies of whole entries.
//
// All bookkeeping is whole numbers in device memory and every result is a function of the arguments: the
// pages that a list of sequences receives are the lowest-numbered free ones in the list's order.
// With need_i new pages for entry i and off_i the sum of the needs before it, the free page with k
// free pages below it goes to the entry with off_i <= k < off_i + need_i.  One block of 1024 threads does
// that: a scan over the needs, then scans over 4096 counts, and then 16384 at a time, until enough pages are found.
// What moves keys and values is a kernel of its own that fills the chip: a page's filled rows are one run of bytes in
// each pool.
#include <algorithm>

#include "common.h"
#include "paged.h"

namespace q35 {
namespace {

constexpr int PLAN_THREADS = 1024, PLAN_WAVES = PLAN_THREADS / 64;
constexpr int PER_MAX = MAX_LISTED / PLAN_THREADS;  // list entries a thread has at most
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

// Counts of pages from `base` on: a wave has 64 N of them in a row, a lane every 64th.
constexpr int NEAR = 4, FAR = 16;
constexpr int DIRECT = 64;  // pages that are few
template <int N>
struct Counts {
    int of[N];
};
template <int N>
__device__ __forceinline__ Counts<N> page_counts(const int32_t* __restrict__ refs, int npages, int base) {
    Counts<N> c;
    const uint32_t p = (uint32_t)base + (threadIdx.x >> 6) * (64 * N) + (threadIdx.x & 63);
#pragma unroll
    for (int j = 0; j < N; j++) c.of[j] = refs[min(p + j * 64, (uint32_t)npages - 1)];
    return c;
}

// Free pages, by their number k among all free ones, as far as they are found.  They are collected in LDS and taken all
// at once, a thread each: taking one is a search and two loads, one after the other, and where few pages are free among
// many every scan would wait for its own (200 sequences of 39 new tokens, 800 free pages among 52000: 30 us with
// scans of 4096 that took what they found, 16 with a thread for each found, 14 so).  Up to DIRECT pages that the first scan
// finds all are taken by the waves that have them, a lane each, without that way through LDS: one token of 1, 32 and 64
// sequences that need a page each 4.3, 5.0 and 5.0 us so, 4.9, 5.6 and 5.6 by LDS.
struct Free {
    int page[4096], wave[PLAN_WAVES];  // numbers from `taken` on
};
template <int N, typename Take>
__device__ __forceinline__ void find_among(const Counts<N>& counts, int npages, int base, int total, int& taken, int& found,
                                           Free& f, Take take) {
    constexpr int ROOM = sizeof(f.page) / sizeof(int);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int at = base + wave * (64 * N);
    uint64_t free[N];
    int mine = 0;
#pragma unroll
    for (int j = 0; j < N; j++) {
        free[j] = __ballot(at + j * 64 + lane < npages && counts.of[j] == 0);
        mine += __popcll(free[j]);
    }
    __syncthreads();
    if (lane == 0) f.wave[wave] = mine;
    __syncthreads();
    int first = found, all = 0;
#pragma unroll
    for (int w = 0; w < PLAN_WAVES; w++) {
        const int r = f.wave[w];
        if (w < wave) first += r;
        all += r;
    }
    found = min(total, found + all);
    if (N == NEAR && total <= DIRECT && found == total) {
        // lane i has the wave's i-th: the 64 pages that it is in, then by halves
        uint64_t among = free[0];
        int i = lane, p = at;
#pragma unroll
        for (int j = 0; j < N - 1; j++) {
            const int n = __popcll(free[j]);
            if (p == at + j * 64 && i >= n) {
                i -= n;
                p += 64;
                among = free[j + 1];
            }
        }
#pragma unroll
        for (int half = 32; half > 0; half >>= 1) {
            const int n = __popcll(among & ((uint64_t{1} << half) - 1));
            if (i >= n) {
                i -= n;
                p += half;
                among >>= half;
            }
        }
        if (lane < mine && first + lane < total) take(first + lane, p);
        taken = total;
        return;
    }
    for (;;) {
        int k0 = first;
        if (mine > 0)
#pragma unroll
            for (int j = 0; j < N; j++) {
                const int k = k0 + __popcll(free[j] & ((uint64_t{1} << lane) - 1));
                if ((free[j] >> lane & 1) && k >= taken && k < min(found, taken + ROOM)) f.page[k - taken] = at + j * 64 + lane;
                k0 += __popcll(free[j]);
            }
        if (found - taken < ROOM) break;
        __syncthreads();
        for (int k = threadIdx.x; k < ROOM; k += PLAN_THREADS) take(taken + k, f.page[k]);
        __syncthreads();
        taken += ROOM;
    }
}

// Calls take(k, page) for the `total` lowest free pages, k = 0 .., or for all there are; returns their number.  near: the
// counts of the first pages, asked for early by the caller.
template <typename Take>
__device__ __forceinline__ int take_free(const int32_t* refs, int npages, int total, const Counts<NEAR>& near, Free& f,
                                         Take take) {
    int found = 0, taken = 0, base = NEAR * PLAN_THREADS;
    if (total <= 0) return 0;
    find_among(near, npages, 0, total, taken, found, f, take);
    if (taken == total) return total;
    if (found < total && base < npages) {
        auto counts = page_counts<FAR>(refs, npages, base);
        for (; base < npages && found < total; base += FAR * PLAN_THREADS) {
            const auto next = page_counts<FAR>(refs, npages, base + FAR * PLAN_THREADS);  // (on its way meanwhile)
            find_among(counts, npages, base, total, taken, found, f, take);
            counts = next;
        }
    }
    __syncthreads();
    for (int k = taken + (int)threadIdx.x; k < found; k += PLAN_THREADS) take(k, f.page[k - taken]);
    return found;
}

// PER: list entries a thread has at most. Lists of up to 1024 have one each, which leaves a third of the code: what
// runs once takes its time to arrive (6.4 us with eight, 4.9 with one).  ROWS: the entries' tokens are the differences
// of the device's offsets `rows`, and not of cu.
template <int PER, bool ROWS>
__global__ void __launch_bounds__(PLAN_THREADS)
    kv_reserve_kernel(const Cs1PageTable t, const int32_t* __restrict__ seqs, const Offsets cu,
                      const int32_t* __restrict__ rows, int n, int32_t* status) {
    __shared__ int work[MAX_LISTED];  // first entry that names a sequence, then the offsets off_i
    __shared__ int red[PLAN_WAVES];
    __shared__ Free free;
    const int tid = threadIdx.x;
    asm volatile("" ::"s"(t.table), "s"(t.lens), "s"(t.refs), "s"(t.nseq), "s"(t.max_pages), "s"(t.npages), "s"(t.page),
                 "s"(seqs), "s"(cu.n), "s"(n), "s"(status));
    const Counts<NEAR> near = page_counts<NEAR>(t.refs, t.npages, 0);
    const int per = PER == 1 ? 1 : (n + PLAN_THREADS - 1) / PLAN_THREADS, i0 = tid * per;
    int seq[PER], len[PER];
    int64_t add[PER];
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int i = i0 + e;
        const bool in = e < per && i < n;
        seq[e] = in ? listed_seq(seqs, i, t.nseq) : -1;
        if (ROWS) add[e] = in ? max((int64_t)rows[i + 1] - rows[i], (int64_t)0) : 0;
        len[e] = seq[e] >= 0 ? max(t.lens[seq[e]], 0) : 0;
    }
    auto grows = [&](int e) -> int64_t { return ROWS ? add[e] : cu.n ? cu.at[i0 + e + 1] - cu.at[i0 + e] : 1; };
    for (int s = tid; s < t.nseq; s += PLAN_THREADS) work[s] = n;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; e++)
        if (seq[e] >= 0) atomicMin(&work[seq[e]], i0 + e);
    __syncthreads();
    int need[PER], mine = 0;
    bool wide = false;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int i = i0 + e;
        need[e] = 0;
        if (seq[e] >= 0 && work[seq[e]] != i) seq[e] = -1;
        if (seq[e] < 0) continue;
        const int64_t to = (int64_t)len[e] + grows(e);
        if (to > (int64_t)t.max_pages * t.page)
            wide = true;
        else
            mine += need[e] = pages_of(to, t.page) - pages_of(len[e], t.page);
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
    const int found = take_free(t.refs, t.npages, total, near, free, [&](int k, int p) {
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
            if (seq[e] >= 0) t.lens[seq[e]] = (int)(len[e] + grows(e));
    }
    if (tid == 0) *status = total - found;
}

// Where the rows of a packed batch are: a row a thread.  Every block makes the list's first entries for itself (n <= 8192
// loads that a block has under way at once) and has the offsets in LDS, so that a row's chain is entry, length,
// page, and the search between costs no memory.  (7800 rows of 200 entries: 4.0 us.)  status: no row is anywhere if it is
// not 0 (null: not looked at).
__global__ void __launch_bounds__(PLAN_THREADS)
    kv_rows_kernel(const Cs1PageTable t, const int32_t* __restrict__ seqs, const int32_t* __restrict__ cu, int n,
                   int rows, const int32_t* __restrict__ status, int32_t* __restrict__ pos,
                   int32_t* __restrict__ slot) {
    extern __shared__ int lists[];
    int* const end = lists;          // [n] each entry's end
    int* const first = lists + n;    // [nseq] the first entry that names a sequence
    const int tid = threadIdx.x, r = blockIdx.x * PLAN_THREADS + tid;
    asm volatile("" ::"s"(t.table), "s"(t.lens), "s"(t.nseq), "s"(t.max_pages), "s"(t.npages), "s"(t.page), "s"(seqs),
                 "s"(cu), "s"(n), "s"(rows), "s"(status), "s"(pos), "s"(slot));
    const bool room = !status || *status == 0;
    for (int s = tid; s < t.nseq; s += PLAN_THREADS) first[s] = n;
    int seq[PER_MAX];
#pragma unroll
    for (int e = 0; e < PER_MAX; e++) {
        const int i = tid + e * PLAN_THREADS;
        seq[e] = -1;
        if (i < n) {
            seq[e] = listed_seq(seqs, i, t.nseq);
            end[i] = cu[i + 1];
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER_MAX; e++)
        if (seq[e] >= 0) atomicMin(&first[seq[e]], tid + e * PLAN_THREADS);
    __syncthreads();
    if (r >= rows) return;
    int lo = 0, hi = n;  // the entries that end at or before row r
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (end[mid] <= r)
            lo = mid + 1;
        else
            hi = mid;
    }
    int p = -1, at = -1;
    const int i = lo, s = i < n ? listed_seq(seqs, i, t.nseq) : -1;
    // (offsets that do not rise may leave a row to an entry that begins behind it)
    if (room && s >= 0 && first[s] == i && (i == 0 || end[i - 1] <= r)) {
        const int64_t here = (int64_t)t.lens[s] - (end[i] - r);
        if (here >= 0 && here < (int64_t)t.max_pages * t.page) {
            p = (int)here;
            const int pg = t.table[(size_t)s * t.max_pages + p / t.page];
            if (pg >= 0 && pg < t.npages) at = pg * t.page + p % t.page;
        }
    }
    pos[r] = p;
    slot[r] = at;
}

// Tokens taken off the ends of sequences.  One block, since whether a page is shared is asked of all entries before any
// count falls: the answer does not depend on which entry is first.
template <int PER>
__global__ void __launch_bounds__(PLAN_THREADS)
    kv_trim_kernel(const Cs1PageTable t, const int32_t* __restrict__ seqs, const int32_t* __restrict__ drop, int n,
                   int32_t* status) {
    __shared__ int work[MAX_LISTED];  // first entry that names a sequence
    __shared__ int red[PLAN_WAVES];
    const int tid = threadIdx.x, lane = tid & 63;
    asm volatile("" ::"s"(t.table), "s"(t.lens), "s"(t.refs), "s"(t.nseq), "s"(t.max_pages), "s"(t.npages), "s"(t.page),
                 "s"(seqs), "s"(drop), "s"(n), "s"(status));
    const int per = PER == 1 ? 1 : (n + PLAN_THREADS - 1) / PLAN_THREADS, i0 = tid * per;
    int seq[PER], len[PER], to[PER];
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const bool in = e < per && i0 + e < n;
        seq[e] = in ? listed_seq(seqs, i0 + e, t.nseq) : -1;
        const int off = in ? max(drop[i0 + e], 0) : 0;
        len[e] = seq[e] >= 0 ? max(t.lens[seq[e]], 0) : 0;
        to[e] = max(len[e] - off, 0);
    }
    for (int s = tid; s < t.nseq; s += PLAN_THREADS) work[s] = n;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; e++)
        if (seq[e] >= 0) atomicMin(&work[seq[e]], i0 + e);
    __syncthreads();
    int left = 0;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        if (seq[e] >= 0 && work[seq[e]] != i0 + e) seq[e] = -1;
        if (seq[e] < 0 || to[e] == len[e]) {
            seq[e] = -1;
            continue;
        }
        const int last = to[e] / t.page;  // the page that is cut
        if (to[e] % t.page == 0 || last >= t.max_pages) continue;
        const int p = t.table[(size_t)seq[e] * t.max_pages + last];
        if (p >= 0 && p < t.npages && t.refs[p] > 1) {
            seq[e] = -1;
            left++;
        }
    }
    int all;
    (void)block_scan(left, red, all);  // (its barriers stand between the counts' reads and their changes)
    __syncthreads();
    if (tid == 0) *status = all;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        int j = 0, held = 0;
        int32_t* row = nullptr;
        if (seq[e] >= 0) {
            row = t.table + (size_t)seq[e] * t.max_pages;
            j = pages_of(to[e], t.page);
            held = min(pages_of(len[e], t.page), t.max_pages);
            t.lens[seq[e]] = to[e];
        }
        auto release = [&](int p) {
            if (p >= 0 && p < t.npages) atomicSub(&t.refs[p], 1);
        };
        // a few pages a thread, and where there are many a wave
        constexpr int FEW = 4;
        if (held - j <= 2 * FEW) {
            for (; j < held; j += FEW) {
                int p[FEW];
#pragma unroll
                for (int u = 0; u < FEW; u++) p[u] = j + u < held ? row[j + u] : -1;
#pragma unroll
                for (int u = 0; u < FEW; u++) {
                    if (j + u < held) row[j + u] = -1;
                    release(p[u]);
                }
            }
        }
        for (uint64_t many = __ballot(j < held); many; many &= many - 1) {
            const int w = __ffsll((unsigned long long)many) - 1, to_page = __shfl(held, w, 64);
            const int s = __shfl(seq[e], w, 64);
            for (int k = __shfl(j, w, 64) + lane; k < to_page; k += 64) {
                int32_t* const entry = t.table + (size_t)s * t.max_pages + k;
                const int p = *entry;
                *entry = -1;
                release(p);
            }
        }
    }
}

// One wave a row.  The first of its keys and values are asked for before it is known where they go.
constexpr int ROWS_BLOCK = MOVE_THREADS / 64;

__global__ void __launch_bounds__(MOVE_THREADS)
    kv_write_kernel(const Cs1PageTable t, const int32_t* __restrict__ seqs, const Offsets cu, int first, int rows,
                    const bf16* __restrict__ k, int ldk, const bf16* __restrict__ v, int ldv, char* kp, char* vp,
                    int width) {
    const int lane = threadIdx.x & 63, r = __builtin_amdgcn_readfirstlane(blockIdx.x * ROWS_BLOCK + (threadIdx.x >> 6));
    // all arguments at once, here and in the other kernels: where they are asked for one by one, as they are used, each
    // is a wait (64 forks and a token each in 16 layers take 104 us so, 93 with this)
    asm volatile("" ::"s"(t.table), "s"(t.lens), "s"(t.nseq), "s"(t.max_pages), "s"(t.npages), "s"(t.page), "s"(seqs),
                 "s"(cu.n), "s"(cu.at[0]), "s"(first), "s"(rows), "s"(k), "s"(ldk), "s"(v), "s"(ldv), "s"(kp), "s"(vp),
                 "s"(width));
    if (r >= rows) return;
    const size_t row = cu.n ? (size_t)cu.at[0] + r : (size_t)r;
    const int packs = width / 8;
    const u32x4* const kr = reinterpret_cast<const u32x4*>(k + row * ldk);
    const u32x4* const vr = reinterpret_cast<const u32x4*>(v + row * ldv);
    u32x4 a[2], b[2];
#pragma unroll
    for (int i = 0; i < 2; i++)
        if (lane + 64 * i < packs) {
            a[i] = kr[lane + 64 * i];
            b[i] = vr[lane + 64 * i];
        }
    int i = r, back = 1;  // list entry, and how far from the end of its sequence the row is
    if (cu.n) {
        // (the last offset is behind every row)
        i = __popcll(__ballot(lane < cu.n && r >= cu.at[min(lane, cu.n - 1) + 1] - cu.at[0]));
        back = cu.at[i + 1] - cu.at[0] - r;
        i += first;
    }
    const int early = early_entry(seqs, i);
    const int s = __builtin_amdgcn_readfirstlane(listed_seq(seqs, i, t.nseq));
    if (s < 0) return;
    const int pos = __builtin_amdgcn_readfirstlane(t.lens[s]) - back;
    if (pos < 0 || pos / t.page >= t.max_pages || named_before(seqs, i, s, early)) return;
    const int pg = __builtin_amdgcn_readfirstlane(t.table[(size_t)s * t.max_pages + pos / t.page]);
    if (pg < 0 || pg >= t.npages) return;
    const size_t to = ((size_t)pg * t.page + pos % t.page) * packs;
    u32x4* const kt = reinterpret_cast<u32x4*>(kp) + to;
    u32x4* const vt = reinterpret_cast<u32x4*>(vp) + to;
#pragma unroll
    for (int i = 0; i < 2; i++)
        if (lane + 64 * i < packs) {
            kt[lane + 64 * i] = a[i];
            vt[lane + 64 * i] = b[i];
        }
    for (int e = lane + 128; e < packs; e += 64) {
        kt[e] = kr[e];
        vt[e] = vr[e];
    }
}

// What a fork does for one pair: the last page that is not full (rows of it, 0: none), copied from `from` to `to`.
struct Pair {
    int32_t on, from, to, rows;
};

template <int PER>
__global__ void __launch_bounds__(PLAN_THREADS)
    kv_fork_plan_kernel(const Cs1PageTable t, const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int n,
                        Pair* __restrict__ plan, int32_t* status) {
    __shared__ int work[MAX_LISTED];
    __shared__ int red[PLAN_WAVES];
    __shared__ Free free;
    const int tid = threadIdx.x;
    asm volatile("" ::"s"(t.table), "s"(t.lens), "s"(t.refs), "s"(t.nseq), "s"(t.max_pages), "s"(t.npages), "s"(t.page),
                 "s"(src), "s"(dst), "s"(n), "s"(plan), "s"(status));
    const Counts<NEAR> near = page_counts<NEAR>(t.refs, t.npages, 0);
    const int per = PER == 1 ? 1 : (n + PLAN_THREADS - 1) / PLAN_THREADS, i0 = tid * per;
    int from[PER], to[PER];
    Pair mine[PER];
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const bool in = e < per && i0 + e < n;
        from[e] = in ? listed_seq(src, i0 + e, t.nseq) : -1;
        to[e] = in ? listed_seq(dst, i0 + e, t.nseq) : -1;
        mine[e] = Pair{0, -1, -1, 0};
        if (from[e] < 0 || to[e] < 0 || t.lens[to[e]] > 0) continue;
        const int len = t.lens[from[e]];
        if (len <= 0 || pages_of(len, t.page) > t.max_pages) continue;
        mine[e].on = 1;
        mine[e].rows = len % t.page;
        if (mine[e].rows) mine[e].from = t.table[(size_t)from[e] * t.max_pages + len / t.page];
    }
    for (int s = tid; s < t.nseq; s += PLAN_THREADS) work[s] = n;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; e++)
        if (to[e] >= 0) atomicMin(&work[to[e]], i0 + e);
    __syncthreads();
    int need = 0;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        if (mine[e].on && (work[to[e]] != i0 + e || work[from[e]] != n)) mine[e] = Pair{0, -1, -1, 0};
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
    const int found = take_free(t.refs, t.npages, total, near, free, [&](int k, int p) {
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

// How entries are copied: a block has a chunk of one pool for `run` pairs in a row and reads it once for all that have
// the same source, so that copies of one entry cost their writing alone (8 copies of 50 MiB: 73 us, and 110 with a
// block for each).  What is written goes past the caches; so does what is read, where it is read once.  One access a
// thread: with four, and a quarter of the blocks, the 8 copies take 78 us and the compaction below 302 in place of 268.
constexpr int CHUNK = MOVE_THREADS * 16;

__device__ __forceinline__ void load_chunk(u32x4& r, const char* from, size_t chunk, size_t bytes, bool once) {
    const size_t e = chunk * CHUNK + threadIdx.x * 16;
    const u32x4* const p = reinterpret_cast<const u32x4*>(from + e);
    if (e < bytes) r = once ? __builtin_nontemporal_load(p) : *p;
}
__device__ __forceinline__ void store_chunk(const u32x4& r, char* to, size_t chunk, size_t bytes) {
    const size_t e = chunk * CHUNK + threadIdx.x * 16;
    if (e < bytes) __builtin_nontemporal_store(r, reinterpret_cast<u32x4*>(to + e));
}

constexpr int RUN_MAX = 8;

// Runs where there are blocks enough without the pairs apart (2048: eight a CU).
int run_of(size_t chunks, int pools, int n) {
    const size_t blocks = chunks * pools * n;
    const int most = blocks >= 2048 * RUN_MAX ? RUN_MAX : blocks <= 2048 ? 1 : (int)(blocks / 2048);
    return (int)cdiv(n, (int)cdiv(n, most));  // as even as it goes
}

// Blocks y = 0 of the first launch: the pairs' rows of the table, the shared pages' counts, the lengths. The others: a
// chunk of the filled rows of the unfinished pages, in pool y - 1.
__global__ void __launch_bounds__(MOVE_THREADS)
    kv_fork_kernel(const Cs1PageTable t, const int32_t* __restrict__ src, const int32_t* __restrict__ dst,
                   const Pair* __restrict__ plan, const Pools pools, size_t row_bytes, int tables, int n, int run) {
    asm volatile("" ::"s"(t.table), "s"(t.lens), "s"(t.refs), "s"(t.max_pages), "s"(t.npages), "s"(t.page), "s"(src),
                 "s"(dst), "s"(plan), "s"(row_bytes), "s"(tables), "s"(n), "s"(run));
    const int pool = (int)blockIdx.y - tables, i0 = blockIdx.z * run, i1 = min(n, i0 + run);
    if (pool < 0) {
        for (int i = i0 + blockIdx.x; i < i1; i += gridDim.x) {
            const Pair pr = plan[i];
            if (!pr.on) continue;
            const int s = src[i], d = dst[i], len = t.lens[s], full = len / t.page;
            for (int j = threadIdx.x; j < full; j += MOVE_THREADS) {
                const int p = t.table[(size_t)s * t.max_pages + j];
                t.table[(size_t)d * t.max_pages + j] = p;
                if (p >= 0 && p < t.npages) atomicAdd(&t.refs[p], 1);
            }
            if (threadIdx.x == 0) {
                if (pr.rows) t.table[(size_t)d * t.max_pages + full] = pr.to;
                t.lens[d] = len;
            }
        }
        return;
    }
    const size_t page_bytes = t.page * row_bytes;
    const int lane = threadIdx.x & 63, i = min(i0 + lane, n - 1);
    const Pair mine = plan[i];  // lane k has pair k of the run
    const int on = lane < i1 - i0 && mine.on && mine.from >= 0 && mine.from < t.npages ? mine.rows : 0;
    u32x4 r = {};
    int held = -1, held_rows = 0;
    for (int k = 0; k < i1 - i0; k++) {
        const int rows = __builtin_amdgcn_readlane(on, k), from = __builtin_amdgcn_readlane(mine.from, k);
        if (blockIdx.x * (size_t)CHUNK >= rows * row_bytes) continue;
        if (from != held || rows != held_rows)
            load_chunk(r, pools.p[pool] + from * page_bytes, blockIdx.x, rows * row_bytes, false);
        held = from;
        held_rows = rows;
        char* const to = pools.p[pool] + __builtin_amdgcn_readlane(mine.to, k) * page_bytes;
        store_chunk(r, to, blockIdx.x, rows * row_bytes);
    }
}

__global__ void __launch_bounds__(MOVE_THREADS)
    kv_free_kernel(const Cs1PageTable t, const int32_t* __restrict__ seqs) {
    asm volatile("" ::"s"(t.table), "s"(t.lens), "s"(t.refs), "s"(t.nseq), "s"(t.max_pages), "s"(t.npages), "s"(t.page),
                 "s"(seqs));
    const int i = blockIdx.x, early = early_entry(seqs, i), s = listed_seq(seqs, i, t.nseq);
    if (s < 0) return;
    const int len = t.lens[s];
    if (named_before(seqs, i, s, early)) return;
    int32_t* const row = t.table + (size_t)s * t.max_pages;
    const int held = min(pages_of(max(len, 0), t.page), t.max_pages);
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
    const uint32_t chunks = (uint32_t)((page_bytes + CHUNK - 1) / CHUNK), pages = (uint32_t)moves * chunks;
    for (uint32_t it = block; it < pages * npools; it += blocks) {
        const uint32_t pool = it / max(pages, 1u), left = it - pool * pages;
        const uint32_t k = left / chunks, chunk = left - k * chunks;
        u32x4 r = {};
        load_chunk(r, pools.p[pool] + from[k] * page_bytes, chunk, page_bytes, true);
        store_chunk(r, pools.p[pool] + to[k] * page_bytes, chunk, page_bytes);
    }
}

// Block: a chunk (x) of a run of pairs (z) in pool y.
__global__ void __launch_bounds__(MOVE_THREADS)
    kv_copy_kernel(const Pools pools, size_t bytes, int entries, const int32_t* __restrict__ src,
                   const int32_t* __restrict__ dst, int n, int run) {
    char* const pool = pools.p[blockIdx.y];
    asm volatile("" ::"s"(pool), "s"(bytes), "s"(entries), "s"(src), "s"(dst), "s"(n), "s"(run));
    const int i0 = blockIdx.z * run, count = min(n - i0, run), lane = threadIdx.x & 63;
    // each wave for itself: lane k has pair k of the run, and all of them are held against 64 destinations at a time
    const int s = lane < count ? src[i0 + lane] : -1, d = lane < count ? dst[i0 + lane] : -1;
    uint32_t out = 0;
    for (int j0 = 0; j0 < n; j0 += 64) {
        const int j = j0 + lane, other = j < n ? dst[j] : -1;
        for (int k = 0; k < count; k++)
            if (__any(j < n && (other == __builtin_amdgcn_readlane(s, k) ||
                                (j < i0 + k && other == __builtin_amdgcn_readlane(d, k)))))
                out |= 1u << k;
    }
    u32x4 r = {};
    int held = -1;
    for (int k = 0; k < count; k++) {
        const int from = __builtin_amdgcn_readlane(s, k), to = __builtin_amdgcn_readlane(d, k);
        if (out >> k & 1 || from < 0 || from >= entries || to < 0 || to >= entries) continue;
        const bool again = k + 1 < count && __builtin_amdgcn_readlane(s, k + 1) == from;
        if (from != held) load_chunk(r, pool + from * bytes, blockIdx.x, bytes, !again);
        held = from;
        store_chunk(r, pool + to * bytes, blockIdx.x, bytes);
    }
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

bool row_ok(size_t row_bytes) { return row_bytes > 0 && row_bytes % 16 == 0 && row_bytes <= ((size_t)1 << 32); }

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
    const auto kernel = n <= PLAN_THREADS ? kv_reserve_kernel<1, false> : kv_reserve_kernel<PER_MAX, false>;
    kernel<<<1, PLAN_THREADS, 0, static_cast<hipStream_t>(stream)>>>(*pages, seqs, cu, nullptr, n, status);
    return hipGetLastError();
}

extern "C" int cs1_kv_extend(const Cs1PageTable* pages, const int32_t* seqs, const int32_t* cu_seqlens, int n,
                             int32_t* status, void* stream) {
    if (!table_ok(pages) || n < 0 || n > MAX_LISTED || !status || (n > 0 && !cu_seqlens)) return hipErrorInvalidValue;
    // new pages are counted in 32 bits; offsets on the device that fall and rise again can ask for any number of them
    if ((int64_t)std::min(n, pages->nseq) * pages->max_pages > INT32_MAX) return hipErrorInvalidValue;
    Offsets none;
    none.n = 0;
    const auto kernel = n <= PLAN_THREADS ? kv_reserve_kernel<1, true> : kv_reserve_kernel<PER_MAX, true>;
    kernel<<<1, PLAN_THREADS, 0, static_cast<hipStream_t>(stream)>>>(*pages, seqs, none, cu_seqlens, n, status);
    return hipGetLastError();
}

static int kv_rows(const Cs1PageTable* pages, const int32_t* seqs, const int32_t* cu_seqlens, int n, int rows,
                   const int32_t* status, int32_t* pos, int32_t* slot, void* stream) {
    if (!table_ok(pages) || n < 0 || n > MAX_LISTED || rows < 0 || (int64_t)pages->npages * pages->page > INT32_MAX)
        return hipErrorInvalidValue;
    if (rows == 0) return hipSuccess;
    if (!all_set({pos, slot}) || (n > 0 && !cu_seqlens)) return hipErrorInvalidValue;
    kv_rows_kernel<<<cdiv(rows, PLAN_THREADS), PLAN_THREADS, 4 * ((size_t)n + pages->nseq),
                     static_cast<hipStream_t>(stream)>>>(*pages, seqs, cu_seqlens, n, rows, status, pos, slot);
    return hipGetLastError();
}

extern "C" int cs1_kv_rows(const Cs1PageTable* pages, const int32_t* seqs, const int32_t* cu_seqlens, int n, int rows,
                           int32_t* pos, int32_t* slot, void* stream) {
    return kv_rows(pages, seqs, cu_seqlens, n, rows, nullptr, pos, slot, stream);
}

extern "C" int cs1_kv_rows_if_room(const Cs1PageTable* pages, const int32_t* seqs, const int32_t* cu_seqlens, int n,
                                   int rows, const int32_t* status, int32_t* pos, int32_t* slot, void* stream) {
    if (!status) return hipErrorInvalidValue;
    return kv_rows(pages, seqs, cu_seqlens, n, rows, status, pos, slot, stream);
}

extern "C" int cs1_kv_trim(const Cs1PageTable* pages, const int32_t* seqs, const int32_t* drop, int n, int32_t* status,
                           void* stream) {
    if (!table_ok(pages) || n < 0 || n > MAX_LISTED || !status || (n > 0 && !drop)) return hipErrorInvalidValue;
    const auto kernel = n <= PLAN_THREADS ? kv_trim_kernel<1> : kv_trim_kernel<PER_MAX>;
    kernel<<<1, PLAN_THREADS, 0, static_cast<hipStream_t>(stream)>>>(*pages, seqs, drop, n, status);
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
        kv_write_kernel<<<cdiv(rows, ROWS_BLOCK), MOVE_THREADS, 0, st>>>(
            *pages, seqs, cu, first, rows, static_cast<const bf16*>(k), ldk, static_cast<const bf16*>(v), ldv,
            static_cast<char*>(kp), static_cast<char*>(vp), (int)width);
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
    if (npools > 0 && !row_ok(row_bytes)) return hipErrorInvalidValue;
    const size_t chunks = npools > 0 ? ((pages->page - 1) * row_bytes + CHUNK - 1) / CHUNK : 1;
    if (chunks > CHUNKS_MAX) return hipErrorInvalidValue;
    if (n > 0 && (!all_set({src, dst, workspace}) || !on16(workspace))) return hipErrorInvalidValue;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    Pair* const plan = static_cast<Pair*>(workspace);
    const auto kernel = n <= PLAN_THREADS ? kv_fork_plan_kernel<1> : kv_fork_plan_kernel<PER_MAX>;
    kernel<<<1, PLAN_THREADS, 0, st>>>(*pages, src, dst, n, plan, status);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || n == 0) return e;
    int first = 0;
    do {
        Pools some = {};
        const int k = some_pools(pools, npools, first, some), tables = first == 0;
        const int run = run_of(chunks, k, n);
        kv_fork_kernel<<<dim3((unsigned)chunks, k + tables, cdiv(n, run)), MOVE_THREADS, 0, st>>>(
            *pages, src, dst, plan, some, row_bytes, tables, n, run);
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
    if (npools > 0 && !row_ok(row_bytes)) return hipErrorInvalidValue;
    const size_t page_bytes = pages->page * row_bytes;
    if (npools > 0 && (page_bytes / CHUNK > CHUNKS_MAX ||
                       (uint64_t)(pages->npages / 2 + 1) * POOLS_MAX * (page_bytes / CHUNK + 1) >= uint64_t{1} << 31))
        return hipErrorInvalidValue;
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
        // a block for each chunk that may move, as far as that is 512 a CU (blocks that go on to a second chunk wait
        // for the first one's stores to be taken: 268 us so, 284 with 128 and 326 with 8, in a pool of 1400 pages of
        // 128 KiB with 700 held in 16 pools; 299 with 2048, when half of them find nothing to do)
        const size_t most = (size_t)(pages->npages / 2) * k * (page_bytes / CHUNK + 1), cap = (size_t)512 * cus;
        const unsigned movers = (unsigned)(most < cap ? most + 1 : cap);
        kv_compact_kernel<<<tables + movers, MOVE_THREADS, 0, st>>>(*pages, ws, some, k, npools > 0 ? page_bytes : 0,
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
    const size_t chunks = (entry_bytes + CHUNK - 1) / CHUNK;
    if (chunks > CHUNKS_MAX) return hipErrorInvalidValue;
    if (npools == 0 || n == 0 || entries == 0 || entry_bytes == 0) return hipSuccess;
    if (!all_set({src, dst})) return hipErrorInvalidValue;
    for (int first = 0; first < npools; first += POOLS_MAX) {
        Pools some = {};
        const int k = some_pools(pools, npools, first, some);
        const int run = run_of(chunks, k, n);
        kv_copy_kernel<<<dim3((unsigned)chunks, k, cdiv(n, run)), MOVE_THREADS, 0, static_cast<hipStream_t>(stream)>>>(
            some, entry_bytes, entries, src, dst, n, run);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
