// The page table of the decode operations: its checks on the host and the lists of sequences on the device.
#pragma once

#include "common.h"

namespace q35 {

constexpr int MAX_LISTED = 8192;  // sequences of a table, rows of a list (kv_pages.hip keeps one int each in LDS)
// A scan's step past the last page is an int, and so is the last of compaction's entries (half as many again).
constexpr int MAX_PAGES = 1 << 30;

inline bool table_ok(const Cs1PageTable* t) {
    return t && all_set({t->table, t->lens, t->refs}) && t->nseq > 0 && t->nseq <= MAX_LISTED && t->max_pages > 0 &&
           t->npages > 0 && t->npages <= MAX_PAGES && t->page >= 16 && t->page % 16 == 0 &&
           (int64_t)t->max_pages * t->page < (int64_t{1} << 31);
}

inline bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The sequence of list entry i, or -1 for a padding row.
__device__ __forceinline__ int listed_seq(const int32_t* __restrict__ seqs, int i, int nseq) {
    const int s = seqs ? seqs[i] : i;
    return s >= 0 && s < nseq ? s : -1;
}

// Whether an entry before i names the same sequence, asked by a whole wave for itself; early: the lane's of the first 64
// entries, asked for when the kernel begins.
__device__ __forceinline__ int early_entry(const int32_t* __restrict__ seqs, int i) {
    const int j = threadIdx.x & 63;
    return seqs && j < i ? seqs[j] : -1;
}
__device__ __forceinline__ bool named_before(const int32_t* __restrict__ seqs, int i, int s, int early) {
    bool hit = early == s;
    if (seqs)
        for (int j = 64 + (threadIdx.x & 63); j < i; j += 64) hit |= seqs[j] == s;
    return __any(hit);
}

}  // namespace q35
