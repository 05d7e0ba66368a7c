// What the kernels on the 32x32x16 bfloat16 MFMA share: the product, the places of 16-byte chunks in LDS rows, transposing
// reads and exchanges between the lane halves.
#pragma once

#include "common.h"

namespace q35 {
namespace tile32 {

// Chunk placement, conflict-free whether the LDS serves 128 or 256 bytes per cycle: 16-byte
// chunk c of K row r sits at slot c ^ (r & 15) (8 or 16 consecutive rows read at one chunk hit
// distinct slots); of V row r at slot c ^ f(r & 3), f = {0, 6, 12, 10}, which separates the
// four rows of a transposing read both within 8 slots (two adjacent chunks per row, one lane
// group) and within 16 (four chunks per row, two lane groups).
__device__ __forceinline__ int k_slot(int r, int c) { return c ^ (r & 15); }
__device__ __forceinline__ int v_slot(int r, int c) { return c ^ ((0xAC60 >> (4 * (r & 3))) & 15); }

__device__ __forceinline__ f32x16 mfma32(const u32x4& a, const u32x4& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

// Maximum over the two lane halves (lanes l and l ^ 32): one v_permlane32_swap, no LDS trip.
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2 read_tr(const unsigned char* p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (__attribute__((address_space(3))) s16x4*)(p)));
}

}  // namespace tile32
}  // namespace q35
