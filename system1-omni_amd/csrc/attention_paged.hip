// Attention of one new token per row over a paged key-value cache (cs1_attention_paged).  For a row of
// sequence s with n = lens[s] keys and q head h on kv head h / (Hq / Hk):
//
//   S_j = scale q . k_j,  m = max S_j,  l = sum exp(S_j - m),  out = sigmoid(gate) (sum exp(S_j - m) v_j) / l,
//   lse = m + log l.
//
// The keys and values are read once and nothing else is of size, so the rate of that stream is the bound.
//
// Work: the q heads of a kv head are the rows of one matrix tile, up to 16 of them (more take several tiles, which
// read the keys again).  The keys of all rows, kv heads and tiles, in chunks of 64 or 128, are one line of work that
// is cut into equal stretches, one for each CU: whatever the lengths, every block streams the same amount and all end
// about together (9 sequences of 9000 to 32768 keys, 24/4 heads of 256: 176 us, 5.5 TB/s; with a block for each share
// of a sequence, two and four to a CU, 185 and 203 us).  A stretch may begin and end inside a sequence; what it has
// of one (a segment) is joined with the other blocks' parts by the last of them to end.  Within a block four waves
// take every fourth unit of 32 keys, each with a running maximum and sum of its own, and join through LDS.
//
// A unit in registers, without LDS: S^T = K Q^T takes K rows as they lie (lane l: key l % 16, 8 dims a load) and
// leaves lane l with q head l % 16 and keys 4 (l / 16) .. + 3 of each 16; that is the layout in which O^T = V^T P^T
// wants P^T, with the unit's keys in the order (i < 4: 4 g + i, else 16 + 4 g + i - 4) for lane group g.  V rows are
// loaded 16 lanes x 16 bytes at a time (256 bytes in a row), lane l holding dims 8 (l % 16) .. + 7 of its group's
// eight keys, and two-byte permutes make columns of eight keys of them: the tile's row m is dim 8 m + j.  Each q head
// stays in its lanes from the scores to the output, so maximum and sum need no exchange but between lane groups, and
// that only when the maximum rises by more than RISE or at the end.  The next unit's K is on its way while this one's
// probabilities are formed, its V while the next scores are.
//
// P goes to the product in three bfloat16 parts, which hold its 24 bits (two cut off, the rest as it is): the matrix
// cores wait for memory here (9 sequences as above: 175.3 us with two parts, 175.6 with three), and out is rounded once
// and in its own type only.  With two parts (p to 2^-16) 0.4% of the outputs fell to the other side of a rounding, with
// three 0.05% do.  Where p is not zero no part is (LEAST), so that an infinite v gives the infinity that it should and
// not inf + 0 inf.
#include <algorithm>
#include <new>
#include <type_traits>

#include "common.h"
#include "paged.h"

namespace q35 {
namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;
static_assert(WAVES == 4, "the waves' maxima and the rows' sums are joined by name");
constexpr int UNIT = 32, ROWS = 16;
constexpr int GROUP = 64, BATCH = 16;  // parts that one block joins, and how many of them are on their way at once
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LEAST = 0x1p-126f;  // bfloat16's smallest normal value
constexpr float RISE = 6.f;  // in powers of two: P stays under 2^6, far from where float32 sums lose anything

struct Args {
    const bf16 *q, *kp, *vp, *gate;
    bf16* out;
    float *lse, *part, *ml;
    int *count, *count2;
    const int32_t *table, *lens, *seqs;
    int nseq, max_pages, npages, page, B, Hq, Hk, G, tiles, blocks, halve, unit, pad_alone;
    uint32_t page_inverse, blocks_inverse;  // 2^32 over page / 16, rounded down, and over blocks, rounded up
    float scale_log2;
    // several tokens a row: the offsets of their rows, at most how many, the buffers' rows, 2^16 over G rounded up
    const int32_t* cu;
    int max_new, all_rows;
    uint32_t G_inverse;

    __device__ __forceinline__ int pad() const { return pad_alone & 255; }
    __device__ __forceinline__ int alone() const { return pad_alone >> 8; }
};

// What a part of p leaves of it, at least LEAST unless p is zero: the median, since p is zero or no less than LEAST.  (A
// zero must stay one: LEAST times a value of bfloat16's largest size is 4.)
__device__ __forceinline__ float rest(float p, float part) { return __builtin_amdgcn_fmed3f(p - part, p, LEAST); }

// Row r's sequence (of its keys: none for padding).  SEVERAL: row r is a list entry, whose tokens are `tokens` rows from
// row0 on; n is the number of keys that the last of them sees.
struct Row {
    int s, n;
};
struct Rows16 : Row {
    int row0, tokens;
};
__device__ __forceinline__ int held_by(const Args& a, int s) {
    return (int)min((int64_t)max(a.lens[s], 0), (int64_t)a.max_pages * a.page);
}
template <bool SEVERAL>
__device__ __forceinline__ auto row_of(const Args& a, int r) {
    if constexpr (SEVERAL) {
        Rows16 x{{0, 0}, 0, 0};
        if (r >= a.B) return x;
        const int lo = a.cu[r], hi = a.cu[r + 1], s = listed_seq(a.seqs, r, a.nseq);  // (asked for together)
        if (lo < 0 || hi <= lo || lo >= a.all_rows) return x;
        x.row0 = lo;
        x.tokens = min(min(hi, a.all_rows) - lo, a.max_new);
        if (x.tokens > ROWS || x.tokens * a.G > ROWS) return Rows16{{0, 0}, 0, 0};  // (another kernel's)
        if (s < 0) return x;
        x.s = s;
        x.n = (int)max((int64_t)held_by(a, s) - (hi - lo) + x.tokens, (int64_t)0);
        return x;
    } else {
        const int s = r < a.B ? listed_seq(a.seqs, r, a.nseq) : -1;
        return s < 0 ? Row{0, 0} : Row{s, held_by(a, s)};
    }
}

__device__ __forceinline__ int units_of(int n) { return n / UNIT + (n % UNIT != 0); }

// Chunks of a row's work for one kv head and tile, of a.unit units each.  A row without keys has one: its zeros are
// written. The first a.pad() chunks stand for the time that a block needs to begin with it, and have no keys.
__device__ __forceinline__ int chunks_of(const Args& a, int n) {
    return a.pad() + (n <= a.alone() * UNIT ? 1 : (units_of(n) + a.unit - 1) / (uint32_t)a.unit);
}

// Sum over this lane and those below: within rows of 16 lanes, then each row's last lane to the next row (into rows
// 1 and 3), then lane 31 to the upper half.
__device__ __forceinline__ int wave_scan(int x) {
#define Q35_ADD(ctrl, rows) x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, false)
    Q35_ADD(0x111, 0xf);
    Q35_ADD(0x112, 0xf);
    Q35_ADD(0x114, 0xf);
    Q35_ADD(0x118, 0xf);
    Q35_ADD(0x142, 0xa);
    Q35_ADD(0x143, 0xc);
#undef Q35_ADD
    return x;
}

// Lane i's value, one for the wave.
__device__ __forceinline__ int scalar(int x, int i) { return __builtin_amdgcn_readlane(x, i); }

// The lane's number, found again where it is asked for: what follows from it would otherwise be kept in registers
// over the loop over the keys, which has none to spare.
__device__ __forceinline__ int lane_here() {
    int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));
    asm volatile("" : "+v"(lane));
    return lane;
}

// One value from the four of a lane's column (lanes 16 apart), in each of them: rows of 16 lanes are swapped, then
// halves.
template <typename F>
__device__ __forceinline__ float over_groups(float x, F f) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Rows in the work's order, a wave's 64 at a time: only the device knows the lengths.
template <typename R>
struct Rows {
    R row;             // one row,
    int chunks, upto;  // its chunks, and those of the wave's rows up to it
};

struct Segment {
    int row, s, n, head, tile;  // the n keys of row `row`'s sequence s for kv head `head` and a tile of q heads
    int from, to, next;         // units of it (none: the stretch ends before its keys), and the chunk behind them
    int first, parts, part;     // the first block that has some of it, how many have, and which of them this is
    int slot0;                  // where the first one's results go; the others' go to 2 x their block
    int row0, tokens;           // several tokens: as in Rows16

    __device__ __forceinline__ int slot(int k) const { return k == 0 ? slot0 : 2 * (first + k); }
};

// Looks for the segment that begins at chunk `pos` of this block's stretch, which ends at `end`, among 64 rows from
// r0 on, which begin at chunk `before`; stretches are `each` chunks long. (What runs once a launch is kept short: its
// instructions come from memory, and divisions are long.)
template <typename R>
__device__ __forceinline__ bool segment_at(const Args& a, const Rows<R>& rows, int r0, int before, int pos, int end,
                                           int each, Segment& s) {
    const int heads = a.Hk * a.tiles;
    const uint64_t hit = __ballot(pos < before + rows.upto * heads);
    if (!hit) return false;
    const int w = __ffsll((unsigned long long)hit) - 1, chunks = scalar(rows.chunks, w);
    int whole = before + (scalar(rows.upto, w) - chunks) * heads;
    s = {};
    s.row = r0 + w;
    s.s = scalar(rows.row.s, w);
    s.n = scalar(rows.row.n, w);
    if constexpr (!std::is_same_v<R, Row>) {
        s.row0 = scalar(rows.row.row0, w);
        s.tokens = scalar(rows.row.tokens, w);
    }
    for (; whole + chunks <= pos; whole += chunks)
        if (++s.tile == a.tiles) {
            s.tile = 0;
            s.head++;
        }
    s.next = min(whole + chunks, end);
    const int keys = whole + a.pad(), begin = max(pos, keys);
    if (begin >= end) return true;
    s.from = (begin - keys) * a.unit;
    s.to = whole + chunks <= end ? units_of(s.n) : (end - keys) * a.unit;
    s.first = keys >= (int)blockIdx.x * each ? blockIdx.x : keys / (uint32_t)each;
    s.part = blockIdx.x - s.first;
    s.parts = (whole + chunks <= end ? blockIdx.x : (whole + chunks - 1) / (uint32_t)each) - s.first + 1;
    s.slot0 = 2 * s.first + (keys > s.first * each);
    return true;
}

// Four dims of an output from sums o over l (zero: no key); g: their gates, if there are any.
__device__ __forceinline__ u32x2 load_gate(const Args& a, size_t at) {
    return a.gate ? *reinterpret_cast<const u32x2*>(a.gate + at) : u32x2{0, 0};
}
template <bool SEVERAL>
__device__ __forceinline__ void store_out(const Args& a, size_t at, const f32x4& o, float l, const u32x2& g) {
    float y[4];
    if constexpr (SEVERAL) {  // a thread has some: the hardware's reciprocal, within a float32 step, and no branches (0.7 us)
        const float inv = __builtin_amdgcn_rcpf(l);
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = o[e] * inv;
        if (a.gate)
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] *= gate_sigmoid(e & 1 ? hi_f32(g[e / 2]) : lo_f32(g[e / 2]));
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = l != 0.f ? y[e] : 0.f;
        *reinterpret_cast<u32x2*>(a.out + at) = u32x2{pack2(y[0], y[1]), pack2(y[2], y[3])};
        return;
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        y[e] = l != 0.f ? o[e] * inv : 0.f;
        if (a.gate && l != 0.f) y[e] *= sigmoid(e & 1 ? hi_f32(g[e / 2]) : lo_f32(g[e / 2]));
    }
    *reinterpret_cast<u32x2*>(a.out + at) = u32x2{pack2(y[0], y[1]), pack2(y[2], y[3])};
}

__device__ __forceinline__ float log_sum(float top, float sum) {
    return sum == 0.f ? -INFINITY : (top + log2f(sum)) * LN2;
}

// Results that another block reads in the same launch.  Each XCD has an L2 of its own, so they are written through
// it and read past it (device scope, the SC1 bit).  A fence instead would write back all that the L2 holds, for every
// wave that executes it: 240 us in place of 25 for 32768 keys in 1024 parts.
struct Shared {
    static constexpr int SC1 = 0x10;
    __amdgpu_buffer_rsrc_t part, ml;

    __device__ __forceinline__ explicit Shared(const Args& a)
        : part(__builtin_amdgcn_make_buffer_rsrc(a.part, (short)0, 0x7fffffff, 0x00020000)),
          ml(__builtin_amdgcn_make_buffer_rsrc(a.ml, (short)0, 0x7fffffff, 0x00020000)) {}
    // byte offsets: under 2^31 for the handle's 2 x blocks slots of at most 16 x 256 floats
    __device__ __forceinline__ f32x4 get(int at) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(part, at, 0, SC1));
    }
    __device__ __forceinline__ void put(int at, const f32x4& v) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), part, at, 0, SC1);
    }
    __device__ __forceinline__ f32x2 get_ml(int at) const {
        return __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(ml, at, 0, SC1));
    }
    __device__ __forceinline__ void put_ml(int at, const f32x2& v) const {
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, v), ml, at, 0, SC1);
    }
};

// SEVERAL: a row of the work is a list entry with up to 16 columns, its tokens' q heads of a kv head; otherwise it is a
// token with the q heads alone.  (Heads of 128 then have more code that wants registers, and the compiler has to be told that
// two blocks share a CU: 200 entries behind up to 400 take 34 us so, 54 with one.)
template <int DH, bool SEVERAL>
__global__ void __launch_bounds__(THREADS, SEVERAL && DH == 128 ? 2 : 1) attention_paged_kernel(const Args a) {
    using R = std::conditional_t<SEVERAL, Rows16, Row>;
    constexpr int C = DH / 32, H = DH / 128, PITCH = DH + 8;
    // Q as operands, [C][64 lanes] x 16 bytes; then the waves' results, [WAVES][rows][PITCH]; then what joins parts
    extern __shared__ __attribute__((aligned(16))) float lds[];
    __shared__ float wm[WAVES][ROWS], wl[WAVES][ROWS];
    const int wave = scalar(threadIdx.x >> 6, 0);
    // THREADS rows at a time, a thread each, in LDS; of more than that, those last looked at
    __shared__ Rows<R> table[THREADS];
    __shared__ int sums[WAVES];
    auto look_at = [&](int r0) {
        const int i = wave * 64 + lane_here(), r = r0 + i;
        Rows<R> x;
        x.row = row_of<SEVERAL>(a, r);
        x.chunks = r < a.B ? chunks_of(a, x.row.n) : 0;
        if constexpr (SEVERAL)
            if (x.row.tokens == 0) x.chunks = 0;
        x.upto = wave_scan(x.chunks);
        __syncthreads();
        table[i] = x;
        if ((i & 63) == 63) sums[wave] = x.upto;
        __syncthreads();
        return sums[0] + sums[1] + sums[2] + sums[3];
    };
    const int heads = a.Hk * a.tiles;
    int total = look_at(0);
    for (int r0 = THREADS; r0 < a.B; r0 += THREADS) total += look_at(r0);
    total = __builtin_amdgcn_readfirstlane(total * heads);
    if (SEVERAL && total == 0) return;
    // With heads of 128 two blocks fit on a CU (and are launched for many sequences): where these are short, on
    // average under 10 chunks (384 keys; 11 where beginning counts for one more), a block's time is that of beginning and ending each, and two at once hide it.
    // 200 sequences of 260 to 384 keys take 35.3 us so and 39.0 with one, of 200 to 800 53.4 and 48.5 (16/4 heads).
    const uint32_t inverse = a.halve && total >= (SEVERAL ? 11 : 10) * a.B * heads ? 2 * a.blocks_inverse : a.blocks_inverse;
    const int each = __umulhi(total - 1, inverse) + 1;  // (one more than need be where the inverse's rounding shows)
    const int begin = (int)blockIdx.x * each, end = min(total, begin + each);
    // (the rows go on from one segment to the next: r0 the 64 that are searched, which begin at chunk `before`)
    int r0 = 0, before = 0, seen = (a.B - 1) / THREADS * THREADS;
    for (int pos = begin; pos < end;) {
        Segment sh = {};
        for (; r0 < a.B; r0 += 64) {
            const int w = r0 / 64 % WAVES;
            if (r0 - w * 64 != seen) (void)look_at(seen = r0 - w * 64);
            if (segment_at(a, table[w * 64 + lane_here()], r0, before, pos, end, each, sh)) break;
            before += __builtin_amdgcn_readfirstlane(sums[w]) * heads;
        }
        const int lane = lane_here(), col = lane & 15, grp = lane >> 4;
        pos = sh.next;
        if (sh.parts == 0) break;
        const int rows = SEVERAL ? sh.tokens * a.G : min(ROWS, a.G - sh.tile * ROWS);
        const int head0 = sh.head * a.G + sh.tile * ROWS;
        // of q, gate and out, the row and head that a row of the tile has
        auto at_row = [&](int row) {
            if constexpr (SEVERAL) {
                const int token = (int)(row * a.G_inverse >> 16);
                return ((size_t)(sh.row0 + token) * a.Hq + head0 + row - token * a.G) * DH;
            } else {
                return ((size_t)sh.row * a.Hq + head0) * DH + row * DH;
            }
        };
        const int u_end = sh.to;
        int u = sh.from + wave;

        // Q and the table are asked for together, and are there before any key is asked for: a wait for Q alone would
        // be one for all of them (2000 sequences of up to 100 keys: 218 us so, 250 with one after the other)
        u32x4* const qf = reinterpret_cast<u32x4*>(lds);
        u32x4 qs[C / WAVES];
#pragma unroll
        for (int i = 0; i < C / WAVES; i++) {
            qs[i] = u32x4{0, 0, 0, 0};
            if (col < rows)
                qs[i] = *reinterpret_cast<const u32x4*>(a.q + at_row(col) + (wave + i * WAVES) * 32 + grp * 8);
        }
        f32x4 acc[H][8];
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
            for (int j = 0; j < 8; j++) acc[h][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;

        // where the next units' halves lie: lane i has half i % 2 of unit i / 2 from here, the pool's row / 16 and 5
        // bits of valid keys
        const size_t token = (size_t)a.Hk * DH;
        uint32_t where = 0;
        int next = 64;
        auto look_up = [&](int from) {
            const int i = lane_here();
            const uint32_t half = 2 * (from + (i >> 1) * WAVES) + (i & 1), page = (uint32_t)a.page / 16;
            uint32_t slot = __umulhi(half, a.page_inverse);
            slot += (slot + 1) * page <= half;
            where = 0;
            if (16 * half < (uint32_t)sh.n) {
                const int pg = a.table[(size_t)sh.s * a.max_pages + slot];
                if (pg >= 0 && pg < a.npages)
                    where = (pg * page + half - slot * page) << 5 | min(16, (int)(sh.n - 16 * half));
            }
        };
        // The next unit is on its way while one is worked on.  A half's rows are read through a buffer descriptor
        // that ends with the last valid one: rows behind it, and whole units behind the wave's last, come as zeros
        // and cost no access.
        u32x4 kf[2][C], vf[H][8];
        size_t at[2];
        int have[2];
        const uint32_t row_b = 2 * (uint32_t)token;  // bytes of a token's row
        const uint32_t k_lane = col * row_b + grp * 16, v_lane = grp * 4 * row_b + col * 16;
        auto half_rows = [&](const bf16* pool, size_t from, int rows) {
            const uint64_t p = reinterpret_cast<uint64_t>(pool + from);
            const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)p);
            const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(p >> 32));
            const int bytes = __builtin_amdgcn_readfirstlane(rows > 0 ? (rows - 1) * row_b + 2 * DH : 0);
            return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>((uint64_t)hi << 32 | lo), (short)0, bytes,
                                                     0x00020000);
        };
        auto load_k = [&](int from) {
            if (next == 64) {
                look_up(from);
                next = 0;
            }
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint32_t w = from < u_end ? __builtin_amdgcn_readlane(where, next + t) : 0;
                at[t] = (size_t)(w >> 5) * (16 * token) + sh.head * DH;
                have[t] = w & 31;
                const auto r = half_rows(a.kp, at[t], have[t]);
#pragma unroll
                for (int c = 0; c < C; c++)
                    kf[t][c] =
                        __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, k_lane + c * 64, 0, 0));
            }
            next += 2;
        };
        auto load_v = [&]() {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const auto r = half_rows(a.vp, at[t], have[t]);
#pragma unroll
                for (int h = 0; h < H; h++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        vf[h][t * 4 + i] = __builtin_bit_cast(
                            u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, v_lane + h * 256, i * row_b, 0));
            }
        };
        if (u < u_end) {
            look_up(u);
            next = 0;
        }
        __syncthreads();  // the segment before is done with LDS
#pragma unroll
        for (int i = 0; i < C / WAVES; i++) qf[(wave + i * WAVES) * 64 + lane] = qs[i];
        if (u < u_end) {
            load_k(u);
            load_v();
        }
        __syncthreads();
        for (; u < u_end; u += WAVES) {
            const int valid[2] = {have[0], have[1]};
            const size_t v_at[2] = {at[0], at[1]};
            f32x4 st[2][2] = {};  // two sums a half: a product does not wait for the one before
#pragma unroll
            for (int c = 0; c < C; c++) {
                const u32x4 q = qf[c * 64 + lane];
#pragma unroll
                for (int t = 0; t < 2; t++) st[t][c & 1] = mfma16(kf[t][c], q, st[t][c & 1]);
            }
            __builtin_amdgcn_sched_barrier(0);
            load_k(u + WAVES);
            __builtin_amdgcn_sched_barrier(0);
            float sc[8], top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; i++) sc[i] = (st[i >> 2][0][i & 3] + st[i >> 2][1][i & 3]) * a.scale_log2;
            if (valid[0] + valid[1] < UNIT)
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (grp * 4 + (i & 3) >= valid[i >> 2]) sc[i] = -INFINITY;
            // the last keys are tokens that those before them do not see
            bool partly = false;
            if constexpr (SEVERAL) {
                partly = (u + 1) * UNIT > sh.n - (sh.tokens - 1);
                if (partly) {
                    const int sees = sh.n - (sh.tokens - 1) + (int)(col * a.G_inverse >> 16) - u * UNIT - grp * 4;
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if ((i >> 2) * 16 + (i & 3) >= sees) sc[i] = -INFINITY;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, sc[i]);
            if (__any(top > m + RISE)) {
                top = fmaxf(m, over_groups(top, [](float x, float y) { return fmaxf(x, y); }));
                const float keep = top == m ? 1.f : __builtin_amdgcn_exp2f(m - top);
                m = top;
                l *= keep;
#pragma unroll
                for (int h = 0; h < H; h++)
#pragma unroll
                    for (int j = 0; j < 8; j++) acc[h][j] *= keep;
            }
            const float base = m == -INFINITY ? 0.f : m;  // no key yet: exp2(-inf) = 0
            u32x4 ph, pm, pl;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p0 = __builtin_amdgcn_exp2f(sc[2 * i] - base);
                const float p1 = __builtin_amdgcn_exp2f(sc[2 * i + 1] - base);
                l += p0 + p1;
                ph[i] = __builtin_amdgcn_perm(__float_as_uint(p1), __float_as_uint(p0), 0x07060302);
                const float r0 = rest(p0, lo_f32(ph[i])), r1 = rest(p1, hi_f32(ph[i]));
                pm[i] = __builtin_amdgcn_perm(__float_as_uint(r1), __float_as_uint(r0), 0x07060302);
                pl[i] = pack2(rest(r0, lo_f32(pm[i])), rest(r1, hi_f32(pm[i])));
            }
            // a value there that is an infinity or NaN leaves the product, and is added to the columns that see it
            bool odd = false;
            if constexpr (SEVERAL) {
                if (partly) {
#pragma unroll
                    for (int h = 0; h < H; h++)
#pragma unroll
                        for (int i = 0; i < 8; i++)
#pragma unroll
                            for (int e = 0; e < 4; e++) odd |= odd16(vf[h][i][e]);
                    odd = __any(odd);
                    if (odd) {
#pragma unroll
                        for (int h = 0; h < H; h++)
#pragma unroll
                            for (int i = 0; i < 8; i++)
#pragma unroll
                                for (int e = 0; e < 4; e++) vf[h][i][e] = common16(vf[h][i][e]);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < H; h++) {
                u32x4 vt[8];
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        vt[j][i] = __builtin_amdgcn_perm(vf[h][2 * i + 1][j >> 1], vf[h][2 * i][j >> 1],
                                                         j & 1 ? 0x07060302 : 0x05040100);
#pragma unroll
                for (int j = 0; j < 8; j++) acc[h][j] = mfma16(vt[j], ph, acc[h][j]);
#pragma unroll
                for (int j = 0; j < 8; j++) acc[h][j] = mfma16(vt[j], pm, acc[h][j]);
#pragma unroll
                for (int j = 0; j < 8; j++) acc[h][j] = mfma16(vt[j], pl, acc[h][j]);
            }
            if constexpr (SEVERAL) {
                if (odd) {
                    // (a lane has dims 8 (4 grp + r) + j of its column)
                    const int sees = sh.n - (sh.tokens - 1) + (int)(col * a.G_inverse >> 16) - u * UNIT;
#pragma unroll 1
                    for (int key = 0; key < UNIT; key++) {
                        const int t = key >> 4, row = key & 15;
                        if (row >= (t ? valid[1] : valid[0])) continue;
                        const bf16* const from = a.vp + (t ? v_at[1] : v_at[0]) + row * token + grp * 32;
#pragma unroll
                        for (int h = 0; h < H; h++)
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                const u32x4 x = *reinterpret_cast<const u32x4*>(from + h * 128 + r * 8);
#pragma unroll
                                for (int j = 0; j < 8; j++) {
                                    const float y = j & 1 ? hi_f32(x[j / 2]) : lo_f32(x[j / 2]);
                                    acc[h][j][r] += key < sees && !(fabsf(y) < INFINITY) ? y : 0.f;
                                }
                            }
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            load_v();
            __builtin_amdgcn_sched_barrier(0);
        }

        // the waves join
        const int tid = wave * 64 + lane_here();
        l = over_groups(l, [](float x, float y) { return x + y; });
        const int row_c = tid & 15, row_g = tid >> 4 & 3;
        if (row_g == 0) {
            wm[wave][row_c] = m;
            wl[wave][row_c] = l;
        }
        __syncthreads();  // Q is no longer read
        if (row_c < rows)
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float* const to = lds + (wave * rows + row_c) * PITCH + h * 128 + (row_g * 4 + r) * 8;
                    *reinterpret_cast<f32x4*>(to) = f32x4{acc[h][0][r], acc[h][1][r], acc[h][2][r], acc[h][3][r]};
                    *reinterpret_cast<f32x4*>(to + 4) = f32x4{acc[h][4][r], acc[h][5][r], acc[h][6][r], acc[h][7][r]};
                }
        __syncthreads();
        const Shared shared(a);
        constexpr int QUADS = DH / 4;  // of a row's dims
        // four dims of a row's result: to the output, or to a slot
        auto store = [&](int slot, int e, float top, float sum, const f32x4& o, const u32x2& g, bool out) {
            const int row = e / QUADS, d = e % QUADS * 4;
            if (out) {
                store_out<SEVERAL>(a, at_row(row) + d, o, sum, g);
                if constexpr (SEVERAL) {
                    const int token = (int)(row * a.G_inverse >> 16);
                    if (a.lse && d == 0)
                        a.lse[(size_t)(head0 + row - token * a.G) * a.all_rows + sh.row0 + token] = log_sum(top, sum);
                } else if (a.lse && d == 0) {
                    a.lse[(size_t)(head0 + row) * a.B + sh.row] = log_sum(top, sum);
                }
                return;
            }
            const int at = slot * ROWS + row;
            shared.put((at * DH + d) * 4, o);
            if (d == 0) shared.put_ml(at * 8, f32x2{top, sum});
        };
        // Groups of `group` parts: the last of a group to end joins it, the last group joins the groups; always in
        // order, so the result does not depend on which ends last.  The counters are zero again afterwards.
        int group = 1, groups = 1, g0 = 0, members = 1;
        if (sh.parts > 1) {
            groups = (sh.parts + GROUP - 1) / GROUP;
            group = (sh.parts + groups - 1) / (uint32_t)groups;
            groups = (sh.parts + group - 1) / (uint32_t)group;
            g0 = sh.part / (uint32_t)group * group;
            members = min(group, sh.parts - g0);
        }
        auto last_of = [&](int* count, int n) {
            __shared__ int last;
            wait_vm_all();  // what this wave has put is where the others look
            __syncthreads();
            if (tid == 0) {
                last = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
                if (last) *count = 0;
            }
            __syncthreads();
            return last != 0;
        };
        // Stage 0: this block's waves.  1: a group's parts, 2: the groups.  A row's four dims are summed by as many
        // threads as there are for them.  The time of 1 and 2 is that of getting at the parts, so many are asked for
        // at once: a thread has every `ways`-th, BATCH of them on their way together, the first while a wave per row
        // finds the parts' weights.
        float* const weight = lds;               // [GROUP, ROWS]
        float* const other = lds + GROUP * ROWS;  // [THREADS, 4]
        const int items = rows * QUADS, rows_log = rows > 1 ? 32 - __builtin_clz(rows - 1) : 0;
        for (int stage = 0;; stage++) {
            const bool out = stage == 0 ? sh.parts == 1 : stage == 2 || groups == 1;
            const int k0 = stage == 1 ? g0 : 0, step = stage == 2 ? group : 1, n = stage == 1 ? members : groups;
            const int ways = stage == 0 ? 1 : max(1, THREADS / QUADS >> rows_log);
            auto find_weights = [&]() {
                if constexpr (SEVERAL) {  // 16 lanes a row, all rows at once (4 rows behind 700: 1.5 us less than with a wave a row)
                    const int me = wave * 64 + lane_here(), r = me / 16, c = me % 16;
                    f32x2 m[GROUP / 16];
                    float most = -INFINITY, all = 0.f;
#pragma unroll
                    for (int j = 0; j < GROUP / 16; j++) {
                        const int k = c + 16 * j;
                        m[j] = shared.get_ml(k < n && r < rows ? (sh.slot(k0 + k * step) * ROWS + r) * 8 : -1);
                        if (k >= n) m[j][0] = -INFINITY;
                    }
#pragma unroll
                    for (int j = 0; j < GROUP / 16; j++) most = fmaxf(most, m[j][0]);
                    most = lane_max<16>(most);
#pragma unroll
                    for (int j = 0; j < GROUP / 16; j++) {
                        const int k = c + 16 * j;
                        const float f = k >= n ? 0.f : m[j][0] == most ? 1.f : __builtin_amdgcn_exp2f(m[j][0] - most);
                        weight[k * ROWS + r] = f;
                        if (k < n) all += m[j][1] * f;
                    }
                    all = lane_sum<16>(all);
                    if (c == 0 && r < rows) {
                        wm[0][r] = most;
                        wl[0][r] = all;
                    }
                    __syncthreads();
                    return;
                }
                const int k = tid & 63;
                for (int r = wave; r < rows; r += WAVES) {
                    const f32x2 m = shared.get_ml((sh.slot(k0 + min(k, n - 1) * step) * ROWS + r) * 8);
                    const float most = lane_max<64>(m[0]);
                    const float f = k >= n ? 0.f : m[0] == most ? 1.f : __builtin_amdgcn_exp2f(m[0] - most);
                    weight[k * ROWS + r] = f;
                    const float all = lane_sum<64>(k < n ? m[1] * f : 0.f);
                    if (k == 0) {
                        wm[0][r] = most;
                        wl[0][r] = all;
                    }
                }
                __syncthreads();
            };
            for (int e0 = 0; e0 < items; e0 += THREADS) {
                const int way = ways > 1 ? tid / QUADS >> rows_log : 0;
                const int e = e0 + (ways > 1 ? tid & ((QUADS << rows_log) - 1) : tid);
                const bool works = e < items;
                const int row = works ? e / QUADS : 0, d = e % QUADS * 4;
                u32x2 g = {0, 0};
                f32x4 o = {0.f, 0.f, 0.f, 0.f};
                float top, sum = 0.f;
                if (out) g = load_gate(a, at_row(row) + d);
                if (stage == 0) {
                    top = fmaxf(fmaxf(wm[0][row], wm[1][row]), fmaxf(wm[2][row], wm[3][row]));
#pragma unroll
                    for (int w = 0; w < WAVES; w++) {
                        const float f = wm[w][row] == top ? 1.f : __builtin_amdgcn_exp2f(wm[w][row] - top);
                        sum += wl[w][row] * f;
                        o += *reinterpret_cast<const f32x4*>(lds + (w * rows + row) * PITCH + d) * f;
                    }
                } else {
                    for (int k1 = way; k1 - way < n; k1 += BATCH * ways) {
                        f32x4 v[BATCH];
#pragma unroll
                        for (int i = 0; i < BATCH; i++) {  // behind the last part: past the buffer's end, no access
                            const int k = k1 + i * ways;
                            v[i] = shared.get(k < n ? ((sh.slot(k0 + k * step) * ROWS + row) * DH + d) * 4 : -1);
                        }
                        if (e0 == 0 && k1 == way) find_weights();
#pragma unroll
                        for (int i = 0; i < BATCH; i++) o += v[i] * weight[min(k1 + i * ways, GROUP - 1) * ROWS + row];
                    }
                    if (ways > 1) {
                        if (works && way > 0) *reinterpret_cast<f32x4*>(other + (way * items + e) * 4) = o;
                        __syncthreads();
                        if (way == 0)
                            for (int w = 1; w < ways; w++)
                                o += *reinterpret_cast<const f32x4*>(other + (w * items + (works ? e : 0)) * 4);
                    }
                    top = wm[0][row];
                    sum = wl[0][row];
                }
                if (works && way == 0) store(out ? 0 : sh.slot(stage == 0 ? sh.part : k0), e, top, sum, o, g, out);
            }
            if (out) break;
            int* const count = stage == 0 ? a.count + sh.slot(g0) : a.count2 + sh.slot0;
            if (!last_of(count, stage == 0 ? members : groups)) break;
        }
    }
}

template <int DH>
size_t lds_bytes(int rows) {
    const size_t q = 16 * 64 * (DH / 32), join = sizeof(float) * WAVES * rows * (DH + 8);
    const size_t parts = sizeof(float) * (GROUP * ROWS + THREADS * 4);
    return std::max(q, std::max(join, parts));
}

template <int DH>
bool configure() {
    for (const void* kernel : {reinterpret_cast<const void*>(attention_paged_kernel<DH, false>),
                               reinterpret_cast<const void*>(attention_paged_kernel<DH, true>)})
        if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds_bytes<DH>(ROWS)) != hipSuccess)
            return false;
    return true;
}

template <int DH>
int launch(const Args& a, hipStream_t st) {
    if (a.cu)
        attention_paged_kernel<DH, true><<<a.blocks, THREADS, lds_bytes<DH>(a.max_new < ROWS ? std::min(a.max_new * a.G, ROWS) : ROWS), st>>>(a);
    else
        attention_paged_kernel<DH, false><<<a.blocks, THREADS, lds_bytes<DH>(a.G < ROWS ? a.G : ROWS), st>>>(a);
    return hipGetLastError();
}

}  // namespace

// A call's operands as they come: n rows, or with cu (device) n list entries of up to max_new tokens each.
int paged_rows(const Paged* p, const Call& c, const int32_t* cu, int max_new, int all_rows, void* stream) {
    Args a;
    a.q = static_cast<const bf16*>(c.q);
    a.kp = static_cast<const bf16*>(c.kp);
    a.vp = static_cast<const bf16*>(c.vp);
    a.gate = static_cast<const bf16*>(c.gate);
    a.out = static_cast<bf16*>(c.out);
    a.lse = c.lse;
    a.part = p->part;
    a.ml = p->part + (size_t)2 * p->blocks * ROWS * 256;
    a.count = p->count;
    a.count2 = p->count + 2 * p->blocks;
    a.table = c.pages->table;
    a.lens = c.pages->lens;
    a.seqs = c.seqs;
    a.nseq = c.pages->nseq;
    a.max_pages = c.pages->max_pages;
    a.npages = c.pages->npages;
    a.page = c.pages->page;
    a.B = c.n;
    a.Hq = c.Hq;
    a.Hk = c.Hk;
    a.G = c.Hq / c.Hk;
    a.tiles = cu ? 1 : (a.G + ROWS - 1) / ROWS;
    a.cu = cu;
    a.max_new = max_new;
    a.all_rows = all_rows;
    a.G_inverse = (65536 + a.G - 1) / a.G;  // (exact for up to 16 columns)
    const int64_t pairs = (int64_t)c.n * c.Hk * a.tiles;
    a.halve = c.Dh == 128 && pairs >= p->blocks;  // the blocks, if the sequences are long
    a.blocks = a.halve ? p->blocks : p->cus;
    // A pair is a row with a kv head and tile.  From a pair to 16 blocks on the chunks are small, and beginning a pair
    // counts as work: as much as 6 units of keys up to a pair a CU, as 8 beyond (about 7 us). 43 sequences of up to
    // 4096, 16/4 heads of 256, take 71 us so, 91 if it counts as nothing.  Fewer pairs are better cut into whole chunks of 4.
    // With several tokens, whose joins have more rows, it counts as 10: 43 entries behind up to 4096 80 us so, 88 with 6; 150
    // behind up to 2000 (32/8 heads of 128) 127, and 136 with 8; 48 of up to 16 rows of one column 27 and 35 with 6.
    // Short sequences are one chunk, which is not cut, and joined by no one; the fewer pairs, the longer they may
    // be without the work being shared out badly: one of 300 keys (heads of 128) takes 8.4 us with 12 units and 9.8 with 8,
    // 64 of 100 to 200 (256) 12.4 with 8 and 20.0 with 4, 40 of up to 1000 22.4 and 25.6 with 12, 300 of up to 400 66 with 4
    // and 80 with 8.
    const bool several = pairs * 16 >= a.blocks, many = pairs > p->cus;
    a.unit = several ? 2 : 4;
    const int pad = cu && several ? 5 : many ? 4 : several ? 3 : 0, alone = many ? 4 : several ? 8 : 12;
    a.pad_alone = alone << 8 | pad;
    a.page_inverse = (uint32_t)std::min<uint64_t>(0xffffffffu, (uint64_t{1} << 32) / (a.page / 16));
    a.blocks_inverse = (uint32_t)(((uint64_t{1} << 32) + a.blocks - 1) / a.blocks);
    a.scale_log2 = c.scale * LOG2E;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return c.Dh == 128 ? launch<128>(a, st) : launch<256>(a, st);
}

}  // namespace q35

using namespace q35;

extern "C" void* cs1_attention_paged_create(void) {
    int device;
    const int cus = device_cus();
    if (cus < 2 || hipGetDevice(&device) != hipSuccess || !configure<128>() || !configure<256>() ||
        !chunk_configure()) {
        (void)hipGetLastError();
        return nullptr;
    }
    Paged* const p = new (std::nothrow) Paged;
    if (!p) return nullptr;
    p->device = device;
    p->cus = std::min(cus, GROUP * GROUP / 2);
    p->blocks = 2 * p->cus;
    const size_t floats = (size_t)2 * p->blocks * ROWS * (256 + 2), counts = (size_t)4 * p->blocks;
    p->part = p->chunk = nullptr;
    if (hipMalloc(reinterpret_cast<void**>(&p->part), 4 * (floats + counts)) != hipSuccess ||
        hipMalloc(reinterpret_cast<void**>(&p->chunk), chunk_bytes(p->cus)) != hipSuccess ||
        hipMemset(p->part + floats, 0, 4 * counts) != hipSuccess || hipStreamSynchronize(nullptr) != hipSuccess) {
        (void)hipGetLastError();
        if (p->part) (void)hipFree(p->part);
        if (p->chunk) (void)hipFree(p->chunk);
        delete p;
        return nullptr;
    }
    p->count = reinterpret_cast<int*>(p->part + floats);
    return p;
}

extern "C" void cs1_attention_paged_destroy(void* paged) {
    Paged* const p = static_cast<Paged*>(paged);
    if (!p) return;
    (void)hipFree(p->part);
    (void)hipFree(p->chunk);
    delete p;
}

extern "C" int cs1_attention_paged(void* paged, const void* q, const void* kp, const void* vp,
                                   const Cs1PageTable* pages, const int32_t* seqs, const void* gate, void* out,
                                   float* lse, int B, int Hq, int Hk, int Dh, float scale, void* stream) {
    const Paged* const p = static_cast<const Paged*>(paged);
    if (!p || !table_ok(pages) || (Dh != 128 && Dh != 256) || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 || B < 0)
        return hipErrorInvalidValue;
    // what the kernel counts in 32 bits: heads, bytes of a half, the pool's rows, all rows' units
    constexpr int64_t LIMIT = int64_t{1} << 31;
    const int64_t pairs = (int64_t)B * Hk * ((Hq / Hk + ROWS - 1) / ROWS);
    if ((int64_t)B * Hq > (1 << 22) || (int64_t)Hk * Dh > (1 << 24) || (int64_t)pages->npages * pages->page >= LIMIT ||
        pairs * ((int64_t)pages->max_pages * pages->page / UNIT + 1) >= LIMIT)
        return hipErrorInvalidValue;
    if (B == 0) return hipSuccess;
    if (!all_set({q, kp, vp, out}) || !on16(q) || !on16(kp) || !on16(vp) || !on16(out) || !on16(gate))
        return hipErrorInvalidValue;
    int device;
    if (hipGetDevice(&device) != hipSuccess || device != p->device) return hipErrorInvalidDevice;
    const Call c{q, kp, vp, pages, seqs, gate, out, lse, B, Hq, Hk, Dh, scale};
    return paged_rows(p, c, nullptr, 0, 0, stream);
}
