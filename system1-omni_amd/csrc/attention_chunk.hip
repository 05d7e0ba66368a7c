// Attention of several new tokens a sequence over the paged cache (cs1_attention_paged_varlen).  Row j of an entry of L
// rows, whose sequence holds n tokens, is at position p = n - L + j and sees the keys 0 .. p:
//
//   S_i = scale q . k_i,  m = max S_i,  l = sum exp(S_i - m),  out = sigmoid(gate) (sum exp(S_i - m) v_i) / l,
//   lse = m + log l.
//
// Work: an item is up to 128 columns (heads of 256) or 256 (of 128), the q heads of one kv head at some of an entry's rows, with
// all keys that they see: however many q heads share a kv head, they share its keys too.  All items of a launch form one
// line, measured in keys, that is cut into equal stretches, one a block: a prompt's part on its own and drafts
// behind long texts share the chip alike, and only the device knows the lengths.  What a stretch has of an
// item that others have parts of goes to memory, and a second launch joins the parts in order.
//
// A block has eight waves: four groups of columns by two halves.  Of a unit of 64 keys a wave makes the scores of one half of
// the keys, S^T = K Q^T, and then, with both halves' probabilities, one half of the dims of O^T += V^T P^T, on the
// 32x32x16 MFMA: what the first product leaves in a lane is what the second wants, so a pair of waves exchanges only maxima
// and the probabilities of its columns through LDS, every value is computed once, and a wave's sums are half as many
// registers as they would be if the halves of the keys stayed apart.
//
// Step t: the scores of unit t beside the exponentials of unit t - 1, whose probabilities the waves then exchange; after a
// barrier, O += P V of unit t - 1 beside the maxima of unit t.  Units move from the pages into LDS without registers; a
// wave's piece of a unit lies in one run of 16 tokens, which no page divides.
//
// P is rounded to bfloat16 for the second product, as in the prefill: the matrix cores set the time here, and a second part of
// P would cost half as much again.  Sums and maxima are float32; out is rounded once, after the gate.
//
// 2048 rows behind 30720 (24/4 heads of 256) take 1430 to 1480 us, 1080 to 1120 TFLOP/s where a large product reaches 1436: 4020
// clocks a unit over the launch, of which the matrix cores are busy 2040.  333 behind 936 (16/4 heads) take 34.5: of about 40
// thousand clocks a block 20 are its four units, 8 finding them, 6 Q and the first K, 5 the sums' way out, and then the join.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "paged.h"
#include "tile32.h"

namespace q35 {
namespace {

using tile32::k_slot;
using tile32::max_halves;
using tile32::mfma32;
using tile32::v_slot;

constexpr int THREADS = 512, WAVES = 8;
constexpr int FEW = 16;       // columns that are few
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float SLACK = 8.f;  // how far (in powers of two) a maximum may pass the exponent's base before that moves

// One stretch's item whose other parts are in other stretches, by the stretch that ends it; parts = 0: none.
struct Cut {
    int row0, tokens, head, first, parts;  // first row, rows, kv head, first stretch and number of stretches
};

struct Args {
    const bf16 *q, *kp, *vp, *gate;
    bf16* out;
    float *lse, *part, *ml;
    Cut* cuts;
    const int32_t *table, *lens, *seqs, *cu;
    int nseq, max_pages, npages, page, n, max_new, rows, Hq, Hk, G, tokens, blocks, pad, least;
    int others;  // entries of up to so many rows are another kernel's
    uint32_t page_inverse;  // 2^32 over page / 16, rounded down
    uint32_t tokens_inverse, G_inverse;  // 2^32 over tokens and 2^16 over G, rounded up
    double blocks_inverse;               // 1 / blocks
    float scale_log2;

    // rows * Hq <= 2^24 and tokens <= 256; columns < 512 and G <= 128: exact
    __device__ __forceinline__ int over_tokens(uint32_t x) const {
        return tokens == 1 ? x : (int)__umulhi(x, tokens_inverse);
    }
    __device__ __forceinline__ int over_G(uint32_t col) const { return (int)(col * G_inverse >> 16); }
};

template <int DH>
struct Form {
    static constexpr int UNIT = 64;                    // keys
    static constexpr int NC = 256 / DH;                // sets of 32 columns a wave
    static constexpr int COLS = 128 * NC;
    static constexpr int KS = DH / 16, DT = DH / 64;   // products along a head, and tiles of 32 dims of a half
    static constexpr int ROW = 2 * DH, TILE = UNIT * ROW;
    static constexpr int STAGES = 2;                   // of K and of V
    static constexpr int P_AT = 2 * STAGES * TILE, P_WAVE = 2048 * NC;
    static constexpr int TOP_AT = P_AT + WAVES * P_WAVE;
    static constexpr int FLAG_AT = TOP_AT + WAVES * 128 * NC;
    static constexpr int OUT_ROW = 2 * DH + 16;        // bytes of a column's half of the sums at the end, padded
    static constexpr int KEPT_AT = FLAG_AT + 16 > WAVES * 32 * NC * OUT_ROW ? FLAG_AT + 16 : WAVES * 32 * NC * OUT_ROW;
    static constexpr int BYTES = KEPT_AT + 3 * 64 * 8;  // (what a wave has for the search of many entries, see find_window)
    static_assert(BYTES <= 160 * 1024, "fits in the LDS");
};

// An entry's sequence, first row, rows, and the position of the first one (less than 0: rows without keys).
struct Entry {
    int s, row0, rows, pos;
};
__device__ __forceinline__ Entry entry_of(const Args& a, int i) {
    Entry e{-1, 0, 0, 0};
    if (i >= a.n) return e;
    const int lo = a.cu[i], hi = a.cu[i + 1], s = listed_seq(a.seqs, i, a.nseq);  // (asked for together)
    if (lo < 0 || hi <= lo || lo >= a.rows) return e;
    const int rows = min(min(hi, a.rows) - lo, a.max_new);
    if (rows <= a.others) return e;
    e.s = s;
    e.row0 = lo;
    e.rows = rows;
    const int64_t held = e.s < 0 ? 0 : min((int64_t)max(a.lens[e.s], 0), (int64_t)a.max_pages * a.page);
    e.pos = (int)(held - (hi - lo));
    return e;
}

// The line: `c` items of an entry for one kv head, tokens (c + 1) keys and the pad more than those before its rows
__device__ __forceinline__ int64_t line_of(const Args& a, int pos, int64_t c) {
    return c * (max(pos, 0) + a.pad) + a.tokens * (c * (c + 1) / 2);
}
__device__ __forceinline__ int items_of(const Args& a, int rows) { return a.over_tokens(rows + a.tokens - 1); }
__device__ __forceinline__ int64_t weight_of(const Args& a, const Entry& e) {
    return line_of(a, e.pos, items_of(a, e.rows)) * a.Hk;
}

__device__ __forceinline__ int scalar(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t scalar64(int64_t x, int lane) {
    return (int64_t)(uint32_t)scalar((int)x, lane) | (int64_t)scalar((int)(x >> 32), lane) << 32;
}
// The lane's number, found again where it is asked for: what follows from it would otherwise be kept in registers
// over the loop over the keys, which has none to spare.
__device__ __forceinline__ int lane_here() {
    int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));
    asm volatile("" : "+v"(lane));
    return lane;
}
// Sum over this lane and those below: within rows of 16 lanes, then each row's last lane to the next row (into rows
// 1 and 3), then lane 31 to the upper half.
__device__ __forceinline__ int64_t wave_scan(int64_t x) {
#define Q35_ADD(ctrl, rows)                                                                                \
    x += (int64_t)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, false) |               \
         (int64_t)__builtin_amdgcn_update_dpp(0, (int)(x >> 32), ctrl, rows, 0xf, false) << 32
    Q35_ADD(0x111, 0xf);
    Q35_ADD(0x112, 0xf);
    Q35_ADD(0x114, 0xf);
    Q35_ADD(0x118, 0xf);
    Q35_ADD(0x142, 0xa);
    Q35_ADD(0x143, 0xc);
#undef Q35_ADD
    return x;
}

__device__ __forceinline__ u32x2 read_tr3(uint32_t at) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u32x2,
                              __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at));
}

// Dims of an output from their sums over l (zero: no key); the words of g have their gates, if there are any.
__device__ __forceinline__ uint32_t out_of(bool gated, float o0, float o1, float l, float inv, uint32_t g) {
    if (gated) {
        o0 *= gate_sigmoid(lo_f32(g));
        o1 *= gate_sigmoid(hi_f32(g));
    }
    return pack2(l != 0.f ? o0 * inv : 0.f, l != 0.f ? o1 * inv : 0.f);
}
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * LN2; }

// Two transfers of 1024 bytes (dma16) in a row of LDS: the offset in the instruction counts in LDS and in memory, so the
// second scalar offset is less by 1024.
__device__ __forceinline__ void dma16x2(const u32x4& rsrc, uint32_t lds, int voff0, int voff1, int soff, int step) {
    const int soff1 = __builtin_amdgcn_readfirstlane(soff + step - 1024);
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 3\n\t"
        "buffer_load_dwordx4 %1, %3, %4 offen lds\n\tbuffer_load_dwordx4 %2, %3, %5 offen offset:1024 lds" ::"s"(lds),
        "v"(voff0), "v"(voff1), "s"(rsrc), "s"(soff), "s"(soff1)
        : "memory");
}

#define Q35_INLINE __attribute__((always_inline))
#define Q35_RARELY(x) __builtin_expect(!!(x), 0)  // (what is rare is laid out behind the loop over the keys)

// The arguments, read again where they are asked for: what only begins or ends an item is not to be held in scalar
// registers over the loop over the keys.  (A kernel's arguments begin the segment that this points to.)
__device__ __forceinline__ const Args& arguments() {
    auto p = __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const Args*)p;
}

template <int DH>
__global__ void __launch_bounds__(THREADS, 1) attention_chunk_kernel(const Args) {
    using F = Form<DH>;
    constexpr int UNIT = F::UNIT, NC = F::NC, COLS = F::COLS, KS = F::KS, DT = F::DT, ROW = F::ROW, TILE = F::TILE;
    constexpr int STAGES = F::STAGES;
    extern __shared__ __align__(16) unsigned char smem[];
    const int wave = uniform(threadIdx.x >> 6);
    const int cg = wave & 3, half = wave >> 2;  // group of columns; half of the keys, then of the dims
    constexpr int MINE = UNIT / WAVES, PER = 1024 / ROW, NI = MINE / PER, CHUNKS = ROW / 16;  // rows of a wave's transfers
    const int r0 = wave * MINE;

    // Of the entries' part of the line in which `pos` is: 64 entries, a lane each, with their weights up to and with them, from
    // the line's place window_at on.
    Entry mine;
    int64_t own_weight, upto, window_at = 0, pos, end, each;
    // more entries: lane i has the weights of windows 2 i and 2 i + 1 of 64 entries, and those up to them (in LDS: the loop over
    // the keys needs the registers)
    int64_t* const kept = reinterpret_cast<int64_t*>(smem + F::KEPT_AT);
    auto find_window = [&](const Args& a) Q35_INLINE {
        const int at = lane_here();
        const int64_t all = kept[128 + at], w0 = kept[at], w1 = kept[64 + at];
        const int lane = __ffsll((unsigned long long)__ballot(all > pos)) - 1;
        const int64_t first = scalar64(w0, lane), before = scalar64(all, lane) - first - scalar64(w1, lane);
        const bool second = pos >= before + first;
        window_at = second ? before + first : before;
        mine = entry_of(a, (2 * lane + second) * 64 + lane_here());
        own_weight = weight_of(a, mine);
        upto = wave_scan(own_weight);
    };
    int block;
    {
        const Args& a = arguments();
        const int lane = lane_here(), windows = (a.n + 63) / 64;
        int64_t total;
        if (windows == 1) {
            mine = entry_of(a, lane);
            own_weight = weight_of(a, mine);
            upto = wave_scan(own_weight);
            total = scalar64(upto, 63);
        } else {
            int64_t* const sums = reinterpret_cast<int64_t*>(smem);
            for (int w = wave; w < windows; w += WAVES) {
                const int64_t all = wave_scan(weight_of(a, entry_of(a, w * 64 + lane)));
                if (lane == 63) sums[w] = all;
            }
            __syncthreads();
            const int64_t w0 = 2 * lane < windows ? sums[2 * lane] : 0, w1 = 2 * lane + 1 < windows ? sums[2 * lane + 1] : 0;
            const int64_t all = wave_scan(w0 + w1);
            if (wave == 0) {
                kept[lane] = w0;
                kept[64 + lane] = w1;
                kept[128 + lane] = all;
            }
            __syncthreads();
            total = scalar64(all, 63);
        }
        // (one more than need be; the line is far shorter than 2^50)
        each = max((int64_t)((double)total * a.blocks_inverse) + 1, (int64_t)a.least);
        each = (int64_t)(uint32_t)uniform((int)each) | (int64_t)uniform((int)(each >> 32)) << 32;
        // neighbours of the line, which share keys, are on one XCD
        block = a.blocks % 8 == 0 ? (blockIdx.x & 7) * (a.blocks / 8) + (blockIdx.x >> 3) : blockIdx.x;
        pos = block * each;
        end = min(total, pos + each);
        if (threadIdx.x == 0) a.cuts[block].parts = 0;
        if (pos >= end) return;
        if (windows > 1) find_window(a);
    }
    const int64_t begin = pos;

    // The end of an item that began elsewhere comes last of a stretch, so that at any time those blocks that have as much
    // of a line (the q heads of a kv head at different rows, all with nearly the same keys) are at the same key: whole items and
    // beginnings go on from key 0 at once, and what is left of the first item is as far from its end as the stretch is.  (Where
    // a stretch is shorter than its item there is less of that than a second search takes.)
    // A unit that is read by the 32 blocks of an XCD comes from its L2 then (2048 rows behind 30720, 24/4 heads of
    // 256: 1617 us in the line's order, 1460 so).
    enum { STRAIGHT, FIRST_IS_LEFT, AT_FIRST } order = STRAIGHT;
    for (;;) {
        int seq, row0, ntok, pos0, keys, head = 0, u0, u1;
        bool whole, began;  // all of the item's keys are in this stretch; they begin there
        int parts = 0;      // of an item that ends here and began elsewhere
        // The item at `pos`.  What a stretch has of the pad alone is no part of the item: a stretch without keys of it goes on.
        // (Item of no keys: its zeros are written where it begins.)
        for (const Args& a = arguments();;) {
            head = 0;
            const int el = __ffsll((unsigned long long)__ballot(window_at + upto > pos)) - 1;
            const int erow = scalar(mine.row0, el), erows = scalar(mine.rows, el);
            const int own_items = items_of(a, mine.rows), epos = scalar(mine.pos, el), items = scalar(own_items, el);
            const int64_t own = scalar64(line_of(a, mine.pos, own_items), el);
            int64_t hstart = window_at + scalar64(upto - own_weight, el);
            seq = scalar(mine.s, el);
#pragma unroll 1
            for (; hstart + own <= pos; hstart += own) head++;
            int c = 0;  // the last item that begins at or before pos, and where it does
            int64_t istart = hstart;
            for (int c0 = 0; c0 < items; c0 += 64) {
                const int it = c0 + lane_here();
                const int64_t at = hstart + line_of(a, epos, it);
                const int n = __popcll(__ballot(it < items && at <= pos));
                if (n == 0) break;
                c = c0 + n - 1;
                istart = scalar64(at, n - 1);
            }
            const int64_t iend = istart + max(epos, 0) + a.pad + (int64_t)a.tokens * (c + 1);
            const int tok0 = c * a.tokens;
            ntok = min(a.tokens, erows - tok0);
            row0 = erow + tok0;
            pos0 = epos + tok0;  // of its first row
            keys = max(pos0 + ntok, 0);
            const int units = (keys + UNIT - 1) / UNIT;
            auto cut = [&](int64_t x) {
                return x <= istart ? 0 : x >= iend ? units : (int)min((int64_t)units, max(x - istart - a.pad, (int64_t)0) / UNIT);
            };
            u0 = uniform(cut(begin));
            u1 = uniform(cut(end));
            began = u0 == 0;
            whole = began && u1 == units;
            pos = min(iend, end);
            const bool some = u0 < u1 || (units == 0 && istart >= begin);
            if (some && order == STRAIGHT && !began && pos < end && iend - istart <= each) {
                order = FIRST_IS_LEFT;
            } else if (some) {
                if (began || u1 < units) break;
                parts = 2;
#pragma unroll 1
                for (int64_t x = begin - each; cut(x) > 0; x -= each) parts++;
                break;
            }
            if (pos >= end) {
                if (order != FIRST_IS_LEFT) return;
                order = AT_FIRST;
                pos = begin;
            }
            if (a.n > 64) find_window(a);
        }
        // a column is a row and a q head of the kv head's
        const int G = uniform(arguments().G), Hq = uniform(arguments().Hq), cols = ntok * G;
        const uint32_t G_inverse = uniform(arguments().G_inverse);
        const bool active = cg * 32 * NC < cols;
        const int low_key = pos0 + (int)(cg * 32 * NC * G_inverse >> 16);  // that the wave's first column sees
        struct Column {
            int token, head;
            size_t at;  // of q, gate and out
        };
        auto column = [&](int col) Q35_INLINE {
            Column x;
            x.token = (int)(col * G_inverse >> 16);
            x.head = head * G + col - x.token * G;
            x.at = ((size_t)(row0 + x.token) * Hq + x.head) * DH;
            return x;
        };
        // Q, a pair's columns by halves: whole lines here, and as operands by way of LDS (operands from memory, 16 bytes a
        // column at a time, took 2 us more)
        constexpr int QN = 16 * NC * CHUNKS / 64;
        u32x4 qs[QN];
        {
            const bf16* const q = arguments().q;
#pragma unroll
            for (int i = 0; i < QN; i++) {
                const int at = i * 64 + lane_here(), col = cg * 32 * NC + half * 16 * NC + at / CHUNKS;
                qs[i] = *reinterpret_cast<const u32x4*>(q + column(min(col, cols - 1)).at + at % CHUNKS * 8);
            }
        }
        int last_key[NC];  // that this lane's columns see
#pragma unroll
        for (int n = 0; n < NC; n++) {
            const int col = (cg * NC + n) * 32 + (lane_here() & 31);
            last_key[n] = col < cols ? pos0 + column(col).token : -1;
        }

        // The next 64 runs of 16 tokens: lane i has the pool's run of run number i from here on, -1 if its page is out of range
        constexpr int RUNS = UNIT / 16, LOOK = 64 / RUNS;
        int where = 0, from_unit = 0;
        uint64_t bad = 0;
        auto look_up = [&](int unit) Q35_INLINE {
            const auto& a = arguments();
            from_unit = unit;
            const uint32_t run = unit * RUNS + lane_here(), page = (uint32_t)a.page / 16;
            where = -1;
            const bool held = 16 * run < (uint32_t)keys;
            if (held) {
                uint32_t slot = __umulhi(run, a.page_inverse);
                slot += (slot + 1) * page <= run;
                const int pg = a.table[(size_t)seq * a.max_pages + slot];
                if (pg >= 0 && pg < a.npages) where = pg * page + run - slot * page;
            }
            bad = __ballot(held && where < 0);
        };
        look_up(u0);
        const int keys_here = min(keys, u1 * UNIT);
        const uint32_t token = 2 * (uint32_t)arguments().Hk * DH;  // bytes
        const uint64_t k_pool = reinterpret_cast<uint64_t>(arguments().kp) + (uint32_t)(head * ROW) + r0 % 16 * token;
        const uint64_t v_pool = reinterpret_cast<uint64_t>(arguments().vp) + (uint32_t)(head * ROW) + r0 % 16 * token;
        // This wave's rows of a unit: where they lie in a pool, and bytes up to the last one's end (0: none)
        struct Piece {
            uint64_t at;
            uint32_t bytes;
        };
        constexpr uint32_t NO_STRIDE = 0xffffu;
        const uint32_t whole_bytes = (MINE - 1) * token + ROW;
        auto run_of = [&](int unit) Q35_INLINE { return scalar(where, ((unit - from_unit) * RUNS + r0 / 16) & 63); };
        auto piece_of = [&](int unit) Q35_INLINE {
            const int run = run_of(unit);
            const int rows = max(0, min(MINE, min(keys_here - unit * UNIT - r0, run * MINE + MINE)));  // (none for run -1)
            return Piece{(uint32_t)max(run, 0) * (uint64_t)(16 * token), rows > 0 ? (rows - 1) * token + ROW : 0};
        };
        auto rows_at = [&](uint64_t pool, const Piece& p) Q35_INLINE {
            const uint64_t at = pool + p.at;
            return u32x4{(uint32_t)uniform((int)(uint32_t)at), (uint32_t)uniform((int)(uint32_t)(at >> 32)) & NO_STRIDE,
                         (uint32_t)uniform(p.bytes), 0x00020000u};
        };
        // Lane l fills place l % CHUNKS of row l / CHUNKS of a transfer with the chunk that belongs there.  Other rows of a piece
        // exchange other bits (k_slot, v_slot).
        const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
        const uint32_t lds0 = (uint32_t)uniform((int)lds) + r0 * ROW;
        int k_lane, v_lane;
        {
            const int lane = lane_here(), row = lane / CHUNKS, place = lane % CHUNKS;
            k_lane = row * token + (k_slot(r0 + row, place) << 4);
            v_lane = row * token + (v_slot(row, place) << 4);
        }
        // A wave's transfers of a unit go one by one between the products; where there are only two, together, which saves a
        // few instructions (1000 rows behind 8000, 32/8 heads of 128: 160 us apart, 157 so; of four, twos are slower: 2048
        // behind 30720, 24/4 heads of 256, 1460 us apart, 1471 in twos).
        constexpr int SET = NI == 2 ? 2 : 1, SETS = NI / SET;
        auto move = [&](const u32x4& r, int at, int set, auto lane_of) Q35_INLINE {
            const uint32_t to = (uint32_t)uniform((int)(lds0 + at + set * SET * 1024));
            const int from = uniform(set * SET * PER * token);
            if constexpr (SET == 2)
                dma16x2(r, to, lane_of(0), lane_of(1), from, PER * token);
            else
                dma16(r, to, lane_of(set), from);
        };
        auto move_k = [&](const u32x4& r, int stage, int set) Q35_INLINE {
            move(r, stage * TILE, set, [&](int i) Q35_INLINE { return k_lane ^ (i * PER) << 4; });
        };
        auto move_v = [&](const u32x4& r, int stage, int set) Q35_INLINE {
            move(r, (STAGES + stage) * TILE, set, [&](int i) Q35_INLINE { return PER == 2 && i & 1 ? v_lane ^ 12 << 4 : v_lane; });
        };

        f32x16 o[NC][DT], s[NC], old[NC];  // scores of the last unit, and of the one before
#pragma unroll
        for (int n = 0; n < NC; n++)
#pragma unroll
            for (int t = 0; t < DT; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[n][t][i] = 0.f;
        float m[NC], l[NC], top[NC];
#pragma unroll
        for (int n = 0; n < NC; n++) m[n] = top[n] = -INFINITY, l[n] = 0.f;

        Piece now = piece_of(u0), next = piece_of(u0 + 1);  // of units t and t + 1
#pragma unroll
        for (int j = 0; j < SETS; j++) move_k(rows_at(k_pool, now), 0, j);
        constexpr int Q_AT = STAGES * TILE;  // (where no value is before the first step's barrier)
#pragma unroll
        for (int i = 0; i < QN; i++) {
            const int at = i * 64 + lane_here(), col = half * 16 * NC + at / CHUNKS;
            *reinterpret_cast<u32x4*>(smem + Q_AT + (cg * 32 * NC + col) * ROW + (k_slot(col, at % CHUNKS) << 4)) = qs[i];
        }
        if (threadIdx.x == 0) *reinterpret_cast<int*>(smem + F::FLAG_AT) = 0;
        const float scale_log2 = arguments().scale_log2;
        wait_vm_all();
        __syncthreads();
        int stage = 0;  // of unit t's K, and of its V

        // Operands in LDS, by lane.  K: row c32 of a half, chunk 2 i + hh; in its place (k_slot) the chunk's low bits are
        // exchanged by the row's, and 2 i is an exchange of bits too.  V^T as the transposing read hands it out: of a tile of this
        // half's dims, keys 16 j .. of this wave's half (j < 2) and of the other one; a tile is four chunks, which are an
        // exchange of bits again.
        uint32_t k_base, v_base, p_base, top_base;
        {
            const int lane = lane_here(), c32 = lane & 31, gi = lane & 15, gg = lane >> 4, vrow = 4 * (gg >> 1) + (gi >> 2);
            const int vdim = half * (DH / 2) + 16 * (gg & 1) + 4 * (gi & 3);
            k_base = lds + (32 * half + c32) * ROW + (k_slot(c32, lane >> 5) << 4);
            v_base = lds + STAGES * TILE + (half * 32 + vrow) * ROW + (v_slot(vrow, vdim >> 3) << 4) + 2 * (vdim & 7);
            p_base = lds + F::P_AT + wave * F::P_WAVE + lane * 16;
            top_base = lds + F::TOP_AT + (wave * NC * 32 + c32) * 4;
        }
        const int other = 4 - 8 * half;  // from this wave to the other one of its pair
        auto lds_u4 = [](uint32_t at) Q35_INLINE { return (__attribute__((address_space(3))) u32x4*)at; };
        auto lds_f = [](uint32_t at) Q35_INLINE { return (__attribute__((address_space(3))) float*)at; };
        u32x4 qf[NC][KS];
        {
            const int lane = lane_here(), c32 = lane & 31;
            const uint32_t q = lds + Q_AT + (cg * 32 * NC + c32) * ROW + (k_slot(c32, lane >> 5) << 4);
#pragma unroll
            for (int n = 0; n < NC; n++)
#pragma unroll
                for (int i = 0; i < KS; i++) qf[n][i] = *lds_u4((q + n * 32 * ROW ^ (i & 7) << 5) + (i >> 3) * 256);
        }
        constexpr int K_READ = DH == 256 ? 6 : 3, V_READ = DH == 256 ? 6 : 3;  // operands read ahead
        u32x4 kf[KS], vf[4 * DT];
        auto read_k = [&](uint32_t k, int i) Q35_INLINE { kf[i] = *lds_u4((k ^ (i & 7) << 5) + (i >> 3) * 256); };
        auto read_v = [&](uint32_t v, int i) Q35_INLINE {
            const int d = i % DT, j = i / DT;
            const uint32_t from = (v ^ d << 6) + (j < 2 ? 0 : (32 - 64 * half) * ROW) + (j & 1) * 16 * ROW;
            const u32x2 lo = read_tr3(from), hi = read_tr3(from + 8 * ROW);
            vf[i] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        };
        // The values of a unit from key k0 on that are no finite numbers, from the pages.
        auto add_odd = [&](int k0) Q35_INLINE {
            const auto& a = arguments();
            const int lane = lane_here();
            for (int key = k0; key < min(k0 + UNIT, keys); key++) {
                const int page = key / a.page, pg = a.table[(size_t)seq * a.max_pages + page];
                if (pg < 0 || pg >= a.npages) continue;
                const size_t slot = (size_t)pg * a.page + (key - page * a.page);
                const bf16* const from = a.vp + (slot * a.Hk + head) * DH + half * (DH / 2) + 4 * (lane >> 5);
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        const u32x2 x = *reinterpret_cast<const u32x2*>(from + 32 * d + 8 * g);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float y = e & 1 ? hi_f32(x[e / 2]) : lo_f32(x[e / 2]);
#pragma unroll
                            for (int n = 0; n < NC; n++)
                                o[n][d][4 * g + e] += key <= last_key[n] && !(fabsf(y) < INFINITY) ? y : 0.f;
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
            }
        };
        // Of a unit's scores in `x`: the exponentials, from a base that moves (seldom) with the maxima of both halves.
        float base[NC];
        auto move_base = [&](const float* theirs) Q35_INLINE {
            bool rises = false;
#pragma unroll
            for (int n = 0; n < NC; n++) {
                top[n] = fmaxf(top[n], theirs[n]);
                rises |= !(top[n] <= m[n] + SLACK);
            }
            if (Q35_RARELY(__any(rises))) {
#pragma unroll
                for (int n = 0; n < NC; n++) {
                    const float to = fmaxf(m[n], top[n]);
                    const float by = __builtin_amdgcn_exp2f(m[n] - (to == -INFINITY ? 0.f : to));
                    m[n] = to;
                    l[n] *= by;
#pragma unroll
                    for (int d = 0; d < DT; d++) o[n][d] *= by;
                }
            }
#pragma unroll
            for (int n = 0; n < NC; n++) base[n] = m[n] == -INFINITY ? 0.f : m[n];
        };
        u32x4 pf[NC][2];
        auto exponential = [&](f32x16* x, int e) Q35_INLINE {
#pragma unroll
            for (int n = 0; n < NC; n++) {
                x[n][e] = __builtin_amdgcn_exp2f(fmaf(x[n][e], scale_log2, -base[n]));
                l[n] += x[n][e];
                if (e & 1) pf[n][e >> 3][e >> 1 & 3] = pack2(x[n][e - 1], x[n][e]);
            }
        };
        // (a lane's probabilities are in the second product's order: keys 16 j + 4 hh .. + 3 and 8 behind these)
        auto hand_out = [&]() Q35_INLINE {
#pragma unroll
            for (int n = 0; n < NC; n++)
#pragma unroll
                for (int j = 0; j < 2; j++) *lds_u4(p_base + (n * 2 + j) * 1024) = pf[n][j];
        };
        auto read_top = [&](float* theirs) Q35_INLINE {
#pragma unroll
            for (int n = 0; n < NC; n++) theirs[n] = *lds_f(top_base + (other * NC + n) * 128);
        };
        auto read_p = [&](u32x4 (*theirs)[2]) Q35_INLINE {
#pragma unroll
            for (int n = 0; n < NC; n++)
#pragma unroll
                for (int j = 0; j < 2; j++) theirs[n][j] = *lds_u4(p_base + other * F::P_WAVE + (n * 2 + j) * 1024);
        };
        auto add_product = [&](const u32x4 (*theirs)[2], int i) Q35_INLINE {
#pragma unroll
            for (int n = 0; n < NC; n++)
                o[n][i % DT] = mfma32(vf[i], i < 2 * DT ? pf[n][i / DT] : theirs[n][i / DT - 2], o[n][i % DT]);
        };
        auto write_top = [&]() Q35_INLINE {  // (both lane halves have the same)
#pragma unroll
            for (int n = 0; n < NC; n++) *lds_f(top_base + n * 128) = top[n];
        };
        auto end_half = [&]() Q35_INLINE {
            __builtin_amdgcn_s_waitcnt(0x0f70 | NI);
            __syncthreads();
        };
        // Step t where units t - 1 and t are whole, all rows see all of them, and so are the two behind.
        auto plain_step = [&](int t) Q35_INLINE {
            u32x4 rows = rows_at(k_pool, next);
            const uint32_t k = k_base + stage * TILE, v = v_base + (stage ^ 1) * TILE;
            float their_top[NC];
            read_top(their_top);
#pragma unroll
            for (int n = 0; n < NC; n++) old[n] = s[n];
#pragma unroll
            for (int i = 0; i < K_READ; i++) read_k(k, i);
#pragma unroll
            for (int n = 0; n < NC; n++)
#pragma unroll
                for (int i = 0; i < 16; i++) s[n][i] = 0.f;
            __builtin_amdgcn_sched_barrier(0);
            // a product, the exponentials of scores and a transfer beside it
            constexpr int LEAD = 3, N = 16 - LEAD;  // products before the exponentials begin
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const int i = j / NC, n = j % NC;
                if (j == LEAD) {
                    move_base(their_top);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (n == 0 && i + K_READ < KS) read_k(k, i + K_READ);
                s[n] = mfma32(kf[i], qf[n][i], s[n]);
#pragma unroll
                for (int x = 0; x < SETS; x++)
                    if (j == LEAD + 1 + x * (8 / SETS)) move_k(rows, stage ^ 1, x);
                if (j >= LEAD)
#pragma unroll
                    for (int e = (j - LEAD) * 16 / N; e < (j - LEAD + 1) * 16 / N; e++) exponential(old, e);
                __builtin_amdgcn_sched_barrier(0);
            }
            hand_out();
            rows = rows_at(v_pool, now);
            end_half();
            now = next;
            next = Piece{(uint32_t)run_of(t + 2) * (uint64_t)(16 * token), whole_bytes};
            u32x4 their_p[NC][2];
#pragma unroll
            for (int i = 0; i < V_READ; i++) read_v(v, i);
            read_p(their_p);
            __builtin_amdgcn_sched_barrier(0);
            // a product, the maxima of scores and a transfer beside it
            float most[NC];
#pragma unroll
            for (int n = 0; n < NC; n++) most[n] = s[n][0];
#pragma unroll
            for (int i = 0; i < 4 * DT; i++) {
                if (i + V_READ < 4 * DT) read_v(v, i + V_READ);
                add_product(their_p, i);
#pragma unroll
                for (int x = 0; x < SETS; x++)
                    if (i == 1 + x * (2 * DT / SETS)) move_v(rows, stage, x);
                constexpr int E = 16 / (2 * DT);  // scores each, in the first half
#pragma unroll
                for (int n = 0; n < NC; n++) {
                    if (i < 2 * DT)
#pragma unroll
                        for (int e = i * E; e < (i + 1) * E; e++) most[n] = fmaxf(most[n], s[n][e]);
                    if (i == 2 * DT) top[n] = max_halves(most[n]) * scale_log2;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            write_top();
            end_half();
            stage ^= 1;
        };
        // Any step: the first has no unit before it, the last none of its own.  (One copy of the code, part behind part: what a
        // short item runs has to come from memory first.)
        auto step = [&](int t) Q35_INLINE {
            const bool first = t == u0, last = t == u1;
            if (active && !first) {
                float their_top[NC];
                read_top(their_top);
                move_base(their_top);
#pragma unroll
                for (int e = 0; e < 16; e++) exponential(s, e);
                hand_out();
            }
            if (!last) {
                const u32x4 rows = rows_at(k_pool, next);
#pragma unroll
                for (int i = 0; i < SETS; i++) move_k(rows, stage ^ 1, i);
                if (active) {
                    const uint32_t k = k_base + stage * TILE;
#pragma unroll
                    for (int i = 0; i < K_READ; i++) read_k(k, i);
#pragma unroll
                    for (int n = 0; n < NC; n++)
#pragma unroll
                        for (int i = 0; i < 16; i++) s[n][i] = 0.f;
#pragma unroll
                    for (int i = 0; i < KS; i++) {
                        if (i + K_READ < KS) read_k(k, i + K_READ);
#pragma unroll
                        for (int n = 0; n < NC; n++) s[n] = mfma32(kf[i], qf[n][i], s[n]);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                __builtin_amdgcn_s_waitcnt(0x0f70 | NI);
            } else {
                wait_vm_all();
            }
            __syncthreads();
            // Where some rows must not see some of the keys, a value that is an infinity or NaN is not taken away by a weight of
            // zero: it leaves the unit here, and is added below to the rows that see it.
            const bool partly = !first && t * UNIT - 1 > pos0;
            int odd = 0;
            if (partly) {
                u32x4* const x = reinterpret_cast<u32x4*>(smem + (STAGES + (stage ^ 1)) * TILE) + wave * 64 * NI + lane_here();
                bool here = false;
#pragma unroll 1
                for (int i = 0; i < NI; i++) {
                    u32x4 y = x[64 * i];
                    bool any = false;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        any |= odd16(y[e]);
                        y[e] = common16(y[e]);
                    }
                    if (any) x[64 * i] = y;
                    here |= any;
                }
                int* const flag = reinterpret_cast<int*>(smem + F::FLAG_AT);
                if (here) *flag = 1;
                __syncthreads();
                odd = uniform(*flag);
            }
            if (!last) {
                const u32x4 rows = rows_at(v_pool, now);
#pragma unroll
                for (int i = 0; i < SETS; i++) move_v(rows, stage, i);
                const uint32_t lost = (uint32_t)(bad >> ((t - from_unit) * RUNS + 2 * half & 63)) & 3;  // runs without a page
                if (t + 2 >= from_unit + LOOK && t + 2 < u1) look_up(t + 1);
                now = next;
                next = piece_of(t + 2);
                if (active) {
                    const int k0 = t * UNIT + 32 * half;
                    if (k0 + 31 > low_key || lost) {
                        const int hh = lane_here() >> 5;
#pragma unroll
                        for (int n = 0; n < NC; n++)
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                const int key = 8 * (i >> 2) + 4 * hh + (i & 3);
                                if (k0 + key > last_key[n] || (lost >> (i >> 3) & 1)) s[n][i] = -INFINITY;
                            }
                    }
#pragma unroll
                    for (int n = 0; n < NC; n++) {
                        float most = s[n][0];
#pragma unroll
                        for (int e = 1; e < 16; e++) most = fmaxf(most, s[n][e]);
                        top[n] = max_halves(most) * scale_log2;
                    }
                    write_top();
                }
            }
            if (active && !first) {
                const uint32_t v = v_base + (stage ^ 1) * TILE;
                u32x4 their_p[NC][2];
#pragma unroll
                for (int i = 0; i < V_READ; i++) read_v(v, i);
                read_p(their_p);
#pragma unroll
                for (int i = 0; i < 4 * DT; i++) {
                    if (i + V_READ < 4 * DT) read_v(v, i + V_READ);
                    add_product(their_p, i);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (odd) add_odd((t - 1) * UNIT);
            }
            if (!last) __builtin_amdgcn_s_waitcnt(0x0f70 | NI);
            __syncthreads();
            if (partly && threadIdx.x == 0) *reinterpret_cast<int*>(smem + F::FLAG_AT) = 0;
            if (!last) stage ^= 1;
        };
        if (u0 < u1)
            for (int t = u0; t <= u1;) {
                // units that all rows see, with whole units behind them whose pages are known and in range
                int stop = min(min((pos0 + 1) / UNIT, keys_here / UNIT - 2), from_unit + LOOK - 2);
                if (bad != 0 || !active || t == u0) stop = t;
                for (; t < stop; t++) plain_step(t);
                step(t++);
            }
        wait_vm_all();  // (transfers of nothing, behind the last unit)

        // l: this wave's keys, both lane halves, and the other wave's
        if (active) {
#pragma unroll
            for (int n = 0; n < NC; n++) {
                l[n] += __shfl_xor(l[n], 32, 64);
                *lds_f(top_base + n * 128) = l[n];
            }
        }
        __syncthreads();
        if (active) {
#pragma unroll
            for (int n = 0; n < NC; n++) {
                const float theirs = *lds_f(top_base + (other * NC + n) * 128);
                l[n] = half == 0 ? l[n] + theirs : theirs + l[n];
            }
        }
        __syncthreads();  // (what was read may lie where another wave writes now)
        // The sums go through LDS, so that whole lines of a column are stored (and one loop's code does it, not one for
        // each register: code that runs once comes from memory).
        const Args& a = arguments();
        const int slot = 2 * block + began;
        if (active) {
            const int lane = lane_here(), c32 = lane & 31, hh = lane >> 5;
            unsigned char* const mine_at = smem + wave * 32 * NC * F::OUT_ROW;
#pragma unroll
            for (int n = 0; n < NC; n++)
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int g = 0; g < 4; g++)
                        *reinterpret_cast<f32x4*>(mine_at + (n * 32 + c32) * F::OUT_ROW + (32 * d + 8 * g + 4 * hh) * 4) =
                            f32x4{o[n][d][4 * g], o[n][d][4 * g + 1], o[n][d][4 * g + 2], o[n][d][4 * g + 3]};
            if (!whole) {
                constexpr int QUADS = DH / 8, AT_ONCE = 64 / QUADS;  // quads of a column's half; columns at a time
#pragma unroll 2
                for (int i = 0; i < 32 * NC / AT_ONCE; i++) {
                    const int here = i * AT_ONCE + lane / QUADS, d = lane % QUADS * 4, col = cg * 32 * NC + here;
                    const f32x4 x = *reinterpret_cast<const f32x4*>(mine_at + here * F::OUT_ROW + d * 4);
                    if (col < cols)
                        *reinterpret_cast<f32x4*>(a.part + ((size_t)slot * COLS + col) * DH + half * (DH / 2) + d) = x;
                }
            } else {
                // a lane has eight dims of every AT_ONCE-th column, whose gates are asked for together
                constexpr int LANES = DH / 16, AT_ONCE = 64 / LANES, EACH = 32 * NC / AT_ONCE;
                const int first = lane / LANES, d = lane % LANES * 8;
                u32x4 gates[EACH];
                size_t to[EACH];
#pragma unroll
                for (int i = 0; i < EACH; i++) {
                    to[i] = column(min(cg * 32 * NC + i * AT_ONCE + first, cols - 1)).at + half * (DH / 2) + d;
                    gates[i] = u32x4{0, 0, 0, 0};
                    if (a.gate) gates[i] = *reinterpret_cast<const u32x4*>(a.gate + to[i]);
                }
                float inv[NC];  // (the hardware's reciprocal, within a float32 step as the gate's)
#pragma unroll
                for (int n = 0; n < NC; n++) inv[n] = __builtin_amdgcn_rcpf(l[n]);
#pragma unroll
                for (int i = 0; i < EACH; i++) {
                    const int here = i * AT_ONCE + first, n = i * AT_ONCE / 32;
                    const f32x4* const x = reinterpret_cast<const f32x4*>(mine_at + here * F::OUT_ROW + d * 4);
                    const f32x4 x0 = x[0], x1 = x[1];
                    const float sum = __shfl(l[n], here & 31, 64), r = __shfl(inv[n], here & 31, 64);
                    const bool gated = a.gate != nullptr;
                    const u32x4 y = {out_of(gated, x0[0], x0[1], sum, r, gates[i][0]), out_of(gated, x0[2], x0[3], sum, r, gates[i][1]),
                                     out_of(gated, x1[0], x1[1], sum, r, gates[i][2]), out_of(gated, x1[2], x1[3], sum, r, gates[i][3])};
                    if (cg * 32 * NC + here < cols) *reinterpret_cast<u32x4*>(a.out + to[i]) = y;
                }
            }
            if (half == 0 && hh == 0) {
#pragma unroll
                for (int n = 0; n < NC; n++) {
                    const int col = (cg * NC + n) * 32 + c32;
                    if (col >= cols) continue;
                    const Column x = column(col);
                    if (!whole)
                        *reinterpret_cast<f32x2*>(a.ml + ((size_t)slot * COLS + col) * 2) = f32x2{m[n], l[n]};
                    else if (a.lse)
                        a.lse[(size_t)x.head * a.rows + row0 + x.token] = log_sum(m[n], l[n]);
                }
            }
        }
        if (parts > 0 && threadIdx.x == 0) a.cuts[block] = Cut{row0, ntok, head, block - parts + 1, parts};
        if (order == AT_FIRST) return;
        if (pos >= end) {
            if (order == STRAIGHT) return;
            order = AT_FIRST;
            pos = begin;
        }
        __syncthreads();  // the sums are read
        if (a.n <= 64) {
            mine = entry_of(a, lane_here());
            own_weight = weight_of(a, mine);
            upto = wave_scan(own_weight);
        } else {
            find_window(a);
        }
    }
}

// Joins the parts of the items that are cut, in the order of the stretches: a thread has four dims of a column, a block a
// few columns, one piece after another of all the pieces there are. The time is that of getting at the parts, so
// BATCH of them are asked for at once.
constexpr int JOIN_THREADS = 256, JOIN_A_CU = 8, BATCH = 4;
template <int DH>
__global__ void __launch_bounds__(JOIN_THREADS, JOIN_A_CU) attention_chunk_join_kernel(const Args a) {
    constexpr int COLS = Form<DH>::COLS, QUADS = DH / 4, MINE = JOIN_THREADS / QUADS, PIECES = COLS / MINE;
    __shared__ int list[JOIN_THREADS], counts[JOIN_THREADS / 64];
    const int tid = threadIdx.x, wave = tid >> 6;
    const int d = tid % QUADS * 4;
    for (int block0 = 0; block0 < a.blocks; block0 += JOIN_THREADS) {
        const bool cut_here = block0 + tid < a.blocks && a.cuts[block0 + tid].parts > 0;
        const uint64_t hits = __ballot(cut_here);
        if ((tid & 63) == 0) counts[wave] = __popcll(hits);
        __syncthreads();
        int at = __popcll(hits & ((uint64_t{1} << (tid & 63)) - 1)), all = 0;
        for (int w = 0; w < JOIN_THREADS / 64; w++) {
            if (w < wave) at += counts[w];
            all += counts[w];
        }
        if (cut_here) list[at] = block0 + tid;
        __syncthreads();
        for (int i = blockIdx.x; i < all * PIECES; i += gridDim.x) {
            const Cut cut = a.cuts[list[i / PIECES]];
            const int col = i % PIECES * MINE + tid / QUADS;
            if (col >= cut.tokens * a.G) continue;
            const int tk = a.over_G(col), head = cut.head * a.G + col - tk * a.G, row = cut.row0 + tk;
            const size_t to = ((size_t)row * a.Hq + head) * DH + d;
            const u32x2 gate = a.gate ? *reinterpret_cast<const u32x2*>(a.gate + to) : u32x2{0, 0};
            float top = -INFINITY, sum = 0.f;
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
            for (int k0 = 0; k0 < cut.parts; k0 += BATCH) {
                f32x4 v[BATCH];
                f32x2 ml[BATCH];
#pragma unroll
                for (int j = 0; j < BATCH; j++) {
                    const int k = min(k0 + j, cut.parts - 1);
                    const size_t slot = (size_t)(k == 0 ? 2 * cut.first + 1 : 2 * (cut.first + k)) * COLS + col;
                    ml[j] = *reinterpret_cast<const f32x2*>(a.ml + slot * 2);
                    v[j] = *reinterpret_cast<const f32x4*>(a.part + slot * DH + d);
                }
                float most = top;
#pragma unroll
                for (int j = 0; j < BATCH; j++) most = fmaxf(most, ml[j][0]);
                const float base = most == -INFINITY ? 0.f : most, keep = __builtin_amdgcn_exp2f(top - base);
                sum *= keep;
                o *= keep;
#pragma unroll
                for (int j = 0; j < BATCH; j++) {
                    if (k0 + j >= cut.parts) break;
                    const float f = __builtin_amdgcn_exp2f(ml[j][0] - base);
                    sum += ml[j][1] * f;
                    o += v[j] * f;
                }
                top = most;
            }
            const float inv = __builtin_amdgcn_rcpf(sum);
            *reinterpret_cast<u32x2*>(a.out + to) = u32x2{out_of(a.gate != nullptr, o[0], o[1], sum, inv, gate[0]),
                                                          out_of(a.gate != nullptr, o[2], o[3], sum, inv, gate[1])};
            if (a.lse && d == 0) a.lse[(size_t)head * a.rows + row] = log_sum(top, sum);
        }
        __syncthreads();
    }
}

template <int DH>
int launch(const Args& a, hipStream_t st) {
    attention_chunk_kernel<DH><<<a.blocks, THREADS, Form<DH>::BYTES, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    attention_chunk_join_kernel<DH><<<a.blocks * JOIN_A_CU, JOIN_THREADS, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace

bool chunk_configure() {
    auto set = [](const void* kernel, int bytes) {
        return hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess;
    };
    return set(reinterpret_cast<const void*>(attention_chunk_kernel<128>), Form<128>::BYTES) &&
           set(reinterpret_cast<const void*>(attention_chunk_kernel<256>), Form<256>::BYTES);
}
// [2 cus][a slot's columns] of sums, [2 cus][columns] of maxima and sums of weights, [cus] cuts
constexpr size_t PART = Form<256>::COLS * 256, ML = Form<128>::COLS * 2;
static_assert(Form<128>::COLS * 128 == PART, "the same room for both");
size_t chunk_bytes(int cus) { return 4 * 2 * cus * (PART + ML) + cus * sizeof(Cut); }

}  // namespace q35

using namespace q35;

extern "C" int cs1_attention_paged_varlen(void* paged, const void* q, const void* kp, const void* vp,
                                          const Cs1PageTable* pages, const int32_t* seqs, const int32_t* cu_seqlens, int n,
                                          int max_new, const void* gate, void* out, float* lse, int rows, int Hq, int Hk,
                                          int Dh, float scale, void* stream) {
    const Paged* const p = static_cast<const Paged*>(paged);
    if (!p || !table_ok(pages) || (Dh != 128 && Dh != 256) || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 || Hq / Hk > Form<256>::COLS)
        return hipErrorInvalidValue;
    if (n < 0 || n > MAX_LISTED || rows < 0 || max_new < 0 || !(scale >= 1e-30f && scale <= 1e30f)) return hipErrorInvalidValue;
    constexpr int64_t LIMIT = int64_t{1} << 31;
    if ((int64_t)rows * Hq > (1 << 24) || (int64_t)Hk * Dh > (1 << 24) || (int64_t)pages->npages * pages->page >= LIMIT)
        return hipErrorInvalidValue;
    if (rows == 0 || n == 0 || max_new == 0) return hipSuccess;
    if (!all_set({q, kp, vp, out, cu_seqlens}) || !on16(q) || !on16(kp) || !on16(vp) || !on16(out) || !on16(gate))
        return hipErrorInvalidValue;
    int device;
    if (hipGetDevice(&device) != hipSuccess || device != p->device) return hipErrorInvalidDevice;
    // Entries of up to 16 columns are each one tile of the kernel for single tokens, where others may be, in a launch before
    // theirs: 43 entries of 1 to 4 tokens behind up to 4096 (16/4 heads of 256) take 80 us so and 82 in the tiles here,
    // one of 4 behind 700 (heads of 128) 12.3 and 19.8, 29 of a token beside a prompt's 1021 94 and 99. One entry that may
    // be longer is taken for longer.
    const int64_t pairs = (int64_t)n * Hk;
    const bool all_few = max_new <= FEW / (Hq / Hk);
    Args a;
    a.others = 0;
    if ((all_few || (n > 1 && Hq / Hk <= FEW)) && pairs <= 1 << 22 &&
        pairs * ((int64_t)pages->max_pages * pages->page / 32 + 1) < LIMIT) {
        const Call c{q, kp, vp, pages, seqs, gate, out, lse, n, Hq, Hk, Dh, scale};
        const int e = paged_rows(p, c, cu_seqlens, max_new, rows, stream);
        if (e != hipSuccess || all_few) return e;
        a.others = FEW / (Hq / Hk);
    }
    a.q = static_cast<const bf16*>(q);
    a.kp = static_cast<const bf16*>(kp);
    a.vp = static_cast<const bf16*>(vp);
    a.gate = static_cast<const bf16*>(gate);
    a.out = static_cast<bf16*>(out);
    a.lse = lse;
    a.part = p->chunk;
    a.ml = p->chunk + 2 * p->cus * PART;
    a.cuts = reinterpret_cast<Cut*>(a.ml + 2 * p->cus * ML);
    a.table = pages->table;
    a.lens = pages->lens;
    a.seqs = seqs;
    a.cu = cu_seqlens;
    a.nseq = pages->nseq;
    a.max_pages = pages->max_pages;
    a.npages = pages->npages;
    a.page = pages->page;
    a.n = n;
    a.max_new = max_new;
    a.rows = rows;
    a.Hq = Hq;
    a.Hk = Hk;
    a.G = Hq / Hk;
    a.tokens = (Dh == 128 ? Form<128>::COLS : Form<256>::COLS) / a.G;
    a.blocks = p->cus;
    // What an item takes around its steps counts as 256 keys (four units), and no stretch is shorter than three units: a prompt's
    // 1021 rows beside 29 tokens (16/4 heads of 128) take 94.2 us so, 96.8, 95.2 and 94.6 with 128, 192 and 320 keys, 333 behind
    // 936 (256) 35.2, and 36.3, 35.9 and 37.1; 20 behind 300 20.3, and 22.8 and 24.3 with stretches of at least 256 and 384.
    a.pad = 256;
    a.least = 192;
    a.tokens_inverse = (uint32_t)(((uint64_t{1} << 32) + a.tokens - 1) / a.tokens);
    a.G_inverse = (65536 + a.G - 1) / a.G;
    a.blocks_inverse = 1.0 / a.blocks;
    a.page_inverse = (uint32_t)std::min<uint64_t>(0xffffffffu, (uint64_t{1} << 32) / (a.page / 16));
    a.scale_log2 = scale * LOG2E;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return Dh == 128 ? launch<128>(a, st) : launch<256>(a, st);
}
