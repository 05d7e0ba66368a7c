// Attention of several new tokens a sequence over the paged cache (cs1_attention_paged_varlen).  Row j of an entry of L
// rows, whose sequence holds n tokens, is at position p = n - L + j and sees the keys 0 .. p:
//
//   S_i = scale q . k_i,  m = max S_i,  l = sum exp(S_i - m),  out = sigmoid(gate) (sum exp(S_i - m) v_i) / l,
//   lse = m + log l.
//
// Work: an item is up to COLS columns, the q heads of one kv head at some of an entry's rows, with all keys that
// they see: however many q heads share a kv head, they share its keys too.  All items of a launch form one line, measured in
// keys, that is cut into equal stretches, one a block: a prompt's part on its own, drafts of a few tokens behind
// long texts and single tokens share the chip alike, and only the device knows the lengths.  What a stretch has of an
// item that others have parts of goes to memory, and a second launch joins the parts in order.
//
// A block has eight waves: four groups of 32 columns, two halves of the keys of each unit (64 keys with heads of 256, 128 with
// heads of 128: 32 KiB of K and of V).  S^T = K Q^T and O^T += V^T P^T on the 32x32x16 MFMA: what the first leaves in a
// lane is what the second wants, so probabilities stay in registers.  Units move from the pages into LDS without
// registers, K two ahead and V one ahead; a wave's piece of a unit lies in one run of 16 tokens, which no page divides.
// The halves' waves that share a SIMD take turns: one multiplies while the other has its exponentials (priority to the
// first half).  At the end the halves are joined through LDS.
//
// P is rounded to bfloat16 for the second product, as in the prefill: the matrix cores set the time here, and a second part of
// P would cost half as much again.  Sums and maxima are float32; out is rounded once, after the gate.
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
using tile32::read_tr;
using tile32::v_slot;

constexpr int THREADS = 512, WAVES = 8, COLS = CHUNK_COLS;
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
    uint32_t page_inverse;  // 2^32 over page / 16, rounded down
    float scale_log2;
};

template <int DH>
struct Form {
    static constexpr int UNIT = DH == 256 ? 64 : 128;  // keys
    static constexpr int SUB = UNIT / 64;              // pieces of 32 keys of a wave's half
    static constexpr int KS = DH / 16, DT = DH / 32;   // products along a head, and tiles of 32 of its dims
    static constexpr int ROW = 2 * DH, TILE = UNIT * ROW;
    static constexpr int KST = 3, VST = 2;             // LDS stages
    static constexpr int BYTES = (KST + VST) * TILE;   // all of the LDS
    static constexpr int XS = DT / 2 * 16 + 4;         // floats a lane of the exchange
    static_assert(THREADS * XS * 4 <= BYTES && BYTES <= 160 * 1024, "the exchange fits in the stages");
};

// An entry's sequence, first row, rows, and the position of the first one (less than 0: rows without keys).
struct Entry {
    int s, row0, rows, pos;
};
__device__ __forceinline__ Entry entry_of(const Args& a, int i) {
    Entry e{-1, 0, 0, 0};
    if (i >= a.n) return e;
    const int lo = a.cu[i], hi = a.cu[i + 1];
    if (lo < 0 || hi <= lo || lo >= a.rows) return e;
    e.s = listed_seq(a.seqs, i, a.nseq);
    e.row0 = lo;
    e.rows = min(min(hi, a.rows) - lo, a.max_new);
    const int64_t held = e.s < 0 ? 0 : min((int64_t)max(a.lens[e.s], 0), (int64_t)a.max_pages * a.page);
    e.pos = (int)(held - (hi - lo));
    return e;
}

// The line: `c` items of an entry for one kv head, tokens (c + 1) keys and the pad more than those before its rows
__device__ __forceinline__ int64_t line_of(const Args& a, int pos, int64_t c) {
    return c * (max(pos, 0) + a.pad) + a.tokens * (c * (c + 1) / 2);
}
__device__ __forceinline__ int items_of(const Args& a, int rows) { return (rows + a.tokens - 1) / (uint32_t)a.tokens; }

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
// Sum over this lane and those below.
__device__ __forceinline__ int64_t wave_scan(int64_t x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int lo = __shfl_up((int)x, o, 64), hi = __shfl_up((int)(x >> 32), o, 64);
        if ((int)(threadIdx.x & 63) >= o) x += (int64_t)(uint32_t)lo | (int64_t)hi << 32;
    }
    return x;
}

// Of two bfloat16 values: is one no finite number; those that are; and 1 for each that is an infinity of this sign or a NaN.
__device__ __forceinline__ bool odd16(uint32_t x) {
    return ((x & 0x7f80u) == 0x7f80u) | ((x & 0x7f800000u) == 0x7f800000u);
}
__device__ __forceinline__ uint32_t common16(uint32_t x) {
    return ((x & 0x7f80u) == 0x7f80u ? 0u : x & 0xffffu) | ((x & 0x7f800000u) == 0x7f800000u ? 0u : x & 0xffff0000u);
}
__device__ __forceinline__ uint32_t ones16(uint32_t x, uint32_t sign) {
    auto one = [&](uint32_t v) { return (v & 0x7f80u) == 0x7f80u && ((v & 0x7fu) != 0 || (v & 0x8000u) == sign); };
    return (one(x & 0xffffu) ? 0x3f80u : 0u) | (one(x >> 16) ? 0x3f800000u : 0u);
}

// Four dims of an output from sums o over l (0: no key).
__device__ __forceinline__ void store_out(const Args& a, size_t at, const f32x4& o, float l) {
    const float inv = l != 0.f ? 1.f / l : 0.f;
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = l != 0.f ? o[e] * inv : 0.f;
    if (a.gate) {
        const u32x2 g = *reinterpret_cast<const u32x2*>(a.gate + at);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (l != 0.f) y[e] *= sigmoid(e & 1 ? hi_f32(g[e / 2]) : lo_f32(g[e / 2]));
    }
    *reinterpret_cast<u32x2*>(a.out + at) = u32x2{pack2(y[0], y[1]), pack2(y[2], y[3])};
}
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * LN2; }

template <int DH>
__global__ void __launch_bounds__(THREADS, 1) attention_chunk_kernel(const Args a) {
    using F = Form<DH>;
    constexpr int UNIT = F::UNIT, SUB = F::SUB, KS = F::KS, DT = F::DT, ROW = F::ROW, TILE = F::TILE, KST = F::KST;
    extern __shared__ __align__(16) unsigned char smem[];
    const int wave = uniform(threadIdx.x >> 6);
    const int cg = wave & 3, kg = wave >> 2;  // group of columns, half of the keys
    if (kg == 0) __builtin_amdgcn_s_setprio(1);

    // The line's length, from the sums of windows of 64 entries; lane i has windows 2 i and 2 i + 1.
    const int windows = (a.n + 63) / 64;
    auto weight_of = [&](const Entry& e) { return line_of(a, e.pos, items_of(a, e.rows)) * a.Hk; };
    int64_t w0, w1, upto;
    {
        const int lane = lane_here();
        int64_t* const sums = reinterpret_cast<int64_t*>(smem);
        for (int w = wave; w < windows; w += WAVES) {
            const int64_t all = wave_scan(weight_of(entry_of(a, w * 64 + lane)));
            if (lane == 63) sums[w] = all;
        }
        __syncthreads();
        w0 = 2 * lane < windows ? sums[2 * lane] : 0;
        w1 = 2 * lane + 1 < windows ? sums[2 * lane + 1] : 0;
        __syncthreads();
        upto = wave_scan(w0 + w1);
    }
    const int64_t total = scalar64(upto, 63);
    const int64_t each = max((total + a.blocks - 1) / a.blocks, (int64_t)a.least);
    // neighbours of the line, which share keys, are on one XCD
    const int block = a.blocks % 8 == 0 ? (blockIdx.x & 7) * (a.blocks / 8) + (blockIdx.x >> 3) : blockIdx.x;
    const int64_t begin = block * each, end = min(total, begin + each);
    if (threadIdx.x == 0) a.cuts[block].parts = 0;
    if (begin >= end) return;

    constexpr int MINE = UNIT / WAVES, PER = 1024 / ROW, NI = MINE / PER, CHUNKS = ROW / 16;  // rows of a wave's transfers
    const int token = 2 * a.Hk * DH;  // bytes
    const int r0 = wave * MINE;
    const uint32_t lds0 = (uint32_t)uniform((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem) +
                          r0 * ROW;
    const int half_at = kg * (UNIT / 2) * ROW;

    // What is looked at once an item lies in memory in between: the loop over the keys needs the registers.
    volatile int64_t kept[4];
    kept[0] = w0;
    kept[1] = w1;
    kept[2] = upto;
    for (int64_t pos = begin; pos < end;) {
        const int lane = lane_here(), c32 = lane & 31, hh = lane >> 5;
        // the item at `pos`
        const int64_t windows_upto = kept[2], window0 = kept[0], window1 = kept[1];
        const int l0 = __ffsll((unsigned long long)__ballot(windows_upto > pos)) - 1;
        const int64_t first0 = scalar64(window0, l0), before0 = scalar64(windows_upto, l0) - first0 - scalar64(window1, l0);
        const bool second = pos >= before0 + first0;
        const int64_t window_at = second ? before0 + first0 : before0;
        const Entry mine = entry_of(a, (2 * l0 + second) * 64 + lane);
        const int64_t entry_own = weight_of(mine), entry_upto = wave_scan(entry_own);
        const int el = __ffsll((unsigned long long)__ballot(window_at + entry_upto > pos)) - 1;
        const int seq = scalar(mine.s, el), erow = scalar(mine.row0, el), erows = scalar(mine.rows, el);
        const int epos = scalar(mine.pos, el), items = items_of(a, erows);
        const int64_t own = line_of(a, epos, items);
        const int64_t estart = window_at + scalar64(entry_upto - entry_own, el);
        const int head = (int)((uint64_t)(pos - estart) / (uint64_t)own);
        const int64_t hstart = estart + head * own;
        int c = 0;  // the last item that begins at or before pos
        for (int up = items - 1; c < up;) {
            const int mid = (c + up + 1) >> 1;
            if (hstart + line_of(a, epos, mid) <= pos)
                c = mid;
            else
                up = mid - 1;
        }
        const int64_t istart = hstart + line_of(a, epos, c), iend = hstart + line_of(a, epos, c + 1);
        const int tok0 = c * a.tokens, ntok = min(a.tokens, erows - tok0);
        const int row0 = erow + tok0, pos0 = epos + tok0;  // of its first row
        const int keys = max(pos0 + ntok, 0), units = (keys + UNIT - 1) / UNIT;
        auto cut = [&](int64_t x) {
            return x <= istart ? 0 : x >= iend ? units : (int)min((int64_t)units, max(x - istart - a.pad, (int64_t)0) / UNIT);
        };
        const int u0 = uniform(cut(begin)), u1 = uniform(cut(end));
        const bool whole = istart >= begin && iend <= end;
        pos = min(iend, end);

        // this lane's column: a row and a q head of the kv head's
        const int cols = ntok * a.G, col = cg * 32 + c32, tk = col / (uint32_t)a.G;
        const bool used = col < cols;
        const int head0 = head * a.G;
        const size_t at_q = ((size_t)(row0 + (used ? tk : 0)) * a.Hq + head0 + (used ? col - tk * a.G : 0)) * DH;
        const int last_key = used ? pos0 + tk : -1;
        const bool active = cg * 32 < cols;
        const int low_key = pos0 + cg * 32 / (uint32_t)a.G, high_key = pos0 + min(ntok - 1, (cg * 32 + 31) / (uint32_t)a.G);

        u32x4 qf[KS];
#pragma unroll
        for (int i = 0; i < KS; i++) {
            qf[i] = u32x4{0, 0, 0, 0};
            if (used) qf[i] = *reinterpret_cast<const u32x4*>(a.q + at_q + 16 * i + 8 * hh);
        }

        // The next 64 runs of 16 tokens: lane i has the pool's run of run number runs0 + i, -1 if its page is out of range
        constexpr int RUNS = UNIT / 16, AHEAD = 64 / RUNS;
        int where = 0, from_unit = -AHEAD;
        uint64_t bad = 0;
        auto look_up = [&](int unit) {
            from_unit = unit;
            const uint32_t run = unit * RUNS + lane, page = (uint32_t)a.page / 16;
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
        struct Piece {
            int run, rows;      // of the pool; rows that are there, of the wave's
            uint32_t bad;       // runs of the unit whose page is out of range
        };
        auto piece_of = [&](int unit) {
            Piece p{0, 0, 0};
            if (unit >= u1) return p;
            if (unit >= from_unit + AHEAD) look_up(unit);
            const int i = (unit - from_unit) * RUNS;
            p.run = scalar(where, i + r0 / 16);
            p.rows = p.run < 0 ? 0 : max(0, min(MINE, keys - unit * UNIT - r0));
            p.bad = (uint32_t)(bad >> i) & ((1u << RUNS) - 1);
            return p;
        };
        auto move = [&](const bf16* pool, const Piece& p, uint32_t to, auto chunk) {
            const uint64_t at = reinterpret_cast<uint64_t>(pool) +
                                ((uint64_t)(uint32_t)max(p.run, 0) * 16 + r0 % 16) * (uint32_t)token + (uint32_t)(head * ROW);
            const u32x4 r = {(uint32_t)uniform((int)(uint32_t)at), (uint32_t)uniform((int)(uint32_t)(at >> 32)) & 0xffffu,
                             (uint32_t)uniform(p.rows > 0 ? (p.rows - 1) * token + ROW : 0), 0x00020000u};
            // lane l fills place l % CHUNKS of row l / CHUNKS with the chunk that belongs there
            const int lane = lane_here(), row = lane / CHUNKS, place = lane % CHUNKS;
#pragma unroll
            for (int i = 0; i < NI; i++)
                dma16(r, (uint32_t)uniform((int)(to + i * 1024)), row * token + (chunk(i * PER + row, place) << 4),
                      uniform(i * PER * token));
        };
        auto move_k = [&](const Piece& p, int stage) {
            move(a.kp, p, lds0 + stage * TILE, [&](int r, int c) { return k_slot(r0 + r, c); });
        };
        auto move_v = [&](const Piece& p, int stage) {
            move(a.vp, p, lds0 + (KST + stage) * TILE, [&](int r, int c) { return v_slot(r, c); });
        };

        f32x16 o[DT];
#pragma unroll
        for (int t = 0; t < DT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[t][i] = 0.f;
        float m = -INFINITY, l = 0.f;

        Piece now = piece_of(u0), next = piece_of(u0 + 1);
        if (u0 < u1) {
            move_k(now, 0);
            move_v(now, 0);
            move_k(next, 1);
        }
#pragma unroll
        for (int i = 0; i < KS; i++) asm volatile("" ::"v"(qf[i]));
        wait_vm_all();
        __syncthreads();

        int ks = 0, vs = 0;
        for (int u = u0; u < u1; u++) {
            const Piece after = piece_of(u + 2);
            move_v(next, vs ^ 1);
            move_k(after, ks == 0 ? 2 : ks - 1);
            const int k0 = u * UNIT + kg * (UNIT / 2);  // this wave's first key
            if (active && k0 <= high_key) {
                const unsigned char *kb = smem + ks * TILE + half_at, *vb = smem + (KST + vs) * TILE + half_at;
                f32x16 s[SUB];
#pragma unroll
                for (int sub = 0; sub < SUB; sub++)
#pragma unroll
                    for (int i = 0; i < 16; i++) s[sub][i] = 0.f;
                // K: row c32 of a piece, chunk 2 i + hh, K_AHEAD products ahead
                constexpr int K_AHEAD = 3;
                u32x4 kf[KS * SUB];
                auto read_k = [&](int j) {
                    const int sub = j / KS, i = j % KS;
                    kf[j] = *reinterpret_cast<const u32x4*>(kb + (32 * sub + c32) * ROW + (k_slot(c32, 2 * i + hh) << 4));
                };
#pragma unroll
                for (int j = 0; j < K_AHEAD; j++) read_k(j);
#pragma unroll
                for (int j = 0; j < KS * SUB; j++) {
                    if (j + K_AHEAD < KS * SUB) read_k(j + K_AHEAD);
                    s[j / KS] = mfma32(kf[j], qf[j % KS], s[j / KS]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                // s[sub][i] is key k0 + 32 sub + 8 (i / 4) + 4 hh + i % 4
                const uint32_t lost = now.bad >> (kg * RUNS / 2) & ((1u << RUNS / 2) - 1);
                const bool masked = k0 + UNIT / 2 - 1 > low_key || lost != 0;
                if (masked) {
#pragma unroll
                    for (int sub = 0; sub < SUB; sub++)
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const int key = 32 * sub + 8 * (i >> 2) + 4 * hh + (i & 3);
                            if (k0 + key > last_key || (lost >> (2 * sub + (i >> 3)) & 1)) s[sub][i] = -INFINITY;
                        }
                }
                float top = s[0][0];
#pragma unroll
                for (int i = 1; i < 16 * SUB; i++) top = fmaxf(top, s[i >> 4][i & 15]);
                top = max_halves(top) * a.scale_log2;
                if (!__all(top <= m + SLACK)) {
                    const float to = fmaxf(m, top), by = __builtin_amdgcn_exp2f(m - (to == -INFINITY ? 0.f : to));
                    m = to;
                    l *= by;
#pragma unroll
                    for (int t = 0; t < DT; t++) o[t] *= by;
                }
                const float base = m == -INFINITY ? 0.f : m;
                // P^T of keys 16 j ..: what a lane has is what it holds of the operand, in the order of v_at's rows
                u32x4 pf[2 * SUB];
#pragma unroll
                for (int sub = 0; sub < SUB; sub++) {
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        s[sub][i] = __builtin_amdgcn_exp2f(fmaf(s[sub][i], a.scale_log2, -base));
                        l += s[sub][i];
                    }
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        pf[2 * sub + j] = u32x4{pack2(s[sub][8 * j], s[sub][8 * j + 1]), pack2(s[sub][8 * j + 2], s[sub][8 * j + 3]),
                                                pack2(s[sub][8 * j + 4], s[sub][8 * j + 5]), pack2(s[sub][8 * j + 6], s[sub][8 * j + 7])};
                }
                // V^T as the transposing read hands it out: of tile t of the dims, keys 16 j ..
                u32x4 v[DT][2 * SUB];
                const int gi = lane & 15, gg = lane >> 4, vrow = 4 * (gg >> 1) + (gi >> 2), vdim = 16 * (gg & 1) + 4 * (gi & 3);
                auto read_v = [&](int t) {
                    const unsigned char* const at = vb + vrow * ROW + (v_slot(vrow, (32 * t + vdim) >> 3) << 4) + 2 * (vdim & 7);
#pragma unroll
                    for (int j = 0; j < 2 * SUB; j++) {
                        const u32x2 lo = read_tr(at + 16 * j * ROW), hi = read_tr(at + (16 * j + 8) * ROW);
                        v[t][j] = u32x4{lo[0], lo[1], hi[0], hi[1]};
                    }
                };
                bool odd = false;
                if (masked) {
                    // A value that some of the columns must not see may be an infinity or NaN, which a weight of zero does
                    // not take away.
                    u32x4 x[4];
                    for (int i = 0; i < UNIT / 2 * ROW / 4096; i++) {
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            x[j] = *reinterpret_cast<const u32x4*>(vb + (4 * i + j) * 1024 + lane * 16);
#pragma unroll
                        for (int j = 0; j < 4; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++) odd |= odd16(x[j][e]);
                    }
                    odd = __any(odd);
                }
                read_v(0);
#pragma unroll
                for (int t = 0; t < DT; t++) {
                    if (t + 1 < DT) read_v(t + 1);
                    if (odd) {  // such values leave the product
#pragma unroll
                        for (int j = 0; j < 2 * SUB; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++) v[t][j][e] = common16(v[t][j][e]);
                    }
#pragma unroll
                    for (int j = 0; j < 2 * SUB; j++) o[t] = mfma32(v[t][j], pf[j], o[t]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (odd) {
                    // and the columns that see them are told so by products of whole numbers: how many +inf (and NaN) are there,
                    // and how many -inf (and NaN)
#pragma unroll
                    for (int j = 0; j < 2 * SUB; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int key = 16 * j + 8 * (e >> 1) + 4 * hh + 2 * (e & 1);
                            const bool gone = lost >> j & 1;
                            pf[j][e] = (!gone && k0 + key <= last_key ? 0x3f80u : 0u) |
                                       (!gone && k0 + key + 1 <= last_key ? 0x3f800000u : 0u);
                        }
                    auto tell = [&](int t, uint32_t sign, float what) {
                        f32x16 found;
#pragma unroll
                        for (int i = 0; i < 16; i++) found[i] = 0.f;
                        read_v(t);
#pragma unroll
                        for (int j = 0; j < 2 * SUB; j++) {
#pragma unroll
                            for (int e = 0; e < 4; e++) v[t][j][e] = ones16(v[t][j][e], sign);
                            found = mfma32(v[t][j], pf[j], found);
                        }
#pragma unroll
                        for (int i = 0; i < 16; i++) o[t][i] += found[i] > 0.f ? what : 0.f;
                        __builtin_amdgcn_sched_barrier(0);
                    };
#pragma unroll
                    for (int t = 0; t < DT; t++) {
                        tell(t, 0, INFINITY);
                        tell(t, 0x8000u, -INFINITY);
                    }
                }
            }
            now = next;
            next = after;
            ks = ks == 2 ? 0 : ks + 1;
            vs ^= 1;
            __builtin_amdgcn_s_waitcnt(0x0f70 | NI);  // all but the K just asked for
            __syncthreads();
        }
        wait_vm_all();  // (transfers of nothing, behind the last unit)
        __syncthreads();

        // The halves of the keys: each wave hands over the sums of the dims that the other one ends, half of them, and puts
        // its results where it found the other's.  (What follows is one loop's code and not one for each register: code that runs
        // once comes from memory.)
        constexpr int J = DT * 2;  // quads of dims that a lane ends
        float* const mine_at = reinterpret_cast<float*>(smem) + (wave * 64 + lane) * F::XS;
        f32x4* const from = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(smem) + ((wave ^ 4) * 64 + lane) * F::XS);
        auto hand_over = [&](auto which) {
            constexpr int K = decltype(which)::value;
            f32x4* const to = reinterpret_cast<f32x4*>(mine_at);
#pragma unroll
            for (int j = 0; j < J; j++) {
                const f32x16& x = o[(1 - K) * (DT / 2) + j / 4];
                to[j] = f32x4{x[4 * (j % 4)], x[4 * (j % 4) + 1], x[4 * (j % 4) + 2], x[4 * (j % 4) + 3]};
            }
            to[J] = f32x4{m, l, 0.f, 0.f};
        };
        float top, sum;
        auto join = [&](auto which) {
            constexpr int K = decltype(which)::value;
            const f32x4 theirs = from[J];
            const float m0 = K == 0 ? m : theirs[0], m1 = K == 0 ? theirs[0] : m;
            const float l0 = K == 0 ? l : theirs[1], l1 = K == 0 ? theirs[1] : l;
            top = fmaxf(m0, m1);
            const float base = top == -INFINITY ? 0.f : top;
            const float f0 = __builtin_amdgcn_exp2f(m0 - base), f1 = __builtin_amdgcn_exp2f(m1 - base);
            sum = l0 * f0 + l1 * f1;
#pragma unroll
            for (int j = 0; j < J; j++) {
                f32x4 x = from[j];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float own = o[K * (DT / 2) + j / 4][4 * (j % 4) + e];
                    x[e] = (K == 0 ? own : x[e]) * f0 + (K == 0 ? x[e] : own) * f1;
                }
                from[j] = x;
            }
        };
        kg == 0 ? hand_over(std::integral_constant<int, 0>{}) : hand_over(std::integral_constant<int, 1>{});
        __syncthreads();
        kg == 0 ? join(std::integral_constant<int, 0>{}) : join(std::integral_constant<int, 1>{});
        sum += __shfl_xor(sum, 32, 64);
        const int slot = 2 * block + (istart >= begin);
        if (active) {
            float* const part = a.part + (size_t)slot * (COLS * DH);
            for (int j = 0; j < J; j++) {
                if (!whole)
                    *reinterpret_cast<f32x4*>(part + ((wave * J + j) * 64 + lane) * 4) = from[j];
                else if (used)
                    store_out(a, at_q + kg * (DH / 2) + 32 * (j / 4) + 8 * (j % 4) + 4 * hh, from[j], sum);
            }
            if (kg == 0 && hh == 0) {
                if (!whole)
                    *reinterpret_cast<f32x2*>(a.ml + ((size_t)slot * COLS + col) * 2) = f32x2{top, sum};
                else if (used && a.lse)
                    a.lse[(size_t)(at_q / DH % a.Hq) * a.rows + row0 + tk] = log_sum(top, sum);
            }
        }
        if (!whole && iend <= end && threadIdx.x == 0) {
            const int first = (int)((uint64_t)istart / (uint64_t)each);
            a.cuts[block] = Cut{row0, ntok, head, first, block - first + 1};
        }
        __syncthreads();  // the exchange is read
    }
}

// Joins the parts of the item that stretch blockIdx.x ended, in the order of the stretches: block y has what wave y of each
// part's block left.
template <int DH>
__global__ void __launch_bounds__(256) attention_chunk_join_kernel(const Args a) {
    constexpr int J = DH / 16, QUADS = J / 4;  // a wave's quads of dims a lane, and a thread's of them
    const Cut cut = a.cuts[blockIdx.x];
    const int wave = blockIdx.y, cg = wave & 3, kg = wave >> 2;
    const int lane = threadIdx.x & 63, j0 = (threadIdx.x >> 6) * QUADS;
    const int col = cg * 32 + (lane & 31), hh = lane >> 5;
    if (cut.parts == 0 || cg * 32 >= cut.tokens * a.G) return;
    auto slot_of = [&](int k) { return k == 0 ? 2 * cut.first + 1 : 2 * (cut.first + k); };
    auto ml_of = [&](int k) { return *reinterpret_cast<const f32x2*>(a.ml + ((size_t)slot_of(k) * COLS + col) * 2); };
    float top = -INFINITY, sum = 0.f;
    for (int k = 0; k < cut.parts; k++) top = fmaxf(top, ml_of(k)[0]);
    const float base = top == -INFINITY ? 0.f : top;
    f32x4 o[QUADS];
#pragma unroll
    for (int j = 0; j < QUADS; j++) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < cut.parts; k++) {
        const f32x2 ml = ml_of(k);
        const float f = __builtin_amdgcn_exp2f(ml[0] - base);
        const float* const part = a.part + (size_t)slot_of(k) * (COLS * DH);
        sum += ml[1] * f;
#pragma unroll
        for (int j = 0; j < QUADS; j++)
            o[j] += *reinterpret_cast<const f32x4*>(part + ((wave * J + j0 + j) * 64 + lane) * 4) * f;
    }
    if (col >= cut.tokens * a.G) return;
    const int tk = col / (uint32_t)a.G, head = cut.head * a.G + col - tk * a.G, row = cut.row0 + tk;
    const size_t at = ((size_t)row * a.Hq + head) * DH + kg * (DH / 2) + 4 * hh;
#pragma unroll
    for (int j = 0; j < QUADS; j++) store_out(a, at + 32 * ((j0 + j) / 4) + 8 * ((j0 + j) % 4), o[j], sum);
    if (a.lse && wave < 4 && j0 == 0 && hh == 0) a.lse[(size_t)head * a.rows + row] = log_sum(top, sum);
}

template <int DH>
int launch(const Args& a, hipStream_t st) {
    attention_chunk_kernel<DH><<<a.blocks, THREADS, Form<DH>::BYTES, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    attention_chunk_join_kernel<DH><<<dim3(a.blocks, WAVES), 256, 0, st>>>(a);
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
size_t chunk_bytes(int cus) { return (size_t)2 * cus * 4 * COLS * (256 + 2) + (size_t)cus * sizeof(Cut); }

}  // namespace q35

using namespace q35;

extern "C" int cs1_attention_paged_varlen(void* paged, const void* q, const void* kp, const void* vp,
                                          const Cs1PageTable* pages, const int32_t* seqs, const int32_t* cu_seqlens, int n,
                                          int max_new, const void* gate, void* out, float* lse, int rows, int Hq, int Hk,
                                          int Dh, float scale, void* stream) {
    const Paged* const p = static_cast<const Paged*>(paged);
    if (!p || !table_ok(pages) || (Dh != 128 && Dh != 256) || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 || Hq / Hk > COLS)
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
    Args a;
    a.q = static_cast<const bf16*>(q);
    a.kp = static_cast<const bf16*>(kp);
    a.vp = static_cast<const bf16*>(vp);
    a.gate = static_cast<const bf16*>(gate);
    a.out = static_cast<bf16*>(out);
    a.lse = lse;
    a.part = p->chunk;
    a.ml = p->chunk + (size_t)2 * p->cus * COLS * 256;
    a.cuts = reinterpret_cast<Cut*>(a.ml + (size_t)2 * p->cus * COLS * 2);
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
    a.tokens = COLS / a.G;
    a.blocks = p->cus;
    a.pad = 128;
    a.least = 256;
    a.page_inverse = (uint32_t)std::min<uint64_t>(0xffffffffu, (uint64_t{1} << 32) / (a.page / 16));
    a.scale_log2 = scale * LOG2E;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return Dh == 128 ? launch<128>(a, st) : launch<256>(a, st);
}
