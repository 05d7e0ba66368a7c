// Attention of one new token per row over a paged key-value cache (cs1_attention_paged).  For a row of
// sequence s with n = lens[s] keys and q head h on kv head h / (Hq / Hk):
//
//   S_j = scale q . k_j,  m = max S_j,  l = sum exp(S_j - m),  out = sigmoid(gate) (sum exp(S_j - m) v_j) / l,
//   lse = m + log l.
//
// The keys and values are read once and nothing else is of size, so the rate of that stream is the bound.
//
// Work: a row and kv head's keys in units of 32, shares of consecutive units to blocks (plan_share below); the q
// heads of a kv head are the rows of one matrix tile, up to 16 of them (more take several tiles, which read
// the keys again).  A block's four waves take every fourth unit, each with a running maximum and sum of its own, and join
// through LDS; the shares of a sequence that has several are joined by the last of them to end.
//
// A unit in registers, without LDS: S^T = K Q^T takes K rows as they lie (lane l: key l % 16, 8 dims a load) and leaves
// lane l with q head l % 16 and keys 4 (l / 16) .. + 3 of each 16; that is the layout in which O^T = V^T P^T wants P^T,
// with the unit's keys in the order (i < 4: 4 g + i, else 16 + 4 g + i - 4) for lane group g.  V rows are loaded 16
// lanes x 16 bytes at a time (256 bytes in a row), lane l holding dims 8 (l % 16) .. + 7 of its group's eight
// keys, and two-byte permutes make columns of eight keys of them: the tile's row m is dim 8 m + j.  Each q head stays
// in its lanes from the scores to the output, so maximum and sum need no exchange but between lane groups,
// and that only when the maximum rises by more than RISE or at the end.  The next unit's K is on its way while this one's
// probabilities are formed, its V while the next scores are.
//
// P goes to the product in two bfloat16 parts (hi cut off, lo the rounded rest: p to 2^-15): the matrix cores wait for
// memory here, and the second product leaves the rounding of out the only one that counts.  lo is never zero (LEAST), so
// that an infinite v gives the infinity that it should and not inf + 0 inf.
#include <algorithm>
#include <new>
#include <type_traits>

#include "common.h"
#include "paged.h"

namespace q35 {
namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int UNIT = 32, ROWS = 16;
constexpr int LEAST_SHARE = 4;               // units
constexpr int GROUP = 16, GROUPS_MAX = 64;   // shares that one block joins, groups of a sequence
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LEAST = 0x1p-126f;  // bfloat16's smallest normal value
constexpr float RISE = 6.f;  // in powers of two: P stays under 2^6, far from where float32 sums lose anything

struct Paged {
    int device, cus, target;
    float* part;  // [2 target, ROWS, 256] partial sums, [2 target, ROWS, 2] maximum and sum
    int* count;   // [2 target] shares of a group, [2 target] groups of a sequence that are done
};

struct Args {
    const bf16 *q, *kp, *vp, *gate;
    bf16* out;
    float *lse, *part, *ml;
    int* count;
    const int32_t *table, *lens, *seqs;
    int nseq, max_pages, npages, page, B, Hq, Hk, G, tiles, target;
    float scale_log2;
};

// Keys of row r (0 for padding).
__device__ __forceinline__ int keys_of(const Args& a, int r) {
    if (r >= a.B) return 0;
    const int s = listed_seq(a.seqs, r, a.nseq);
    return s < 0 ? 0 : (int)min((int64_t)max(a.lens[s], 0), (int64_t)a.max_pages * a.page);
}

__device__ __forceinline__ int units_of(int n) { return n / UNIT + (n % UNIT != 0); }

template <typename T>
__device__ __forceinline__ T wave_scan(T x) {  // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T below = __shfl_up(x, o, 64);
        if (lane >= o) x += below;
    }
    return x;
}

// Lane i's value, one for the wave.
__device__ __forceinline__ int scalar(int x, int i) { return __builtin_amdgcn_readlane(x, i); }

// The units of a share: all sequences' units over the number of shares that fill the chip, at least one
// for each wave.  Each wave works it out from the lengths, which only the device knows (n0: row lane's).
__device__ __forceinline__ int units_per_share(const Args& a, int n0) {
    int64_t total = 0;
    for (int r0 = 0; r0 < a.B; r0 += 64) {
        int64_t u = units_of(r0 == 0 ? n0 : keys_of(a, r0 + (threadIdx.x & 63)));
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) u += __shfl_xor(u, o, 64);
        total += (int64_t)((uint64_t)(uint32_t)scalar((int)(u >> 32), 0) << 32 | (uint32_t)scalar((int)u, 0));
    }
    total *= a.Hk * a.tiles;
    return (int)max((int64_t)LEAST_SHARE, (total + a.target - 1) / a.target);
}

struct Share {
    int row, split, splits, head, tile, n, slot;  // slot: of the first split's partial results
};

// Share number idx: rows in order, a row's splits, and in each the kv heads and tiles.  Rows without keys
// have one share (it writes their zeros).  Slots count the shares of rows that have several: with u units and
// p units a share that is ceil(u / p) < 2 u / p of them, so all slots are fewer than twice the target.
__device__ __forceinline__ bool find_share(const Args& a, int idx, int n0, Share& sh) {
    const int per = units_per_share(a, n0);
    const int lane = threadIdx.x & 63, each = a.Hk * a.tiles;
    int64_t before = 0;
    int slots = 0;
    for (int r0 = 0; r0 < a.B; r0 += 64) {
        const int r = r0 + lane, n = r0 == 0 ? n0 : keys_of(a, r), splits = r < a.B ? max(1, (units_of(n) + per - 1) / per) : 0;
        const int mine = splits * each, in = wave_scan(mine), sl = splits > 1 ? mine : 0, in_sl = wave_scan(sl);
        const uint64_t hit = __ballot(idx >= before + in - mine && idx < before + in);
        if (hit) {
            const int w = __ffsll((unsigned long long)hit) - 1;
            const int k = (int)(idx - before) - scalar(in - mine, w);
            sh.row = r0 + w;
            sh.splits = scalar(splits, w);
            sh.n = scalar(n, w);
            sh.split = k / each;
            sh.head = k % each / a.tiles;
            sh.tile = k % a.tiles;
            sh.slot = slots + scalar(in_sl - sl, w) + (sh.head * a.tiles + sh.tile) * sh.splits;
            return true;
        }
        before += scalar(in, 63);
        slots += scalar(in_sl, 63);
    }
    return false;
}

// The output of q heads [first, first + count) from sums o over l (zero: no key).
__device__ __forceinline__ void store_out(const Args& a, size_t at, const f32x4& o, float l) {
    const float inv = l != 0.f ? 1.f / l : 0.f;
    float y[4];
    u32x2 g = {0, 0};
    if (a.gate) g = *reinterpret_cast<const u32x2*>(a.gate + at);
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

// Values that another block reads in the same launch.  Each XCD has an L2 of its own, so they are written through
// it and read past it (the accesses of an agent-scope atomic); a fence would instead write back all that the L2 holds,
// for every wave that executes it: 240 us in place of 25 for 32768 keys in 1024 shares.
__device__ __forceinline__ void put_shared(float* p, f32x2 v) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x2 get_shared(const float* p) {
    return __builtin_bit_cast(f32x2, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                                       __HIP_MEMORY_SCOPE_AGENT));
}

template <int DH>
__global__ void __launch_bounds__(THREADS, 2) attention_paged_kernel(const Args a) {
    constexpr int C = DH / 32, H = DH / 128, PITCH = DH + 8;
    extern __shared__ __attribute__((aligned(16))) float lds[];  // Q as operands, [C][64 lanes] x 16 bytes; later [WAVES][rows][PITCH]
    __shared__ float wm[WAVES][ROWS], wl[WAVES][ROWS];
    Share sh;
    if (!find_share(a, blockIdx.x, keys_of(a, threadIdx.x & 63), sh)) return;
    const int lane = threadIdx.x & 63, wave = scalar(threadIdx.x >> 6, 0), col = lane & 15, grp = lane >> 4;
    const int rows = min(ROWS, a.G - sh.tile * ROWS), head0 = sh.head * a.G + sh.tile * ROWS;
    const int s = scalar(sh.n > 0 ? (a.seqs ? a.seqs[sh.row] : sh.row) : 0, 0);
    // the row's units in equal parts
    const int units = units_of(sh.n), part = (units + sh.splits - 1) / sh.splits;
    const int u_end = min(units, (sh.split + 1) * part);
    int u = sh.split * part + wave;

    u32x4* const qf = reinterpret_cast<u32x4*>(lds);
#pragma unroll
    for (int c = wave; c < C; c += WAVES) {
        u32x4 q = {0, 0, 0, 0};
        if (col < rows) q = *reinterpret_cast<const u32x4*>(a.q + ((size_t)sh.row * a.Hq + head0 + col) * DH + c * 32 + grp * 8);
        qf[c * 64 + lane] = q;
    }
    f32x4 acc[H][8];
#pragma unroll
    for (int h = 0; h < H; h++)
#pragma unroll
        for (int j = 0; j < 8; j++) acc[h][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

    // where the next units' halves lie: lane i has half i % 2 of unit i / 2 from here (element offset, valid keys)
    const size_t token = (size_t)a.Hk * DH;
    int64_t where = 0;
    int valid = 0, next = 64;
    auto look_up = [&](int from) {
        const uint32_t key = (uint32_t)(from + (lane >> 1) * WAVES) * UNIT + (lane & 1) * 16, slot = key / (uint32_t)a.page;
        where = 0;
        valid = 0;
        if (key < (uint32_t)sh.n) {
            const int pg = a.table[(size_t)s * a.max_pages + slot];
            if (pg >= 0 && pg < a.npages) {
                where = ((int64_t)pg * a.page + (key - slot * a.page)) * token;
                valid = min(16, (int)(sh.n - key));
            }
        }
        where += sh.head * DH;
    };
    auto lane_of = [&](int64_t x, int i) {
        const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)x, i), hi = __builtin_amdgcn_readlane((uint32_t)(x >> 32), i);
        return (int64_t)((uint64_t)hi << 32 | lo);
    };
    u32x4 kf[2][C], vf[H][8];
    int64_t v_at[2];
    int have[2], v_have[2];
    // byte offsets of this lane in a half: 32 bits next to a base that the wave shares
    const uint32_t row_b = 2 * (uint32_t)token, k_lane = col * row_b + grp * 16, v_lane = grp * 4 * row_b + col * 16;
    auto load_k = [&](int from) {
        if (next == 64) {
            look_up(from);
            next = 0;
        }
#pragma unroll
        for (int t = 0; t < 2; t++) {
            v_at[t] = lane_of(where, next + t);
            have[t] = __builtin_amdgcn_readlane(valid, next + t);
            const char* const p = reinterpret_cast<const char*>(a.kp + v_at[t]);
#pragma unroll
            for (int c = 0; c < C; c++) kf[t][c] = *reinterpret_cast<const u32x4*>(p + (k_lane + c * 64));
        }
        next += 2;
    };
    auto load_v = [&]() {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            v_have[t] = have[t];
            const char* const p = reinterpret_cast<const char*>(a.vp + v_at[t]);
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    vf[h][t * 4 + i] = *reinterpret_cast<const u32x4*>(p + (v_lane + i * row_b + h * 256));
        }
    };
    if (u < u_end) {
        load_k(u);
        load_v();
    }
    __syncthreads();
    // one unit; more: the wave has another after it
    auto unit = [&](auto more) {
        f32x4 st[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            st[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < C; c++) st[t] = mfma16(kf[t][c], qf[c * 64 + lane], st[t]);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (decltype(more)::value) load_k(u + WAVES);
        __builtin_amdgcn_sched_barrier(0);
        float sc[8], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; i++) sc[i] = st[i >> 2][i & 3] * a.scale_log2;
        const bool whole = v_have[0] + v_have[1] == UNIT;
        if (!whole)
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (grp * 4 + (i & 3) >= v_have[i >> 2]) sc[i] = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; i++) top = fmaxf(top, sc[i]);
        if (__any(top > m + RISE)) {
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
            const float keep = top == m ? 1.f : __builtin_amdgcn_exp2f(m - top);
            m = top;
            l *= keep;
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int j = 0; j < 8; j++) acc[h][j] *= keep;
        }
        const float base = m == -INFINITY ? 0.f : m;  // no key yet: exp2(-inf) = 0
        u32x4 ph, pl;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float p0 = __builtin_amdgcn_exp2f(sc[2 * i] - base), p1 = __builtin_amdgcn_exp2f(sc[2 * i + 1] - base);
            l += p0 + p1;
            ph[i] = __builtin_amdgcn_perm(__float_as_uint(p1), __float_as_uint(p0), 0x07060302);
            pl[i] = pack2(fmaxf(p0 - lo_f32(ph[i]), LEAST), fmaxf(p1 - hi_f32(ph[i]), LEAST));
        }
        if (!whole)  // what lies where no key is may be anything; zero times it would not be zero
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (grp * 4 + (i & 3) >= v_have[i >> 2]) vf[h][i] = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                u32x4 vt;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    vt[i] = __builtin_amdgcn_perm(vf[h][2 * i + 1][j >> 1], vf[h][2 * i][j >> 1], j & 1 ? 0x07060302 : 0x05040100);
                acc[h][j] = mfma16(vt, ph, acc[h][j]);
                acc[h][j] = mfma16(vt, pl, acc[h][j]);
            }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (decltype(more)::value) load_v();
        __builtin_amdgcn_sched_barrier(0);
    };
    for (; u + WAVES < u_end; u += WAVES) unit(std::true_type{});
    if (u < u_end) unit(std::false_type{});

    // the waves join
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (grp == 0) {
        wm[wave][col] = m;
        wl[wave][col] = l;
    }
    __syncthreads();  // Q is no longer read
    if (col < rows)
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float* const to = lds + ((size_t)wave * rows + col) * PITCH + h * 128 + (grp * 4 + r) * 8;
                *reinterpret_cast<f32x4*>(to) = f32x4{acc[h][0][r], acc[h][1][r], acc[h][2][r], acc[h][3][r]};
                *reinterpret_cast<f32x4*>(to + 4) = f32x4{acc[h][4][r], acc[h][5][r], acc[h][6][r], acc[h][7][r]};
            }
    __syncthreads();
    // four dims of a row's result: to the output, or to a slot
    auto store = [&](int slot, int row, int d, float top, float sum, const f32x4& o, bool out) {
        const int head = head0 + row;
        if (out) {
            store_out(a, ((size_t)sh.row * a.Hq + head) * DH + d, o, sum);
            if (a.lse && d == 0) a.lse[(size_t)head * a.B + sh.row] = log_sum(top, sum);
            return;
        }
        const size_t at = (size_t)slot * ROWS + row;
        put_shared(a.part + at * DH + d, f32x2{o[0], o[1]});
        put_shared(a.part + at * DH + d + 2, f32x2{o[2], o[3]});
        if (d == 0) put_shared(a.ml + at * 2, f32x2{top, sum});
    };
    for (int e = threadIdx.x; e < rows * (DH / 4); e += THREADS) {
        const int row = e / (DH / 4), d = e % (DH / 4) * 4;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) top = fmaxf(top, wm[w][row]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float f = wm[w][row] == top ? 1.f : __builtin_amdgcn_exp2f(wm[w][row] - top);
            sum += wl[w][row] * f;
            o += *reinterpret_cast<const f32x4*>(lds + ((size_t)w * rows + row) * PITCH + d) * f;
        }
        store(sh.slot + sh.split, row, d, top, sum, o, sh.splits == 1);
    }
    if (sh.splits == 1) return;

    // Groups of `group` shares: the last of a group to end joins it, the last group joins the groups; always in order, so the
    // result does not depend on which ends last.  The counters are zero again afterwards.
    const int group = max(GROUP, (sh.splits + GROUPS_MAX - 1) / GROUPS_MAX), groups = (sh.splits + group - 1) / group;
    const int g0 = sh.split / group * group;
    auto last_of = [&](int* count, int n) {
        __shared__ int last;
        wait_vm_all();  // what this wave has put is where the others look
        __syncthreads();
        if (threadIdx.x == 0) {
            last = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
            if (last) *count = 0;
        }
        __syncthreads();
        return last != 0;
    };
    // n results from slot on, `step` slots apart: out, or back to the first slot
    auto join = [&](int slot, int step, int n, bool out) {
        f32x2* const ml = reinterpret_cast<f32x2*>(lds);
        for (int e = threadIdx.x; e < n * rows; e += THREADS)
            ml[e] = get_shared(a.ml + ((size_t)(slot + e / rows * step) * ROWS + e % rows) * 2);
        __syncthreads();
        for (int e = threadIdx.x; e < rows * (DH / 4); e += THREADS) {
            const int row = e / (DH / 4), d = e % (DH / 4) * 4;
            float top = -INFINITY, sum = 0.f;
            for (int k = 0; k < n; k++) top = fmaxf(top, ml[k * rows + row][0]);
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
            float* const from = a.part + ((size_t)slot * ROWS + row) * DH + d;
#pragma unroll 16
            for (int k = 0; k < n; k++) {
                const float* const p = from + (size_t)k * step * ROWS * DH;
                const f32x2 m = ml[k * rows + row], lo = get_shared(p), hi = get_shared(p + 2);
                const float f = m[0] == top ? 1.f : __builtin_amdgcn_exp2f(m[0] - top);
                sum += m[1] * f;
                o += f32x4{lo[0], lo[1], hi[0], hi[1]} * f;
            }
            store(slot, row, d, top, sum, o, out);
        }
    };
    if (!last_of(a.count + sh.slot + g0 / group, min(group, sh.splits - g0))) return;
    join(sh.slot + g0, 1, min(group, sh.splits - g0), groups == 1);
    if (groups == 1 || !last_of(a.count + 2 * a.target + sh.slot, groups)) return;
    join(sh.slot, group, groups, true);
}

template <int DH>
size_t lds_bytes(int rows) {
    const size_t q = 16 * 64 * (DH / 32), join = sizeof(float) * WAVES * rows * (DH + 8);
    const size_t group = sizeof(f32x2) * GROUPS_MAX * rows;
    return std::max(q, std::max(join, group));
}

template <int DH>
bool configure() {
    return hipFuncSetAttribute(reinterpret_cast<const void*>(attention_paged_kernel<DH>),
                               hipFuncAttributeMaxDynamicSharedMemorySize, lds_bytes<DH>(ROWS)) == hipSuccess;
}

template <int DH>
int launch(const Args& a, hipStream_t st) {
    const int64_t shares = (int64_t)a.target + (int64_t)a.B * a.Hk * a.tiles;
    attention_paged_kernel<DH><<<(unsigned)shares, THREADS, lds_bytes<DH>(a.G < ROWS ? a.G : ROWS), st>>>(a);
    return hipGetLastError();
}

}  // namespace
}  // namespace q35

using namespace q35;

extern "C" void* cs1_attention_paged_create(void) {
    int device;
    const int cus = device_cus();
    if (cus == 0 || hipGetDevice(&device) != hipSuccess || !configure<128>() || !configure<256>()) {
        (void)hipGetLastError();
        return nullptr;
    }
    Paged* const p = new (std::nothrow) Paged;
    if (!p) return nullptr;
    p->device = device;
    p->cus = cus;
    p->target = std::min(4 * cus, GROUPS_MAX * GROUPS_MAX);
    const size_t floats = (size_t)2 * p->target * ROWS * (256 + 2), counts = (size_t)4 * p->target;
    p->part = nullptr;
    if (hipMalloc(reinterpret_cast<void**>(&p->part), 4 * (floats + counts)) != hipSuccess ||
        hipMemset(p->part + floats, 0, 4 * counts) != hipSuccess || hipStreamSynchronize(nullptr) != hipSuccess) {
        (void)hipGetLastError();
        if (p->part) (void)hipFree(p->part);
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
    delete p;
}

extern "C" int cs1_attention_paged(void* paged, const void* q, const void* kp, const void* vp, const Cs1PageTable* pages,
                                   const int32_t* seqs, const void* gate, void* out, float* lse, int B, int Hq, int Hk,
                                   int Dh, float scale, void* stream) {
    const Paged* const p = static_cast<const Paged*>(paged);
    if (!p || !table_ok(pages) || (Dh != 128 && Dh != 256) || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 || B < 0 ||
        (int64_t)B * Hq > (1 << 22) || (int64_t)Hk * Dh > (1 << 24))
        return hipErrorInvalidValue;
    if (B == 0) return hipSuccess;
    if (!all_set({q, kp, vp, out}) || !on16(q) || !on16(kp) || !on16(vp) || !on16(out) || !on16(gate))
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
    a.part = p->part;
    a.ml = p->part + (size_t)2 * p->target * ROWS * 256;
    a.count = p->count;
    a.table = pages->table;
    a.lens = pages->lens;
    a.seqs = seqs;
    a.nseq = pages->nseq;
    a.max_pages = pages->max_pages;
    a.npages = pages->npages;
    a.page = pages->page;
    a.B = B;
    a.Hq = Hq;
    a.Hk = Hk;
    a.G = Hq / Hk;
    a.tiles = (a.G + ROWS - 1) / ROWS;
    a.target = p->target;
    a.scale_log2 = scale * LOG2E;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return Dh == 128 ? launch<128>(a, st) : launch<256>(a, st);
}
