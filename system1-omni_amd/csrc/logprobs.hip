// Log-probabilities of given tokens, entropy and the best alternatives of rows of logits (cs1_token_logprobs).  With
// m = max x, z = sum e^(x - m):
//
//   log p_t = (x_t - m) - log z,   H = -sum p log p = log z - sum e^(x - m) (x - m) / z,
//
// and the k largest logits, the lowest index first among equals.  No term of H is negative, so nothing cancels.
//
// Bound by the one pass over the logits.  A thread keeps a running base, sum and weighted sum of its own, and of its
// values the largest with the load that it was in.  The alternatives need no more from that pass: the
// k-th largest of the lanes' largest (64 lanes, each over the block's waves) is a value that k tokens reach at least, so
// only what reaches it can be among the best, and only the threads whose largest does (about k of them) look at
// their loads again.  What they find, k tokens or a few more, is put in order by counting.
//
// A row is cut into parts where there are few rows; a second launch joins the parts in order.
//
// 1217 rows of 248320 bfloat16 logits with 5 alternatives take 118 us (5.1 TB/s), one row of 151936 with 20 in 64 parts 12.8
// in two launches: in the first the load, the sums' and the alternatives' exchanges, in the second the alternatives one by one.
#include <math.h>

#include <algorithm>
#include <limits>

#include "common.h"
#include "paged.h"

namespace q35 {
namespace {

constexpr int LOADS = 4;  // of 16 bytes a thread has under way
constexpr int K_MAX = 32, PARTS_MAX = 64;
constexpr int LIST = 1024;  // tokens that reach the threshold, kept in LDS
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// A logit with its index, larger for larger values and among equals for lower indices; 0 is below all.  (-0 is 0.)
typedef unsigned long long Key;
__device__ __forceinline__ Key key_of(float x, uint32_t index) {
    const uint32_t b = __float_as_uint(x + 0.f), up = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (Key)up << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float value_of(Key k) {
    const uint32_t up = (uint32_t)(k >> 32);
    return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}
__device__ __forceinline__ uint32_t index_of(Key k) { return 0xffffffffu - (uint32_t)k; }

// Over a wave's lanes, the same in each: within rows of 16, then each row's last lane to the next row, then lane 31 to
// the upper half.  (Shuffles go through LDS and take many times as long: a row's alternatives from 38 parts took 11 us by
// them, and take 6 so.)
template <typename T, typename F>
__device__ __forceinline__ T over_wave(T x, T none, F f) {
#define Q35_STEP(ctrl, rows)                                                                                            \
    x = f(x, __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, x), \
                                                               ctrl, rows, 0xf, false)))
    Q35_STEP(0x111, 0xf);
    Q35_STEP(0x112, 0xf);
    Q35_STEP(0x114, 0xf);
    Q35_STEP(0x118, 0xf);
    Q35_STEP(0x142, 0xa);
    Q35_STEP(0x143, 0xc);
#undef Q35_STEP
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    return over_wave(x, 0u, [](uint32_t a, uint32_t b) { return max(a, b); });
}
__device__ __forceinline__ float wave_max(float x) {
    return over_wave(x, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float x) {
    return over_wave(x, 0.f, [](float a, float b) { return a + b; });
}
// The lane that has the largest key of the wave (the first of several), and the key.
__device__ __forceinline__ int wave_best(Key mine, Key& best) {
    const uint32_t hi = (uint32_t)(mine >> 32), lo = (uint32_t)mine, most = wave_max(hi);
    uint64_t have = __ballot(hi == most);
    if (have & (have - 1)) {
        const uint32_t of = hi == most ? lo : 0u, first = wave_max(of);
        have = __ballot(hi == most && of == first);
    }
    const int lane = __ffsll((unsigned long long)have) - 1;
    best = (Key)most << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, lane);
    return lane;
}

// Base m, sum of e^(x - m) and of that times x - m.  Differences and not logarithms of base 2 are kept, so that a large
// base costs no bits.
struct Sums {
    float m, sum, dot, unused;
};
// By how much a base falls, as far as anything is left: -1e4 stands for all that leaves nothing, so that sums of values
// near the type's lowest do not become infinities times zero.
__device__ __forceinline__ float falls(float from, float to) { return fmaxf(from - to, -1e4f); }
__device__ __forceinline__ Sums rebased(const Sums& a, float m) {
    if (a.m == -INFINITY) return Sums{m, a.sum, a.dot, 0.f};  // no value yet, or none above -inf
    const float by = falls(a.m, m), f = __builtin_amdgcn_exp2f(by * LOG2E);
    return Sums{m, a.sum * f, (a.dot + a.sum * by) * f, 0.f};
}
__device__ __forceinline__ Sums merged(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m);
    const Sums x = rebased(a, m), y = rebased(b, m);
    return Sums{m, x.sum + y.sum, x.dot + y.dot, 0.f};
}
__device__ __forceinline__ Sums wave_merged(Sums a) {
    a = rebased(a, wave_max(a.m));
    return Sums{a.m, wave_sum(a.sum), wave_sum(a.dot), 0.f};
}

struct Args {
    const void* logits;
    const int32_t* targets;
    float *logprob, *entropy, *top;
    int32_t* ids;
    Sums* sums;  // [rows, parts]
    Key* keys;   // [rows, parts, k]
    size_t ld;
    int V, k, parts, each;  // each: logits a part, a multiple of 8
};

template <typename T>
__device__ __forceinline__ float as_float(T x) {
    if constexpr (sizeof(T) == 2)
        return f32(x);
    else
        return x;
}

// A row whose sum is no positive number (a NaN or +inf among its logits, or all of them -inf) has no distribution.
__device__ __forceinline__ bool proper(const Sums& s) { return s.sum > 0.f; }
__device__ __forceinline__ float no_number() { return __uint_as_float(0x7fc00000); }

template <typename T>
__device__ __forceinline__ void store_row(const Args& a, int row, const Sums& s) {
    const float log_z = log2f(s.sum) * LN2;
    if (a.logprob) {
        const int t = a.targets[row];
        float lp = 0.f;
        if (t >= 0 && t < a.V)
            lp = proper(s) ? (as_float(static_cast<const T*>(a.logits)[(size_t)row * a.ld + t]) - s.m) - log_z
                           : no_number();
        a.logprob[row] = lp;
    }
    if (a.entropy) a.entropy[row] = proper(s) ? log_z - s.dot / s.sum : no_number();
}
__device__ __forceinline__ void store_top(const Args& a, int row, int i, Key k, const Sums& s) {
    const bool ok = proper(s) && k != 0;
    a.ids[(size_t)row * a.k + i] = ok ? (int)index_of(k) : -1;
    a.top[(size_t)row * a.k + i] = ok ? (value_of(k) - s.m) - log2f(s.sum) * LN2 : no_number();
}

// A part of a row as loads of 16 bytes: number 0 has the logits in front of the first aligned one (fewer, or none), 1 ..
// `whole` are full, and whole + 1 has what is left.  A thread has every so many-th, so its indices rise.
template <typename T>
struct Part {
    static constexpr int N = 16 / sizeof(T);
    const T* p;
    int n, head, whole;

    __device__ __forceinline__ Part(const T* p, int n) : p(p), n(n) {
        const int off = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
        head = min(off ? N - off : 0, n);
        whole = (n - head) / N;
    }
    __device__ __forceinline__ int index(int j) const { return j == 0 ? 0 : head + (j - 1) * N; }
    __device__ __forceinline__ int count(int j) const {
        return j == 0 ? head : j <= whole ? N : j == whole + 1 ? n - head - whole * N : 0;
    }
    __device__ __forceinline__ u32x4 full(int j) const {
        return *reinterpret_cast<const u32x4*>(p + head + (size_t)(j - 1) * N);
    }
    static __device__ __forceinline__ float at(const u32x4& v, int e) {
        if constexpr (sizeof(T) == 2)
            return e & 1 ? hi_f32(v[e / 2]) : lo_f32(v[e / 2]);
        else
            return __uint_as_float(v[e]);
    }
    // f(key) for each logit of load j
    template <typename F>
    __device__ __forceinline__ void each_key(int j, uint32_t first, F f) const {
        if (j >= 1 && j <= whole) {
            const u32x4 v = full(j);
#pragma unroll
            for (int e = 0; e < N; e++) f(key_of(at(v, e), first + index(j) + e));
        } else {
            for (int e = 0; e < count(j); e++) f(key_of(as_float(p[index(j) + e]), first + index(j) + e));
        }
    }
};

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) logprobs_kernel(const Args a) {
    constexpr int N = Part<T>::N, WAVES = THREADS / 64;
    __shared__ Sums wave_sums[WAVES];
    __shared__ Key best_of[64], list[LIST + WAVES], found;
    __shared__ int listed, threads, who[THREADS], above[64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.x / (uint32_t)a.parts, part = blockIdx.x - row * a.parts;
    const int first = part * a.each;
    const Part<T> x(static_cast<const T*>(a.logits) + (size_t)row * a.ld + first, min(a.each, a.V - first));
    if (tid < 64) {
        best_of[tid] = 63 - tid;  // below all, and none like another
        above[tid] = 0;
    }
    if (tid == 0) listed = threads = 0;

    float m = -INFINITY, sum = 0.f, dot = 0.f, best = -INFINITY;
    int best_at = -1;  // the load that has the largest value first
    auto rebase = [&](float top) {
        if (top > m) {
            const float by = falls(m, top), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(by * LOG2E);
            dot = m == -INFINITY ? 0.f : (dot + sum * by) * f;
            sum *= f;
            m = top;
        }
    };
    auto add = [&](float v, float base) {
        const float d = v - base, p = __builtin_amdgcn_exp2f(d * LOG2E);
        sum += p;
        dot += p * fmaxf(d, -1e4f);  // (what is -inf weighs nothing, and must not be multiplied by its zero)
    };
    auto single = [&](int j) {  // load 0 or the last one
        for (int e = 0; e < x.count(j); e++) {
            const float v = as_float(x.p[x.index(j) + e]);
            rebase(v);
            add(v, m == -INFINITY ? 0.f : m);
            if (v > best || best_at < 0) {
                best = fmaxf(v, -INFINITY);
                best_at = j;
            }
        }
    };
    if (tid == 0) single(0);
    for (int j0 = tid == 0 ? THREADS : tid; j0 <= x.whole; j0 += LOADS * THREADS) {
        u32x4 v[LOADS];
        constexpr uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;  // -inf
#pragma unroll
        for (int u = 0; u < LOADS; u++) {
            v[u] = u32x4{none, none, none, none};
            if (j0 + u * THREADS <= x.whole) v[u] = x.full(j0 + u * THREADS);
        }
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < LOADS; u++) {
            float most = x.at(v[u], 0);
#pragma unroll
            for (int e = 1; e < N; e++) most = fmaxf(most, x.at(v[u], e));
            if (most > best || best_at < 0) {
                best = fmaxf(most, -INFINITY);
                best_at = j0 + u * THREADS;
            }
            top = fmaxf(top, most);
        }
        rebase(top);
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int u = 0; u < LOADS; u++)
#pragma unroll
            for (int e = 0; e < N; e++) add(x.at(v[u], e), base);
    }
    if (tid == (x.whole + 1) % THREADS) single(x.whole + 1);

    Sums s = wave_merged(Sums{m, sum, dot, 0.f});
    if (lane == 0) wave_sums[wave] = s;
    __syncthreads();
    s = wave_sums[0];
#pragma unroll
    for (int w = 1; w < WAVES; w++) s = merged(s, wave_sums[w]);
    if (tid == 0) {
        if (a.parts == 1)
            store_row<T>(a, row, s);
        else
            a.sums[blockIdx.x] = s;
    }
    if (a.k == 0) return;

    // where the load has it is not known, so the value counts as its last logit here, and as its first below
    if (best_at >= 0) atomicMax(&best_of[lane], key_of(best, first + x.index(best_at) + x.count(best_at) - 1));
    __syncthreads();
    const Key its = best_of[lane];
    int larger = 0;
#pragma unroll
    for (int j = 0; j < 64 / WAVES; j++) larger += best_of[wave * (64 / WAVES) + j] > its;
    atomicAdd(&above[lane], larger);
    __syncthreads();
    const int kth = __ffsll((unsigned long long)__ballot(above[lane] == a.k - 1)) - 1;
    const Key least = (Key)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(its >> 32), kth) << 32 |
                      (uint32_t)__builtin_amdgcn_readlane((uint32_t)its, kth);
    if (best_at >= 0 && key_of(best, first + x.index(best_at)) >= least) who[atomicAdd(&threads, 1)] = tid;
    __syncthreads();
    const int loads = (x.whole + 1) / THREADS + 1;  // of a thread, at most
    for (int i = tid; i < threads * loads; i += THREADS)
        x.each_key(who[i / (uint32_t)loads] + i % (uint32_t)loads * THREADS, first, [&](Key k) {
            if (k < least) return;
            const int at = atomicAdd(&listed, 1);
            if (at < LIST) list[at] = k;
        });
    __syncthreads();
    auto store = [&](int i, Key k) {
        if (a.parts == 1)
            store_top(a, row, i, k, s);
        else
            a.keys[(size_t)blockIdx.x * a.k + i] = k;
    };
    if (listed <= LIST) {
        for (int i = tid; i < max(listed, a.k); i += THREADS) {
            if (i >= listed) {  // fewer logits than alternatives
                store(i, 0);
                continue;
            }
            const Key mine = list[i];
            int rank = 0;
            for (int j = 0; j < listed; j += WAVES)  // (some on their way at once)
#pragma unroll
                for (int u = 0; u < WAVES; u++) rank += j + u < listed && list[j + u] > mine;
            if (rank < a.k) store(rank, mine);
        }
        return;
    }
    // More than LIST reach it: a few lanes' loads have all large values.  The alternatives are looked for one by one.
    Key before = ~(Key)0;
    for (int i = 0; i < a.k; i++) {
        if (tid == 0) found = 0;
        __syncthreads();
        Key mine = 0;
        for (int j = tid; j <= x.whole + 1; j += THREADS)
            x.each_key(j, first, [&](Key k) {
                if (k < before && k > mine) mine = k;
            });
        (void)wave_best(mine, mine);
        if (lane == 0) atomicMax(&found, mine);
        __syncthreads();
        before = found;
        if (tid == 0) store(i, before);
        __syncthreads();
    }
}

// Joins a row's parts: wave 0 the alternatives, a lane for a part, whose own are in order; wave 1 the sums.
constexpr int JOIN_THREADS = 256;
template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS) logprobs_join_kernel(const Args a) {
    constexpr int MINE = PARTS_MAX * K_MAX / JOIN_THREADS;
    __shared__ Key keys[PARTS_MAX * K_MAX];
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, all = a.parts * a.k;
    Key v[MINE];
#pragma unroll
    for (int i = 0; i < MINE; i++)
        if (tid + i * JOIN_THREADS < all) v[i] = a.keys[(size_t)row * all + tid + i * JOIN_THREADS];
    Sums s = Sums{-INFINITY, 0.f, 0.f, 0.f};
    if (lane < a.parts) s = a.sums[(size_t)row * a.parts + lane];
#pragma unroll
    for (int i = 0; i < MINE; i++)
        if (tid + i * JOIN_THREADS < all) keys[tid + i * JOIN_THREADS] = v[i];
    __syncthreads();
    if (tid >= 128) return;
    s = wave_merged(s);
    if (tid == 64) store_row<T>(a, row, s);
    if (tid >= 64) return;
    Key mine = 0;  // the lane-th best
    int next = 0;
    auto at = [&](int i) { return lane < a.parts && i < a.k ? keys[lane * a.k + i] : (Key)0; };
    Key head = at(0), after = at(1);  // (what follows is on its way while the best is looked for)
    for (int i = 0; i < a.k; i++) {
        Key best;
        const int from = wave_best(head, best);
        if (lane == i) mine = best;
        if (lane == from) {
            head = after;
            after = at(++next + 1);
        }
    }
    if (lane < a.k) store_top(a, row, lane, mine, s);
}

// Parts of a row: enough blocks for the chip, of at least a load a thread.  A block has 256 threads, which begin and end
// sooner, or 512, which read on more evenly, from 2^26 logits on: 300 rows of 151936 take 25.6 and 29.7 us, 2000 of 1400 9.9 and
// 14.4, one of 151936 with 20 alternatives 12.7 and 13.8; 1217 of 248320 119.6 and 117.5, 500 of 151936 in float32 58 and 56.
constexpr int ONE_PART = 1024;  // blocks that are enough: so many rows and more are not cut
struct Plan {
    int parts, each, threads;
};
Plan plan_of(int rows, int V) {
    const int threads = (int64_t)rows * V < 1 << 26 ? 256 : 512;
    const int64_t wanted = (ONE_PART + (int64_t)rows - 1) / rows, most = (V + 8 * threads - 1) / (8 * threads);
    const int parts = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(wanted, most), PARTS_MAX));
    const int each = (int)((((int64_t)V + parts - 1) / parts + 7) / 8 * 8);
    return Plan{(int)(((int64_t)V + each - 1) / each), each, threads};
}

constexpr int V_MAX = 1 << 28, ROWS_MAX = (1 << 23) - 1;  // (a launch has under 2^32 threads, 512 for a row)

}  // namespace
}  // namespace q35

using namespace q35;

extern "C" size_t cs1_token_logprobs_workspace_bytes(int rows, int V, int k) {
    if (rows <= 0 || V <= 0 || V > V_MAX || k < 0 || k > K_MAX) return 0;
    // The plan's own number of parts goes up and down with the rows and tokens; this bound on it only up, so that a
    // program can keep one workspace: up to 64 parts of a row, none shorter than 2048 logits, ceil(1024 / rows) at most.
    constexpr int LEAST = 8 * 256;
    if (rows >= ONE_PART || V <= LEAST) return 0;
    const int most = std::min((V + LEAST - 1) / LEAST, PARTS_MAX);
    return (size_t)std::min(rows * most, rows + ONE_PART - 1) * (sizeof(Sums) + sizeof(Key) * k);
}

extern "C" int cs1_token_logprobs(const void* logits, int is_float, size_t ld, const int32_t* targets, int rows, int V,
                                  int k, float* logprob, float* entropy, int32_t* top_ids, float* top_logprobs,
                                  void* workspace, void* stream) {
    if (rows < 0 || rows > ROWS_MAX || V <= 0 || V > V_MAX || ld < (size_t)V || k < 0 || k > K_MAX) return hipErrorInvalidValue;
    if (rows == 0) return hipSuccess;
    const Plan p = plan_of(rows, V);
    if (!logits || (logprob != nullptr) != (targets != nullptr) ||
        (k > 0 && !all_set({top_ids, top_logprobs})))
        return hipErrorInvalidValue;
    if ((reinterpret_cast<uintptr_t>(logits) & (is_float ? 3 : 1)) != 0) return hipErrorInvalidValue;
    if (p.parts > 1 && (!workspace || !on16(workspace))) return hipErrorInvalidValue;
    Args a;
    a.logits = logits;
    a.targets = targets;
    a.logprob = logprob;
    a.entropy = entropy;
    a.top = top_logprobs;
    a.ids = top_ids;
    a.sums = static_cast<Sums*>(workspace);
    a.keys = reinterpret_cast<Key*>(a.sums + (size_t)rows * p.parts);
    a.ld = ld;
    a.V = V;
    a.k = k;
    a.parts = p.parts;
    a.each = p.each;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const auto kernel = p.threads == 256 ? (is_float ? logprobs_kernel<float, 256> : logprobs_kernel<bf16, 256>)
                                         : (is_float ? logprobs_kernel<float, 512> : logprobs_kernel<bf16, 512>);
    kernel<<<rows * p.parts, p.threads, 0, st>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.parts == 1) return e;
    const auto join = is_float ? logprobs_join_kernel<float> : logprobs_join_kernel<bf16>;
    join<<<rows, JOIN_THREADS, 0, st>>>(a);
    return hipGetLastError();
}
