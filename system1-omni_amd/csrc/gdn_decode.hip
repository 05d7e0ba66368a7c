// One token per sequence through a Gated DeltaNet layer (cs1_gdn_decode).  For the token x at position
// p of a sequence, per value head h with key head h / (H / HK):
//
//   y = silu(sum_i w_{3-i} x_{p-i}),  i = 0..3        (x_{p-1..p-3} from the ring; zero before 0)
//   q = scale q_y / sqrt(|q_y|^2 + 1e-6),  k = k_y / sqrt(|k_y|^2 + 1e-6),  v = v_y
//   d = exp(-exp(A_log) softplus(a + dt_bias)),  beta = sigmoid(b)
//   u = beta (v - d S^T k),   S' = d S + k u^T,   o = S'^T q = d S^T q + (q . k) u
//   out = norm_w o / sqrt(mean o^2 + eps) silu(z)
//
// With o written over S instead of S', one pass over S gives both S^T k and S^T q, and S' is formed from
// the registers that hold S: the state is read once and written once, 128 KiB a head, which is all
// but the whole traffic.  A block has one head of one row: 512 threads hold S in 32 registers each (4
// columns x 8 rows, a wave reads two whole rows at a time), so four blocks share a CU.  The conv of the key
// head's 256 channels is repeated by each of its value heads; the ring has four rows so that the row
// that is written (p % 4) is none of those that other blocks still read.
#include "common.h"
#include "paged.h"

namespace q35 {
namespace {

constexpr int DK = 128, THREADS = 512, WAVES = THREADS / 64;
constexpr int ROWS = 8;        // state rows a thread holds
constexpr int STEP = DK / ROWS;  // and the distance between them

struct Step {
    const bf16 *x, *w, *z, *b, *a, *a_log, *dt, *gw;
    bf16* ring;
    float* state;
    const int32_t *seqs, *lens;
    bf16* out;
    int ld, nseq, H, HK;
    float scale, eps;
};

// Sum over the wave, in a scalar register: rows of 16 lanes first, then row to row.
__device__ __forceinline__ float wave_sum(float x) {
#define Q35_ADD(ctrl, rows) \
    x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), ctrl, rows, 0xf, false))
    Q35_ADD(0x111, 0xf);
    Q35_ADD(0x112, 0xf);
    Q35_ADD(0x114, 0xf);
    Q35_ADD(0x118, 0xf);
    Q35_ADD(0x142, 0xa);
    Q35_ADD(0x143, 0xc);
#undef Q35_ADD
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63));
}

__global__ void __launch_bounds__(THREADS, 8) gdn_decode_kernel(const Step t) {
    __shared__ float y[3 * DK];              // q, k, v after the conv
    __shared__ float gates[2];               // decay, beta
    __shared__ float factor[DK];             // the norm's weight and the gate
    __shared__ float red[WAVES][2][DK];      // S^T k and S^T q by wave
    const int row = blockIdx.x / t.H, h = blockIdx.x % t.H, tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int group = t.H / t.HK, hk = h / group;
    bf16* const out = t.out + ((size_t)row * t.H + h) * DK;
    const int early = early_entry(t.seqs, row);
    const int s = __builtin_amdgcn_readfirstlane(listed_seq(t.seqs, row, t.nseq));
    const int p = __builtin_amdgcn_readfirstlane(s < 0 ? -1 : max(t.lens[s], 0) - 1);
    if (p < 0 || named_before(t.seqs, row, s, early)) {  // a padding row
        if (tid < DK) out[tid] = 0;
        return;
    }

    // Everything is asked for before anything is waited for.  The state goes past the caches (this layer's is not
    // read again before the other layers' have gone through them): 61 rows of 48 heads take 74 us so and 86 with
    // ordinary accesses. Columns 4 c .. 4 c + 3 of rows r0 + 16 i:
    const int c = tid & 31, r0 = tid >> 5;
    constexpr int NT = 2;  // the accesses' cache policy
    const auto st = __builtin_amdgcn_make_buffer_rsrc(t.state + ((size_t)s * t.H + h) * DK * DK, (short)0, DK * DK * 4,
                                                      0x00020000);
    const int at = (r0 * DK + 4 * c) * 4;
    f32x4 S[ROWS];
    if (p > 0) {
#pragma unroll
        for (int i = 0; i < ROWS; i++)
            S[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(st, at, i * STEP * DK * 4, NT));
    } else {
#pragma unroll
        for (int i = 0; i < ROWS; i++) S[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const bf16* const x = t.x + (size_t)row * t.ld;
    const int conv = (2 * t.HK + t.H) * DK;
    if (tid < 3 * DK) {
        const int part = tid >> 7, ch = (part == 2 ? 2 * t.HK + h : part * t.HK + hk) * DK + (tid & 127);
        bf16* const ring = t.ring + (size_t)s * 4 * conv + ch;
        const u32x2 w = *reinterpret_cast<const u32x2*>(t.w + (size_t)ch * 4);
        const bf16 now = x[ch];
        const bf16 x1 = ring[(size_t)((p - 1) & 3) * conv], x2 = ring[(size_t)((p - 2) & 3) * conv];
        const bf16 x3 = ring[(size_t)((p - 3) & 3) * conv];
        float acc = p > 2 ? lo_f32(w[0]) * f32(x3) : 0.f;
        acc = p > 1 ? fmaf(hi_f32(w[0]), f32(x2), acc) : acc;
        acc = p > 0 ? fmaf(lo_f32(w[1]), f32(x1), acc) : acc;
        y[tid] = silu(fmaf(hi_f32(w[1]), f32(now), acc));
        if (part == 2 || h % group == 0) ring[(size_t)(p & 3) * conv] = now;
    } else if (wave == WAVES - 2) {
        if (t.z)
#pragma unroll
            for (int i = lane; i < DK; i += 64)
                factor[i] = f32(t.gw[i]) * silu(f32(t.z[(size_t)row * t.ld + h * DK + i]));
    } else {
        const float xa = f32(t.a[(size_t)row * t.ld + h]) + f32(t.dt[h]);
        const float g = -expf(f32(t.a_log[h])) * (xa > 20.f ? xa : log1pf(expf(xa)));
        gates[0] = expf(g);
        gates[1] = sigmoid(f32(t.b[(size_t)row * t.ld + h]));
    }
    __syncthreads();

    auto dot = [&](const float* a, const float* b) {
        return wave_sum(a[lane] * b[lane] + a[64 + lane] * b[64 + lane]);
    };
    const float qi = rsqrtf(dot(y, y) + 1e-6f) * t.scale, ki = rsqrtf(dot(y + DK, y + DK) + 1e-6f);
    const float d = gates[0], beta = gates[1];
    f32x4 sk = {0.f, 0.f, 0.f, 0.f}, sq = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const float q = y[r0 + i * STEP] * qi, k = y[DK + r0 + i * STEP] * ki;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            S[i][e] *= d;
            sk[e] = fmaf(S[i][e], k, sk[e]);
            sq[e] = fmaf(S[i][e], q, sq[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        sk[e] += __shfl_xor(sk[e], 32, 64);
        sq[e] += __shfl_xor(sq[e], 32, 64);
    }
    if (lane < 32) {
        *reinterpret_cast<f32x4*>(&red[wave][0][4 * c]) = sk;
        *reinterpret_cast<f32x4*>(&red[wave][1][4 * c]) = sq;
    }
    __syncthreads();
    f32x4 u = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; w++) u += *reinterpret_cast<const f32x4*>(&red[w][0][4 * c]);
    u = (*reinterpret_cast<const f32x4*>(&y[2 * DK + 4 * c]) - u) * beta;
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
#pragma unroll
        for (int e = 0; e < 4; e++) S[i][e] = fmaf(y[DK + r0 + i * STEP] * ki, u[e], S[i][e]);
        // (no scalar offset: with one, the compiler writes the next product over S[i] in the instruction after the
        // store, and gfx950 then stores some lanes' new value)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, S[i]), st, at + i * STEP * DK * 4, 0, NT);
    }
    if (wave > 0) return;
    const float qk = dot(y, y + DK) * qi * ki;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; w++) o += *reinterpret_cast<const f32x4*>(&red[w][1][4 * c]);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        o[e] = fmaf(qk, u[e], o[e]);
        ss = fmaf(o[e], o[e], ss);
    }
    if (t.z) {
        const float inv = rsqrtf(lane_sum<32>(ss) * (1.f / DK) + t.eps);
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] *= inv * factor[4 * c + e];
    }
    if (lane < 32) *reinterpret_cast<u32x2*>(out + 4 * c) = u32x2{pack2(o[0], o[1]), pack2(o[2], o[3])};
}

}  // namespace
}  // namespace q35

using namespace q35;

extern "C" int cs1_gdn_decode(const void* qkv, int ld, const void* w, const void* z, const void* b, const void* a,
                              const void* A_log, const void* dt_bias, const void* norm_w, float eps, void* ring,
                              float* state, const int32_t* seqs, const int32_t* lens, int nseq, void* out, int B, int H,
                              int HK, float scale, void* stream) {
    if (B < 0 || B > MAX_LISTED || H <= 0 || HK <= 0 || H % HK != 0 || (int64_t)B * H > (1 << 22) || nseq <= 0)
        return hipErrorInvalidValue;
    const int64_t conv = ((int64_t)2 * HK + H) * DK;
    if (ld < conv || (z == nullptr) != (norm_w == nullptr)) return hipErrorInvalidValue;
    if (B == 0) return hipSuccess;
    if (!all_set({qkv, w, b, a, A_log, dt_bias, ring, state, lens, out}) || !on16(state))
        return hipErrorInvalidValue;
    if ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(out)) & 7) return hipErrorInvalidValue;
    Step t;
    t.x = static_cast<const bf16*>(qkv);
    t.w = static_cast<const bf16*>(w);
    t.z = static_cast<const bf16*>(z);
    t.b = static_cast<const bf16*>(b);
    t.a = static_cast<const bf16*>(a);
    t.a_log = static_cast<const bf16*>(A_log);
    t.dt = static_cast<const bf16*>(dt_bias);
    t.gw = static_cast<const bf16*>(norm_w);
    t.ring = static_cast<bf16*>(ring);
    t.state = state;
    t.seqs = seqs;
    t.lens = lens;
    t.out = static_cast<bf16*>(out);
    t.ld = ld;
    t.nseq = nseq;
    t.H = H;
    t.HK = HK;
    t.scale = scale;
    t.eps = eps;
    gdn_decode_kernel<<<B * H, THREADS, 0, static_cast<hipStream_t>(stream)>>>(t);
    return hipGetLastError();
}
