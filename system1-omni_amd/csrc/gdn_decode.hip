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

__global__ void __launch_bounds__(THREADS) gdn_decode_kernel(const Step t) {
    __shared__ float y[3 * DK];              // q, k, v after the conv
    __shared__ float red[WAVES][2][DK];      // S^T k and S^T q by wave
    const int row = blockIdx.x / t.H, h = blockIdx.x % t.H, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int group = t.H / t.HK, hk = h / group;
    bf16* const out = t.out + ((size_t)row * t.H + h) * DK;
    const int s = listed_seq(t.seqs, row, t.nseq);
    const int p = s < 0 ? -1 : max(t.lens[s], 0) - 1;
    const bool again = p >= 0 && named_before(t.seqs, row, s);

    // columns 4 c .. 4 c + 3 of rows r0 + 16 i
    const int c = tid & 31, r0 = tid >> 5;
    float* const st = t.state + ((size_t)max(s, 0) * t.H + h) * DK * DK + (size_t)r0 * DK + 4 * c;
    f32x4 S[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++)
        S[i] = p > 0 ? *reinterpret_cast<const f32x4*>(st + i * STEP * DK) : f32x4{0.f, 0.f, 0.f, 0.f};

    const int conv = (2 * t.HK + t.H) * DK;
    if (tid < 3 * DK && p >= 0) {
        const int part = tid >> 7, ch = (part == 2 ? 2 * t.HK + h : part * t.HK + hk) * DK + (tid & 127);
        const u32x2 w = *reinterpret_cast<const u32x2*>(t.w + (size_t)ch * 4);
        bf16* const ring = t.ring + (size_t)s * 4 * conv + ch;
        const bf16 x = t.x[(size_t)row * t.ld + ch];
        float acc = 0.f;
        if (p > 2) acc = fmaf(lo_f32(w[0]), f32(ring[(size_t)((p - 3) & 3) * conv]), acc);
        if (p > 1) acc = fmaf(hi_f32(w[0]), f32(ring[(size_t)((p - 2) & 3) * conv]), acc);
        if (p > 0) acc = fmaf(lo_f32(w[1]), f32(ring[(size_t)((p - 1) & 3) * conv]), acc);
        y[tid] = silu(fmaf(hi_f32(w[1]), f32(x), acc));
    }
    if (__syncthreads_or(again) || p < 0) {  // a padding row
        if (tid < DK) out[tid] = 0;
        return;
    }
    // (after the barrier: no row of this list writes the ring of a sequence that an earlier row has)
    if (tid < 3 * DK && (tid >= 2 * DK || h % group == 0)) {
        const int part = tid >> 7, ch = (part == 2 ? 2 * t.HK + h : part * t.HK + hk) * DK + (tid & 127);
        t.ring[((size_t)s * 4 + (p & 3)) * conv + ch] = t.x[(size_t)row * t.ld + ch];
    }

    const float q0 = y[lane], q1 = y[64 + lane], k0 = y[DK + lane], k1 = y[DK + 64 + lane];
    const float qi = rsqrtf(lane_sum<64>(q0 * q0 + q1 * q1) + 1e-6f) * t.scale;
    const float ki = rsqrtf(lane_sum<64>(k0 * k0 + k1 * k1) + 1e-6f);
    const float qk = lane_sum<64>(q0 * k0 + q1 * k1) * qi * ki;
    const float g = -expf(f32(t.a_log[h]));
    const float xa = f32(t.a[(size_t)row * t.ld + h]) + f32(t.dt[h]);
    const float d = expf(g * (xa > 20.f ? xa : log1pf(expf(xa))));
    const float beta = sigmoid(f32(t.b[(size_t)row * t.ld + h]));

    float kr[ROWS];
    f32x4 sk = {0.f, 0.f, 0.f, 0.f}, sq = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const float q = y[r0 + i * STEP] * qi;
        kr[i] = y[DK + r0 + i * STEP] * ki;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            S[i][e] *= d;
            sk[e] = fmaf(S[i][e], kr[i], sk[e]);
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
#pragma unroll
    for (int e = 0; e < 4; e++) u[e] = beta * (y[2 * DK + 4 * c + e] - u[e]);
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
#pragma unroll
        for (int e = 0; e < 4; e++) S[i][e] = fmaf(kr[i], u[e], S[i][e]);
        *reinterpret_cast<f32x4*>(st + i * STEP * DK) = S[i];
    }
    if (wave > 0) return;
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
        for (int e = 0; e < 4; e++)
            o[e] = f32(t.gw[4 * c + e]) * (o[e] * inv) * silu(f32(t.z[(size_t)row * t.ld + h * DK + 4 * c + e]));
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
    if (B < 0 || B > MAX_LISTED || H <= 0 || HK <= 0 || H % HK != 0 || (int64_t)B * H > (1 << 22) || nseq <= 0) return hipErrorInvalidValue;
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
