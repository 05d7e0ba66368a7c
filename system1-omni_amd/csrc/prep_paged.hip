// Attention inputs of rows that continue sequences (cs1_attn_prep_paged): per-head norm, rotary positions, and keys and
// values straight into their pages.  For a head x of a row at position p, with y = x rsqrt(mean x^2 + eps) (1 + w),
// each pair (a, b) of the first `dims` dims becomes m (a cos t - b sin t, b cos t + a sin t), t = p f_i.
//
// Bound by memory: a row of the projection is read once and every value written once, so each thread asks for all that it
// needs of BATCH heads before it waits.  A block has a row: its angles are formed once, in turns in float64 (p f / 2 pi
// less its whole turns, so that float32 sees half a turn at most, at any position), while the row is on its way.  4096
// rows of 16/4 heads of 256 with gates (168 MB): 29.3 us, 5.7 TB/s.
#include <math.h>

#include "common.h"
#include "paged.h"

namespace q35 {
namespace {

constexpr int THREADS = 256, BATCH = 4;

struct Args {
    const bf16 *qg, *kr, *v, *qw, *kw;
    const double* freqs;
    const int32_t *pos, *slot;
    bf16 *q, *gate, *kp, *vp;
    int ld, Hq, Hk, dims, interleaved, slots;
    float eps, magnitude;
};

template <int DH>
__global__ void __launch_bounds__(THREADS) attn_prep_paged_kernel(const Args a) {
    constexpr int LANES = DH / 8, EACH = THREADS / LANES;  // lanes a head, heads at a time
    __shared__ __align__(16) float cs[DH / 2], sn[DH / 2];
    const int t = blockIdx.x, tid = threadIdx.x, sub = tid % LANES, d0 = sub * 8;
    asm volatile("" ::"s"(a.qg), "s"(a.kr), "s"(a.v), "s"(a.qw), "s"(a.kw), "s"(a.freqs), "s"(a.pos), "s"(a.slot),
                 "s"(a.q), "s"(a.gate), "s"(a.kp), "s"(a.vp), "s"(a.ld), "s"(a.Hq), "s"(a.Hk), "s"(a.dims),
                 "s"(a.interleaved), "s"(a.slots), "s"(a.eps), "s"(a.magnitude));
    const int pos = a.pos[t], slot = a.slot[t], half = a.dims / 2, heads = a.Hq + 2 * a.Hk;
    double f = 0.0;
    if (tid < half) f = a.freqs[tid];
    const size_t row = (size_t)t * a.ld;
    const int wide = a.gate ? 2 * DH : DH;
    Pack8 wq = {}, wk = {};
    if (a.qw) wq = *reinterpret_cast<const Pack8*>(a.qw + d0);
    if (a.kw) wk = *reinterpret_cast<const Pack8*>(a.kw + d0);
    for (int h0 = tid / LANES; h0 - tid / LANES < heads; h0 += BATCH * EACH) {
        Pack8 x[BATCH], g[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; i++) {
            const int h = h0 + i * EACH;
            x[i] = g[i] = Pack8{};
            if (h >= heads) continue;
            const bf16* const from = h < a.Hq             ? a.qg + row + (size_t)h * wide
                                     : h < a.Hq + a.Hk ? a.kr + row + (size_t)(h - a.Hq) * DH
                                                       : a.v + row + (size_t)(h - a.Hq - a.Hk) * DH;
            x[i] = *reinterpret_cast<const Pack8*>(from + d0);
            if (a.gate && h < a.Hq) g[i] = *reinterpret_cast<const Pack8*>(from + DH + d0);
        }
        if (h0 == tid / LANES) {  // the first time
            if (tid < half) {
                const double turns = pos * (f * 0.15915494309189535);
                float s, c;
                sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
                cs[tid] = c * a.magnitude;
                sn[tid] = s * a.magnitude;
            }
            __syncthreads();
        }
        if (pos < 0) return;
#pragma unroll
        for (int i = 0; i < BATCH; i++) {
            const int h = h0 + i * EACH;
            const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hk;
            float y[8];
            unpack8(x[i], y);
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) ss += y[e] * y[e];
            ss = lane_sum<LANES>(ss);
            if (is_q ? a.qw != nullptr : a.kw != nullptr) {
                float w[8];
                unpack8(is_q ? wq : wk, w);
                const float inv = rsqrtf(ss / DH + a.eps);
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = y[e] * inv * (1.f + w[e]);
            }
            if (a.interleaved) {
                if (d0 < a.dims)
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const float c = cs[(d0 + e) / 2], s = sn[(d0 + e) / 2], lo = y[e], hi = y[e + 1];
                        y[e] = lo * c - hi * s;
                        y[e + 1] = hi * c + lo * s;
                    }
            } else {
                // the other value of a pair is half / 8 lanes away
                const bool low = d0 < half;
                const int other = ((tid & 63) + (low ? half / 8 : -half / 8)) & 63, at = low ? d0 : d0 - half;
                float z[8];
#pragma unroll
                for (int e = 0; e < 8; e++) z[e] = __shfl(y[e], other, 64);
                if (d0 < a.dims)
#pragma unroll
                    for (int e = 0; e < 8; e++) y[e] = y[e] * cs[at + e] + (low ? -z[e] : z[e]) * sn[at + e];
            }
            if (h >= heads) continue;
            if (is_q) {
                const size_t to = ((size_t)t * a.Hq + h) * DH + d0;
                *reinterpret_cast<Pack8*>(a.q + to) = pack8(y);
                if (a.gate) *reinterpret_cast<Pack8*>(a.gate + to) = g[i];
            } else if (slot >= 0 && slot < a.slots) {
                const size_t to = ((size_t)slot * a.Hk + (h - a.Hq - (is_v ? a.Hk : 0))) * DH + d0;
                if (is_v)
                    *reinterpret_cast<Pack8*>(a.vp + to) = x[i];
                else
                    *reinterpret_cast<Pack8*>(a.kp + to) = pack8(y);
            }
        }
    }
}

}  // namespace
}  // namespace q35

using namespace q35;

extern "C" int cs1_rotary_freqs(double* freqs, int dims, double base, double factor, double original, double slow,
                                double fast) {
    if (!freqs || dims <= 0 || dims % 2 != 0 || !(base > 0.0) || !(factor >= 1.0) || !(original > 0.0) || !(slow >= 0.0) ||
        !(fast >= slow))
        return hipErrorInvalidValue;
    for (int i = 0; i < dims / 2; i++) {
        const double f = pow(base, -2.0 * i / dims), turns = original * f / 6.283185307179586;
        const double keep = turns >= fast ? 1.0 : turns <= slow || fast == INFINITY ? 0.0 : (turns - slow) / (fast - slow);
        freqs[i] = f * ((1.0 - keep) / factor + keep);
    }
    return hipSuccess;
}

extern "C" int cs1_attn_prep_paged(const void* qg, const void* kr, const void* v, int ld, const void* qw,
                                   const void* kw, float eps, const Cs1Rotary* rotary, const Cs1PageTable* pages,
                                   const int32_t* pos, const int32_t* slot, void* q, void* gate, void* kp, void* vp,
                                   int T, int Hq, int Hk, int Dh, void* stream) {
    if (T < 0 || Hq <= 0 || Hk <= 0 || (Dh != 128 && Dh != 256) || !rotary || !pages) return hipErrorInvalidValue;
    if ((int64_t)T * THREADS > UINT32_MAX) return hipErrorInvalidValue;  // (a launch has under 2^32 threads)
    const int64_t wide = (int64_t)Hq * Dh * (gate ? 2 : 1), slots = (int64_t)pages->npages * pages->page;
    if (ld % 8 != 0 || ld < wide || ld < (int64_t)Hk * Dh || (int64_t)Hk * Dh > (1 << 24) || pages->npages <= 0 ||
        pages->page <= 0 || slots > INT32_MAX)
        return hipErrorInvalidValue;
    if (rotary->dims < 0 || rotary->dims % 16 != 0 || rotary->dims > Dh || (rotary->dims > 0 && !rotary->freqs) ||
        (reinterpret_cast<uintptr_t>(rotary->freqs) & 7) != 0)
        return hipErrorInvalidValue;
    if (T == 0) return hipSuccess;
    if (!all_set({qg, kr, v, pos, slot, q, kp, vp})) return hipErrorInvalidValue;
    for (const void* p : {qg, kr, v, qw, kw, (const void*)q, (const void*)gate, (const void*)kp, (const void*)vp})
        if (!on16(p)) return hipErrorInvalidValue;
    Args a;
    a.qg = static_cast<const bf16*>(qg);
    a.kr = static_cast<const bf16*>(kr);
    a.v = static_cast<const bf16*>(v);
    a.qw = static_cast<const bf16*>(qw);
    a.kw = static_cast<const bf16*>(kw);
    a.freqs = rotary->freqs;
    a.pos = pos;
    a.slot = slot;
    a.q = static_cast<bf16*>(q);
    a.gate = static_cast<bf16*>(gate);
    a.kp = static_cast<bf16*>(kp);
    a.vp = static_cast<bf16*>(vp);
    a.ld = ld;
    a.Hq = Hq;
    a.Hk = Hk;
    a.dims = rotary->dims;
    a.interleaved = rotary->interleaved != 0;
    a.slots = (int)slots;
    a.eps = eps;
    a.magnitude = rotary->magnitude;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (Dh == 128)
        attn_prep_paged_kernel<128><<<T, THREADS, 0, st>>>(a);
    else
        attn_prep_paged_kernel<256><<<T, THREADS, 0, st>>>(a);
    return hipGetLastError();
}
