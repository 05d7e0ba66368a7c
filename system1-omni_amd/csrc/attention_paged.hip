// Attention of one new token per row over a paged key-value cache (cs1_attention_paged).  For a row of sequence s
// with n = lens[s] keys and q head h on kv head h / (Hq / Hk):
//
//   S_j = scale q . k_j,  m = max S_j,  l = sum exp(S_j - m),  out = gate_sigmoid * (sum exp(S_j - m) v_j) / l,
//   lse = m + log l.
//
// One block per row and q head; its four waves take every fourth key with a running maximum and
// sum each, a lane holding Dh / 64 dims, and join at the end.
#include <new>

#include "common.h"
#include "paged.h"

namespace q35 {
namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Paged {
    int device;
};

struct Args {
    const bf16 *q, *kp, *vp, *gate;
    bf16* out;
    float* lse;
    const int32_t *table, *lens, *seqs;
    int nseq, max_pages, npages, page, B, Hq, Hk;
    float scale_log2;
};

template <int DH>
__global__ void __launch_bounds__(THREADS) attention_paged_kernel(const Args a) {
    constexpr int V = DH / 64;
    __shared__ float om[WAVES], ol[WAVES], oa[WAVES][DH];
    const int r = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq, hk = h / (a.Hq / a.Hk);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int s = listed_seq(a.seqs, r, a.nseq);
    const int n = s < 0 ? 0 : (int)min((int64_t)max(a.lens[s], 0), (int64_t)a.max_pages * a.page);
    const size_t row = ((size_t)r * a.Hq + h) * DH + lane * V;
    float q[V], acc[V], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < V; e++) {
        q[e] = f32(a.q[row + e]);
        acc[e] = 0.f;
    }
    for (int j = wave; j < n; j += WAVES) {
        const int pg = a.table[(size_t)s * a.max_pages + j / a.page];
        if (pg < 0 || pg >= a.npages) continue;
        const size_t at = (((size_t)pg * a.page + j % a.page) * a.Hk + hk) * DH + lane * V;
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < V; e++) dot = fmaf(q[e], f32(a.kp[at + e]), dot);
        const float sc = lane_sum<64>(dot) * a.scale_log2, to = fmaxf(m, sc);
        const float keep = m == to ? 1.f : exp2f(m - to), p = sc == to ? 1.f : exp2f(sc - to);
        l = l * keep + p;
#pragma unroll
        for (int e = 0; e < V; e++) acc[e] = fmaf(p, f32(a.vp[at + e]), acc[e] * keep);
        m = to;
    }
    if (lane == 0) {
        om[wave] = m;
        ol[wave] = l;
    }
#pragma unroll
    for (int e = 0; e < V; e++) oa[wave][lane * V + e] = acc[e];
    __syncthreads();
    float top = om[0];
#pragma unroll
    for (int w = 1; w < WAVES; w++) top = fmaxf(top, om[w]);
    float sum = 0.f, o[DH / THREADS + 1] = {};
    const int d = threadIdx.x;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        if (ol[w] == 0.f) continue;
        const float f = om[w] == top ? 1.f : exp2f(om[w] - top);
        sum += ol[w] * f;
        if (d < DH) o[0] += oa[w][d] * f;
    }
    if (d < DH) {
        float y = sum > 0.f || sum != sum ? o[0] / sum : 0.f;
        const size_t at = ((size_t)r * a.Hq + h) * DH + d;
        if (a.gate && sum != 0.f) y *= sigmoid(f32(a.gate[at]));
        a.out[at] = to_bf16(y);
    }
    if (a.lse && d == 0) a.lse[(size_t)h * a.B + r] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * LN2;
}

}  // namespace
}  // namespace q35

using namespace q35;

extern "C" void* cs1_attention_paged_create(void) {
    int device;
    if (hipGetDevice(&device) != hipSuccess) return nullptr;
    Paged* const p = new (std::nothrow) Paged;
    if (p) p->device = device;
    return p;
}

extern "C" void cs1_attention_paged_destroy(void* paged) { delete static_cast<Paged*>(paged); }

extern "C" int cs1_attention_paged(void* paged, const void* q, const void* kp, const void* vp, const Cs1PageTable* pages,
                                   const int32_t* seqs, const void* gate, void* out, float* lse, int B, int Hq, int Hk,
                                   int Dh, float scale, void* stream) {
    const Paged* const p = static_cast<const Paged*>(paged);
    if (!p || !table_ok(pages) || (Dh != 128 && Dh != 256) || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 || B < 0 ||
        (int64_t)B * Hq > (1 << 22))
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
    a.scale_log2 = scale * LOG2E;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (Dh == 128)
        attention_paged_kernel<128><<<B * Hq, THREADS, 0, st>>>(a);
    else
        attention_paged_kernel<256><<<B * Hq, THREADS, 0, st>>>(a);
    return hipGetLastError();
}
