// paged.hip - attention layers over a paged key-value cache: the norms and rotation that fill it
// (qk_rope_paged), the attention of one query row per token over its sequence's pages, and the
// layer block made of them.  The dense cache of one sequence is layer.hip's.
#include "paged.h"

#include <math.h>
#include <stdio.h>

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace coli {

static bool heads_view(const ColiHipPages *p, const ColiHipHeads *h, HeadsView &v) {
    if (!h) return paged_refuse("NULL heads");
    if (h->H < 1 || h->H % p->KH || h->H > 65536) return paged_refuse("query heads not a multiple of the kv heads");
    if (h->rot < 0 || h->rot > p->hd || h->rot % 2) return paged_refuse("rotary columns not even, or more than a head");
    if (h->rot && !h->freq) return paged_refuse("NULL inverse frequencies");
    if (h->q_head < p->hd || h->q_row < (h->H - 1) * h->q_head + p->hd || h->kv_row < (int64_t)p->KH * p->hd)
        return paged_refuse("rows that overlap");
    v.H = h->H, v.rot = h->rot, v.interleaved = h->interleaved != 0;
    v.q_row = h->q_row, v.q_head = h->q_head, v.kv_row = h->kv_row;
    v.eps = h->eps, v.mag = h->rope_mag, v.scale = h->scale;
    v.qn = h->qn, v.kn = h->kn, v.freq = h->freq;
    return true;
}

// ---------------------------------------------------------------- values of a page
template <int T>
struct Val;
template <>
struct Val<COLI_HIP_F32> {
    using type = float;
    static __device__ __forceinline__ float up(float x) { return x; }
    static __device__ __forceinline__ float down(float x) { return x; }
};
template <>
struct Val<COLI_HIP_F16> {
    using type = _Float16;
    static __device__ __forceinline__ float up(_Float16 x) { return (float)x; }
    static __device__ __forceinline__ _Float16 down(float x) { return (_Float16)x; }
};
template <>
struct Val<COLI_HIP_BF16> {
    using type = __bf16;
    static __device__ __forceinline__ float up(__bf16 x) { return (float)x; }
    static __device__ __forceinline__ __bf16 down(float x) { return (__bf16)x; }   // to nearest, ties to even
};

// ---------------------------------------------------------------- norms, rotation, pages
// y = x rsqrt(mean x^2 + eps) (1 + w), then the first rot columns turned by pos * freq[j].  The
// angle is taken in 64 bits (24-bit frequencies times positions of up to 31 bits are exact
// there) and reduced to a fraction of a turn before it becomes 32 bits.
// A wave per head row: block (n, j): j < H a query head, then KH key heads, then KH value rows.
template <int T>
__global__ __launch_bounds__(64) void qk_rope_rows(PoolView p, HeadsView h, int layer, const float *__restrict__ q,
                                                   const float *__restrict__ k, const float *__restrict__ v,
                                                   const int *__restrict__ seq, const int *__restrict__ pos,
                                                   float *__restrict__ qo) {
    using D = typename Val<T>::type;
    __shared__ float s_row[256];
    const int n = blockIdx.x, j = blockIdx.y, lane = threadIdx.x;
    int s;
    const int at = row_pos(p, seq, pos, n, s);
    if (s < 0 || at < 0) return;
    const int pg = p.table[(size_t)s * p.max_pages + at / p.page];
    if (j >= h.H && (pg < 0 || pg >= p.n_pages)) {
        if (lane == 0) atomicOr(&p.state[kStErr], kPgPage);
        return;
    }
    const bool isq = j < h.H, isv = j >= h.H + p.KH;
    const int kh = isv ? j - h.H - p.KH : j - h.H;
    const float *src = isq ? q + n * h.q_row + j * h.q_head : (isv ? v : k) + n * h.kv_row + (long)kh * p.hd;
    D *page = (D *)(p.data + (isq ? 0 : (size_t)pg * p.page_bytes + layer * p.layer_bytes + (isv ? p.kv_bytes : 0) +
                                            kh * p.head_bytes + (at % p.page) * p.row_bytes));
    if (isv) {
        for (int d = lane; d < p.hd; d += 64) page[d] = Val<T>::down(src[d]);
        return;
    }
    const float *w = isq ? h.qn : h.kn;
    float x[4], ss = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int d = lane + 64 * i;
        x[i] = d < p.hd ? src[d] : 0.f;
        ss += x[i] * x[i];
    }
    for (int o = 32; o; o >>= 1) ss += __shfl_xor(ss, o);
    const float r = w ? 1.f / sqrtf(ss / p.hd + h.eps) : 1.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int d = lane + 64 * i;
        if (d < p.hd) s_row[d] = w ? x[i] * r * (1.f + w[d]) : x[i];
    }
    __syncthreads();
    const int hr = h.rot / 2;
    for (int d = lane; d < p.hd; d += 64) {
        float o = s_row[d];
        if (d < h.rot) {
            const int jj = h.interleaved ? d / 2 : d < hr ? d : d - hr;
            const bool second = h.interleaved ? d & 1 : d >= hr;
            const float other = s_row[h.interleaved ? d ^ 1 : second ? d - hr : d + hr];
            const double x = (double)at * (double)h.freq[jj], c = 0.15915494309189535;   // c + lo = 1 / (2 pi)
            const double a = fma(x, c, -rint(x * c)) + x * -9.839338337591243e-18;   // a fraction of a turn
            float sn, cs;
            sincospif((float)(2.0 * a), &sn, &cs);
            sn *= h.mag, cs *= h.mag;
            o = second ? o * cs + other * sn : o * cs - other * sn;
        }
        if (isq)
            qo[((size_t)n * h.H + j) * p.hd + d] = o;
        else
            page[d] = Val<T>::down(o);
    }
}

static bool rows_args(const ColiHipPages *p, int layer, int n) {
    if (layer < 0 || layer >= p->n_layers) return paged_refuse("layer index");
    if (n < 0 || n > 1 << 24) return paged_refuse("row count");
    return true;
}

static bool rope_launch(const PoolView &pv, const HeadsView &hv, int dtype, int layer, const float *q, const float *k,
                        const float *v, const int *seq, const int *pos, int n, float *qo, hipStream_t st) {
    const dim3 grid(n, hv.H + 2 * pv.KH);
    switch (dtype) {
    case COLI_HIP_F32:
        hipLaunchKernelGGL(qk_rope_rows<COLI_HIP_F32>, grid, dim3(64), 0, st, pv, hv, layer, q, k, v, seq, pos, qo);
        break;
    case COLI_HIP_F16:
        hipLaunchKernelGGL(qk_rope_rows<COLI_HIP_F16>, grid, dim3(64), 0, st, pv, hv, layer, q, k, v, seq, pos, qo);
        break;
    default:
        hipLaunchKernelGGL(qk_rope_rows<COLI_HIP_BF16>, grid, dim3(64), 0, st, pv, hv, layer, q, k, v, seq, pos, qo);
    }
    return paged_launched("qk rope launch");
}

// ---------------------------------------------------------------- the layer block
enum { P_Q, P_K, P_V, P_QN, P_CTX, P_WORK, P_COUNT };
static struct {
    void *p = nullptr;
    size_t cap = 0;
} g_pw[P_COUNT];

void paged_shutdown() {
    for (auto &w : g_pw) scratch_free(&w.p, &w.cap);
}

__global__ __launch_bounds__(256) void fill_zero(float *x, size_t n) {
    const size_t i = blockIdx.x * (size_t)256 + threadIdx.x;
    if (i < n) x[i] = 0.f;
}

}  // namespace coli

using namespace coli;

COLI_API int coli_hip_heads_check(const ColiHipPages *p, const ColiHipHeads *h) {
    PoolView pv;
    HeadsView hv;
    return pool_view(p, pv) && heads_view(p, h, hv) ? 1 : 0;
}

COLI_API int coli_hip_qk_rope_paged(const ColiHipPages *p, const ColiHipHeads *h, int layer, const float *d_q,
                                    const float *d_k, const float *d_v, const int *d_seq, const int *d_pos, int n,
                                    float *d_qout, void *stream_) {
    PoolView pv;
    HeadsView hv;
    hipStream_t st;
    if (!pool_view(p, pv) || !heads_view(p, h, hv) || !rows_args(p, layer, n)) return 0;
    if (n && (!d_q || !d_k || !d_v || !d_seq || !d_qout)) return paged_refuse("NULL rows") ? 1 : 0;
    if (!paged_stream(stream_, st)) return 0;
    return !n || rope_launch(pv, hv, p->dtype, layer, d_q, d_k, d_v, d_seq, d_pos, n, d_qout, st) ? 1 : 0;
}

COLI_API size_t coli_hip_attn_paged_work(const ColiHipPages *p, const ColiHipHeads *h) {
    PoolView pv;
    HeadsView hv;
    return pool_view(p, pv) && heads_view(p, h, hv) ? attn_paged_work(pv) : 0;
}

COLI_API int coli_hip_attn_paged(const ColiHipPages *p, const ColiHipHeads *h, int layer, const float *d_q,
                                 const float *d_gate, const int *d_seq, const int *d_pos, int n, int max_len,
                                 float *d_out, void *d_work, size_t work_bytes, void *stream_) {
    PoolView pv;
    HeadsView hv;
    hipStream_t st;
    if (!pool_view(p, pv) || !heads_view(p, h, hv) || !rows_args(p, layer, n)) return 0;
    if (n && (!d_q || !d_seq || !d_out)) return paged_refuse("NULL rows") ? 1 : 0;
    if (n && (!d_work || (uintptr_t)d_work % 16 || work_bytes < coli_hip_attn_paged_work(p, h)))
        return paged_refuse("attention workspace missing, too small or not aligned to 16 bytes") ? 1 : 0;
    if (!paged_stream(stream_, st)) return 0;
    return !n || attn_paged(pv, hv, p->dtype, layer, d_q, d_gate, d_seq, d_pos, n, max_len, d_out, d_work, st) ? 1 : 0;
}

COLI_API int coli_hip_gqa_paged(const ColiHipPages *p, const ColiHipHeads *h, int layer, const float *d_x, int D,
                                const ColiVkTensor *gq_t, const ColiVkTensor *gk_t, const ColiVkTensor *gv_t,
                                const ColiVkTensor *out_t, const int *d_seq, const int *d_pos, int n, int max_len,
                                float *d_out, void *stream_) {
    PoolView pv;
    HeadsView hv;
    hipStream_t st;
    if (!pool_view(p, pv) || !h || !rows_args(p, layer, n)) return 0;
    if (n && (!d_x || !d_seq || !d_out)) return paged_refuse("NULL rows") ? 1 : 0;
    const int hd = pv.hd, KH = pv.KH;
    if (!tensor_live(gq_t) || !tensor_live(gk_t) || !tensor_live(gv_t) || !tensor_live(out_t) || gq_t->I != D ||
        gk_t->I != D || gv_t->I != D || gk_t->O != KH * hd || gv_t->O != KH * hd || out_t->I != h->H * hd ||
        (gq_t->O != h->H * hd && gq_t->O != 2 * h->H * hd))
        return paged_refuse("projection shapes") ? 1 : 0;
    const bool gated = gq_t->O == 2 * h->H * hd;
    ColiHipHeads own = *h;   // the rows are the projections' here
    own.q_head = gated ? 2 * hd : hd;
    own.q_row = gq_t->O;
    own.kv_row = (int64_t)KH * hd;
    if (!heads_view(p, &own, hv) || !paged_stream(stream_, st)) return 0;
    if (!n) return 1;
    const size_t rows = n, need[P_COUNT] = {rows * gq_t->O * 4,       rows * KH * hd * 4,     rows * KH * hd * 4,
                                            rows * h->H * hd * 4,     rows * h->H * hd * 4,
                                            coli_hip_attn_paged_work(p, &own)};
    for (int i = 0; i < P_COUNT; i++)
        if (!scratch(&g_pw[i].p, &g_pw[i].cap, need[i])) return 0;
    float *q = (float *)g_pw[P_Q].p, *k = (float *)g_pw[P_K].p, *v = (float *)g_pw[P_V].p;
    float *qn = (float *)g_pw[P_QN].p, *ctx = (float *)g_pw[P_CTX].p;
    if (!gemv(gq_t, d_x, q, n, st) || !gemv(gk_t, d_x, k, n, st) || !gemv(gv_t, d_x, v, n, st)) return 0;
    // a row without a sequence: no attention writes its context
    const size_t nc = rows * h->H * hd;
    hipLaunchKernelGGL(fill_zero, dim3((unsigned)((nc + 255) / 256)), dim3(256), 0, st, ctx, nc);
    if (!rope_launch(pv, hv, p->dtype, layer, q, k, v, d_seq, d_pos, n, qn, st) ||
        !attn_paged(pv, hv, p->dtype, layer, qn, gated ? q + hd : nullptr, d_seq, d_pos, n, max_len, ctx,
                     g_pw[P_WORK].p, st))
        return 0;
    return gemv(out_t, ctx, d_out, n, st) ? 1 : 0;
}
