// paged.hip - attention layers over a paged key-value cache: the norms and rotation that fill it
// (qk_rope_paged), the attention of one query row per token over its sequence's pages, and the
// layer block made of them.  The dense cache of one sequence is layer.hip's.
#include "paged.h"

#include <math.h>
#include <stdio.h>

namespace coli {

static bool heads_view(const ColiHipPages *p, const ColiHipHeads *h, HeadsView &v) {
    if (!h) return paged_refuse("NULL heads");
    if (h->H < 1 || h->H % p->KH || h->H > 4096) return paged_refuse("query heads not a multiple of the kv heads");
    if (h->rot < 0 || h->rot > p->hd || h->rot % 2) return paged_refuse("rotary columns not even, or more than a head");
    if (h->rot && !h->freq) return paged_refuse("NULL inverse frequencies");
    constexpr int64_t kFar = (int64_t)1 << 40;   // times rows or heads: within 63 bits
    if (h->q_head > kFar || h->q_row > kFar || h->kv_row > kFar) return paged_refuse("row stride past 2^40");
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
    static __device__ __forceinline__ float down(float x) { return x; }
};
template <>
struct Val<COLI_HIP_F16> {
    using type = _Float16;
    static __device__ __forceinline__ _Float16 down(float x) { return (_Float16)x; }
};
template <>
struct Val<COLI_HIP_BF16> {
    using type = __bf16;
    static __device__ __forceinline__ __bf16 down(float x) { return (__bf16)x; }   // to nearest, ties to even
};

// ---------------------------------------------------------------- norms, rotation, pages
// y = x rsqrt(mean x^2 + eps) (1 + w), then the first rot columns turned by pos * freq[j].  The
// angle is taken in 64 bits (24-bit frequencies times positions of up to 29 bits are exact
// there) and reduced to a fraction of a turn before it becomes 32 bits.
//
// Bound by its bytes (q in and out, k and v in, the pages' rows out) where there are many rows,
// by a launch and three dependent loads (sequence, length, page) where there are few.  A row is
// LP lanes of four columns each, so a wave has 64 / LP rows (query heads, then key heads, then
// values) at a time and takes more of the same token: the sines and cosines (one pair a lane) and its columns' norm weights
// are found once.  4005 rows of 32 + 8 heads of 128, all columns turned, f16 pages: 39 us,
// 4.6 TB/s; a wave per row with its own sines took 111.  192 rows of 16 + 2 heads of 256: 6 us.
constexpr int kRopeWaves = 4;
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4u4 __attribute__((ext_vector_type(4), aligned(4)));   // rows need not be aligned
template <int T, int LP>
__global__ __launch_bounds__(64 * kRopeWaves) void qk_rope_rows(PoolView p, HeadsView h, int layer,
                                                                const float *__restrict__ q, const float *__restrict__ k,
                                                                const float *__restrict__ v, const int *__restrict__ seq,
                                                                const int *__restrict__ pos, float *__restrict__ qo) {
    using D = typename Val<T>::type;
    typedef D v4d __attribute__((ext_vector_type(4)));
    constexpr int kRows = 64 / LP;
    __shared__ __attribute__((aligned(16))) float s_x[kRopeWaves][256];
    __shared__ float2 s_turn[kRopeWaves][128];
    const int n = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, sub = lane / LP, d0 = lane % LP * 4;
    const int rows = h.H + 2 * p.KH, hr = h.rot / 2;
    const bool in = d0 < p.hd;
    int j0 = (blockIdx.y * kRopeWaves + wave) * kRows;
    const int step = gridDim.y * kRopeWaves * kRows;
    auto source = [&](int j) {
        return j < h.H ? q + n * h.q_row + j * h.q_head
                       : (j < h.H + p.KH ? k : v - (long)p.KH * p.hd) + n * h.kv_row + (long)(j - h.H) * p.hd;
    };
    auto load = [&](int j) -> v4f {
        if (!in || j >= rows) return v4f{0.f, 0.f, 0.f, 0.f};
        return *(const v4u4 *)(source(j) + d0);
    };
    v4f x = load(j0 + sub);
    v4f wq = {0.f, 0.f, 0.f, 0.f}, wk = wq;
    if (in && h.qn) wq = *(const v4u4 *)(h.qn + d0);
    if (in && h.kn) wk = *(const v4u4 *)(h.kn + d0);
    // the frequencies of pairs lane and lane + 64
    float fr[2];
#pragma unroll
    for (int i = 0; i < 2; i++) fr[i] = lane + 64 * i < hr ? h.freq[lane + 64 * i] : 0.f;
    int s;
    const int at = row_pos<true>(p, seq, pos, n, s);
    if (s < 0 || at < 0) return;
    const int pj = at / p.page, slot = at - pj * p.page;
    const int pg = p.table[(size_t)s * p.max_pages + pj];
    const bool bad = pg < 0 || pg >= p.n_pages;
    if (bad && threadIdx.x == 0) atomicOr(&p.state[kStErr], kPgPage);
    char *page = p.data + (bad ? 0 : (size_t)pg * p.page_bytes) + layer * p.layer_bytes + slot * p.row_bytes;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if (64 * i >= hr) break;
        const double t = (double)at * (double)fr[i], c = 0.15915494309189535;   // c + lo = 1 / (2 pi)
        const double a = fma(t, c, -rint(t * c)) + t * -9.839338337591243e-18;  // a fraction of a turn
        float sn, cs;
        sincospif((float)(2.0 * a), &sn, &cs);
        s_turn[wave][lane + 64 * i] = make_float2(cs * h.mag, sn * h.mag);
    }
    wave_sync();
    float cs[4], sn[4];
    bool second[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {   // the column's pair, and which of the two it is
        const int d = d0 + i;
        second[i] = h.interleaved ? d & 1 : d >= hr;
        const float2 t = s_turn[wave][d >= h.rot ? 0 : h.interleaved ? d / 2 : second[i] ? d - hr : d];
        cs[i] = t.x;
        sn[i] = second[i] ? t.y : -t.y;   // (u, v) -> (u cos - v sin, v cos + u sin)
    }
    for (; j0 < rows; j0 += step) {
        const int j = j0 + sub;
        const v4f next = load(j + step);
        const bool isq = j < h.H, isv = j >= h.H + p.KH, live = in && j < rows;
        float ss = (x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3]);
#pragma unroll
        for (int o = LP / 2; o; o >>= 1) ss += __shfl_xor(ss, o);
        const float *w = isq ? h.qn : h.kn;
        v4f y = x;
        if (w) {
            const float r = 1.f / sqrtf(ss / p.hd + h.eps);
            const v4f wv = isq ? wq : wk;
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = x[i] * r * (1.f + wv[i]);
        }
        v4f o = y;
        if (h.interleaved) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (d0 + i < h.rot) o[i] = y[i] * cs[i] + y[i ^ 1] * sn[i];
        } else if (h.rot) {   // the other half's columns are other lanes' of this wave
            float *row = s_x[wave] + sub * 4 * LP;
            *(v4f *)(row + d0) = y;
            wave_sync();
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = d0 + i;
                if (d < h.rot) o[i] = y[i] * cs[i] + row[second[i] ? d - hr : d + hr] * sn[i];
            }
            wave_sync();
        }
        if (isv) o = x;
        if (live && isq) {
            *(v4u4 *)(qo + ((size_t)n * h.H + j) * p.hd + d0) = o;
        } else if (live && !bad) {
            v4d r;
#pragma unroll
            for (int i = 0; i < 4; i++) r[i] = Val<T>::down(o[i]);
            const int kh = isv ? j - h.H - p.KH : j - h.H;
            *(v4d *)(page + (isv ? p.kv_bytes : 0) + kh * p.head_bytes + d0 * sizeof(D)) = r;
        }
        x = next;
    }
}

static bool rows_args(const ColiHipPages *p, int layer, int n) {
    if (layer < 0 || layer >= p->n_layers) return paged_refuse("layer index");
    if (n < 0 || n > 1 << 20) return paged_refuse("row count not in 0..2^20");
    return true;
}

template <int T>
static void rope_rows(const PoolView &pv, const HeadsView &hv, int layer, const float *q, const float *k, const float *v,
                      const int *seq, const int *pos, int n, float *qo, hipStream_t st) {
    const int lp = pv.hd <= 64 ? 16 : pv.hd <= 128 ? 32 : 64, per = kRopeWaves * (64 / lp);
    // few tokens: a wave per row; many: the waves of one block take a token's rows in turn
    const long all = (hv.H + 2 * pv.KH + per - 1) / per, want = (2048 + n - 1) / n;
    const dim3 grid(n, (unsigned)(all < want ? all : want)), t(64 * kRopeWaves);
    if (lp == 16)
        hipLaunchKernelGGL((qk_rope_rows<T, 16>), grid, t, 0, st, pv, hv, layer, q, k, v, seq, pos, qo);
    else if (lp == 32)
        hipLaunchKernelGGL((qk_rope_rows<T, 32>), grid, t, 0, st, pv, hv, layer, q, k, v, seq, pos, qo);
    else
        hipLaunchKernelGGL((qk_rope_rows<T, 64>), grid, t, 0, st, pv, hv, layer, q, k, v, seq, pos, qo);
}

static bool rope_launch(const PoolView &pv, const HeadsView &hv, int dtype, int layer, const float *q, const float *k,
                        const float *v, const int *seq, const int *pos, int n, float *qo, hipStream_t st) {
    switch (dtype) {
    case COLI_HIP_F32: rope_rows<COLI_HIP_F32>(pv, hv, layer, q, k, v, seq, pos, n, qo, st); break;
    case COLI_HIP_F16: rope_rows<COLI_HIP_F16>(pv, hv, layer, q, k, v, seq, pos, n, qo, st); break;
    default: rope_rows<COLI_HIP_BF16>(pv, hv, layer, q, k, v, seq, pos, n, qo, st);
    }
    return paged_launched("qk rope launch");
}

// ---------------------------------------------------------------- the layer block
enum { P_Q, P_K, P_V, P_QN, P_CTX, P_SEQ, P_WORK, P_COUNT };
static struct {
    void *p = nullptr;
    size_t cap = 0;
} g_pw[P_COUNT];

void paged_shutdown() {
    for (auto &w : g_pw) scratch_free(&w.p, &w.cap);
}

// The context cleared (nc floats), and the rows that attend: those at a position which is held, so
// that the rotation has written their query; others get sequence -1 and keep the zeros.
__global__ __launch_bounds__(256) void block_rows(PoolView p, const int *__restrict__ seq, const int *__restrict__ pos,
                                                  int n, int *__restrict__ live, float *__restrict__ ctx, size_t nc) {
    const size_t i0 = blockIdx.x * (size_t)256 + threadIdx.x, step = gridDim.x * (size_t)256;
    for (size_t i = i0; i < nc; i += step) ctx[i] = 0.f;
    for (size_t i = i0; i < (size_t)n; i += step) {
        int s;
        live[i] = row_pos<true>(p, seq, pos, (int)i, s) < 0 ? -1 : s;
    }
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
    if ((uintptr_t)d_out % 16) return paged_refuse("attention output not aligned to 16 bytes") ? 1 : 0;
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
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(st, &cap) != hipSuccess || cap != hipStreamCaptureStatusNone)
        return paged_refuse("the layer block in a captured stream (its scratch may grow)") ? 1 : 0;
    const size_t rows = n, need[P_COUNT] = {rows * gq_t->O * 4,       rows * KH * hd * 4,     rows * KH * hd * 4,
                                            rows * h->H * hd * 4,     rows * h->H * hd * 4,   rows * 4,
                                            coli_hip_attn_paged_work(p, &own)};
    for (int i = 0; i < P_COUNT; i++)
        if (!scratch(&g_pw[i].p, &g_pw[i].cap, need[i])) return 0;
    float *q = (float *)g_pw[P_Q].p, *k = (float *)g_pw[P_K].p, *v = (float *)g_pw[P_V].p;
    float *qn = (float *)g_pw[P_QN].p, *ctx = (float *)g_pw[P_CTX].p;
    if (!gemv(gq_t, d_x, q, n, st) || !gemv(gk_t, d_x, k, n, st) || !gemv(gv_t, d_x, v, n, st)) return 0;
    int *live = (int *)g_pw[P_SEQ].p;
    const size_t nc = rows * h->H * hd, nb = (nc + 255) / 256;   // more than the rows
    hipLaunchKernelGGL(block_rows, dim3((unsigned)(nb < 65536 ? nb : 65536)), dim3(256), 0, st, pv, d_seq, d_pos, n, live,
                       ctx, nc);
    if (!paged_launched("paged layer rows") ||
        !rope_launch(pv, hv, p->dtype, layer, q, k, v, d_seq, d_pos, n, qn, st) ||
        !attn_paged(pv, hv, p->dtype, layer, qn, gated ? q + hd : nullptr, live, d_pos, n, max_len, ctx,
                     g_pw[P_WORK].p, st))
        return 0;
    return gemv(out_t, ctx, d_out, n, st) ? 1 : 0;
}
