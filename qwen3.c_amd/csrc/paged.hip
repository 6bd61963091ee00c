// paged.hip - attention layers over a paged key-value cache: the norms and rotation that fill it
// (qk_rope_paged), the attention of one query row per token over its sequence's pages, and the
// layer block made of them.  The dense cache of one sequence is layer.hip's.
#include "paged.h"

#include <math.h>
#include <stdio.h>

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace coli {

// ColiHipHeads as the kernels take it.
struct HeadsView {
    int H, rot, interleaved;
    long q_row, q_head, kv_row;
    float eps, mag, scale;
    const float *qn, *kn, *freq;
};

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

static bool launched(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess || fail(what, e);
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

// The last position that row n sees (-1: none), and its sequence (-1: no row).
__device__ __forceinline__ int row_pos(const PoolView &p, const int *seq, const int *pos, int n, int &s) {
    s = seq[n];
    if (s < 0 || s >= p.n_seqs) {
        if (s != -1) atomicOr(&p.state[kStErr], kPgIndex);
        s = -1;
        return -1;
    }
    const int len = min(max(p.lens[s], 0), p.max_pages * p.page), at = pos ? pos[n] : len - 1;
    if (at < len && at >= -1) return at;
    atomicOr(&p.state[kStErr], at < -1 ? kPgIndex : kPgPos);
    return at < -1 ? -2 : -3 - len;   // -2: no position; -3 - len: past the end
}

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

// ---------------------------------------------------------------- attention over pages
// o = sum_t softmax_t(scale q . k_t) v_t over t <= pos, one pass with a running maximum m and
// sum l per head (scores in units of log 2, the scale and log2 e folded into q).
//
// The products run on v_mfma_f32_16x16x4_f32 with the pages' values widened to 32 bits (exact), a
// wave on 16 keys of one kv head and up to 16 of its query heads at a time:
//   scores [key][head] = K q^T: A[key l % 16][k = l / 16], one 16-byte load of the lane's key row
//     is the operand of 4 (f32) or 8 products; lane l ends up with keys 4 (l / 16) + i of head
//     l % 16.
//   out [head][column] += P V: the lane's own weight i is A[head l % 16][k = l / 16] for key
//     4 k + i; B[k][column] is the lane's 16-byte piece of that key's row, so product n of a
//     piece covers columns n, n + 8, ..: no transpose, no LDS but for q.
//
// Work: row r's unit is kKeys keys of a kv head, kWaves tiles side by side; the units of all rows
// in one line are cut into equal shares, one per block, whatever the lengths are.  A block's part
// of a (row, kv head) that it does not hold whole goes to the workspace, and attn_join puts the
// parts together.
constexpr int kTile = 16, kWaves = 4, kKeys = kTile * kWaves, kGroup = 16;   // kGroup: heads a wave takes
constexpr int kAttnBlocks = 512;   // two blocks per CU
constexpr int kAttnThreads = 64 * kWaves;
constexpr float kLazy = 8.f;   // the maximum is moved when a score passes it by 2^8: weights stay below

typedef float v4f __attribute__((ext_vector_type(4)));

struct PagedArgs {
    const float *q, *gate;
    const int *seq, *pos;
    float *out, *part;
    float2 *ml;
    int n, layer, groups, khv;   // head groups of kGroup per kv head, khv = KH * groups
    unsigned magic, shift;       // t / page = (umulhi(t, magic) + t) >> shift, t < 2^31
};

// The positions that row r sees (a row of no sequence: -1).
__device__ __forceinline__ int row_count(const PoolView &p, const PagedArgs &a, int r, int &s) {
    const int at = row_pos(p, a.seq, a.pos, r, s);
    return s < 0 ? -1 : at < -2 ? -3 - at : at < 0 ? 0 : at + 1;   // past the end: what is held
}
__device__ __forceinline__ int chunks_of(int cnt) { return cnt < 1 ? cnt + 1 : (int)(((unsigned)cnt + kKeys - 1) / kKeys); }

// The units of all rows in one line.  s_base[t]: the units before the rows of thread t.
struct Line {
    long total, share;
    int per;
};
__device__ __forceinline__ Line line_up(const PoolView &p, const PagedArgs &a, int nblocks, long *s_base, long *s_wave) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    Line l;
    l.per = (a.n + kAttnThreads - 1) / kAttnThreads;
    long mine = 0;
    for (int i = 0; i < l.per; i++) {
        const int r = tid * l.per + i;
        int s;
        if (r < a.n) mine += (long)chunks_of(row_count(p, a, r, s)) * a.khv;
    }
    long x = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    if (lane == 63) s_wave[wave] = x;
    __syncthreads();
    long before = 0;
    l.total = 0;
    for (int w = 0; w < kWaves; w++) {
        before += w < wave ? s_wave[w] : 0;
        l.total += s_wave[w];
    }
    s_base[tid] = before + x - mine;
    l.share = (l.total + nblocks - 1) / nblocks;
    if (l.share < 1) l.share = 1;
    __syncthreads();
    return l;
}
// The row of unit u < total: r, its first unit.
__device__ __forceinline__ int row_of(const PoolView &p, const PagedArgs &a, const Line &l, const long *s_base, long u,
                                      long &first) {
    int lo = 0, hi = kAttnThreads;
    while (hi - lo > 1) {
        const int m = (lo + hi) / 2;
        if (s_base[m] <= u)
            lo = m;
        else
            hi = m;
    }
    int r = lo * l.per;
    first = s_base[lo];
    for (; r < a.n; r++) {
        int s;
        const long k = (long)chunks_of(row_count(p, a, r, s)) * a.khv;
        if (first + k > u) break;
        first += k;
    }
    return r;   // n only if the lengths change under the kernel
}

template <int T>
__device__ __forceinline__ void widen(const uint4 &x, float *f) {
    const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (T == COLI_HIP_F32) {
            f[i] = __uint_as_float(w[i]);
        } else if (T == COLI_HIP_BF16) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            f[2 * i] = (float)__builtin_bit_cast(_Float16, (unsigned short)w[i]);
            f[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (unsigned short)(w[i] >> 16));
        }
    }
}

// max / sum over the four lanes that hold a head's keys (l, l ^ 16, l ^ 32, l ^ 48)
__device__ __forceinline__ float max4(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum4(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

template <int T, int HD, bool kExact>
__global__ __launch_bounds__(kAttnThreads, 2) void attn_part(PoolView p, HeadsView h, PagedArgs a) {
    constexpr int kE = T == COLI_HIP_F32 ? 4 : 8;          // values of a 16-byte piece
    constexpr int kKC = HD / (4 * kE), kVS = HD / (16 * kE) < 1 ? 1 : HD / (16 * kE);
    constexpr int kQ = HD + 4;                             // row of q in LDS
    __shared__ long s_base[kAttnThreads], s_wave[kWaves];
    __shared__ float s_q[kGroup * kQ];
    __shared__ float s_m[kWaves][kGroup], s_l[kWaves][kGroup];
    __shared__ float s_o[2][kVS * kE * 256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
    const int G = h.H / p.KH, pieces = (int)(p.row_bytes / 16);
    const Line ln = line_up(p, a, gridDim.x, s_base, s_wave);
    const long u0 = blockIdx.x * ln.share, end = min(ln.total, u0 + ln.share);
    if (u0 >= end) return;
    long first;
    int r = row_of(p, a, ln, s_base, u0, first);
    for (long u = u0; u < end && r < a.n;) {
        int s;
        const int cnt = row_count(p, a, r, s), nc = chunks_of(cnt);
        const long x = u - first;
        if (x >= (long)nc * a.khv) {   // this row is done (or has none)
            first += (long)nc * a.khv;
            r++;
            continue;
        }
        const int hv = (int)(x / nc), c0 = (int)(x % nc), c1 = (int)min((long)nc, c0 + (end - u));
        const int kh = hv / a.groups, h0 = (hv % a.groups) * kGroup, hn = min(kGroup, G - h0);
        const long head = (long)kh * G + h0;   // first query head
        // q, scaled, zero past the last head and column
        const float *q = a.q + ((long)r * h.H + head) * p.hd;
        const float qs = h.scale * 1.4426950408889634f;
        for (int i = tid; i < kGroup * HD; i += kAttnThreads) {
            const int hh = i / HD, d = i % HD;
            s_q[hh * kQ + d] = hh < hn && (kExact || d < p.hd) ? q[hh * p.hd + d] * qs : 0.f;
        }
        __syncthreads();
        v4f acc[kVS * kE];
#pragma unroll
        for (int i = 0; i < kVS * kE; i++) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        const int *row = p.table + (size_t)s * p.max_pages;
        const char *base = p.data + (size_t)a.layer * p.layer_bytes + (size_t)kh * p.head_bytes;
        const int last = min(cnt, c1 * kKeys);
        // the lane's key of a tile: its page, then where its row lies
        auto page_id = [&](int key0) {
            const unsigned t = (unsigned)min(key0 + c, cnt - 1);
            return row[(__umulhi(t, a.magic) + t) >> a.shift];
        };
        auto locate = [&](int key0, int pg, long &off) {
            const unsigned t = (unsigned)min(key0 + c, cnt - 1), j = (__umulhi(t, a.magic) + t) >> a.shift;
            const bool is = pg >= 0 && pg < p.n_pages;
            if (!is && key0 + c < cnt) atomicOr(&p.state[kStErr], kPgPage);
            off = (is ? (long)pg * p.page_bytes : 0) + (long)(t - j * p.page) * p.row_bytes;
            return is && key0 + c < cnt;
        };
        uint4 kb[kKC], vb[4][kVS];
        auto load_k = [&](long off) {
            const uint4 *k = (const uint4 *)(base + off) + g;
#pragma unroll
            for (int i = 0; i < kKC; i++) {
                kb[i] = uint4{0, 0, 0, 0};
                if (kExact || 4 * i + g < pieces) kb[i] = k[4 * i];
            }
        };
        auto load_v = [&](long off) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const long o = __shfl(off, 4 * g + j);
                const uint4 *v = (const uint4 *)(base + p.kv_bytes + o) + c;
#pragma unroll
                for (int i = 0; i < kVS; i++) {
                    vb[j][i] = uint4{0, 0, 0, 0};
                    if ((kExact && HD >= 16 * kE) || 16 * i + c < pieces) vb[j][i] = v[16 * i];
                }
            }
        };
        int key0 = c0 * kKeys + wave * kTile;
        long off = 0, off_next = 0;
        bool valid = false, valid_next = false;
        int pg_next = 0;
        if (key0 < last) {
            valid = locate(key0, page_id(key0), off);
            load_k(off);
            load_v(off);
            if (key0 + kKeys < last) pg_next = page_id(key0 + kKeys);
        }
        for (; key0 < last; key0 += kKeys) {
            const bool more = key0 + kKeys < last;
            const unsigned vm = (unsigned)(__ballot(valid) & 0xffff);
            v4f sc = {0.f, 0.f, 0.f, 0.f}, sd = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kKC; i++) {
                float kf[8];
                widen<T>(kb[i], kf);
                const float *qp = s_q + c * kQ + (4 * i + g) * kE;
                float qf[kE];
#pragma unroll
                for (int j = 0; j < kE; j += 4) *(float4 *)(qf + j) = *(const float4 *)(qp + j);
#pragma unroll
                for (int j = 0; j < kE; j += 2) {
                    sc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j], qf[j], sc, 0, 0, 0);
                    sd = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j + 1], qf[j + 1], sd, 0, 0, 0);
                }
            }
            if (more) {
                valid_next = locate(key0 + kKeys, pg_next, off_next);
                load_k(off_next);
                if (key0 + 2 * kKeys < last) pg_next = page_id(key0 + 2 * kKeys);
            }
            sc += sd;
            if (vm != 0xffff) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (vm >> (4 * g + i) & 1) continue;
                    sc[i] = -INFINITY;
#pragma unroll
                    for (int j = 0; j < kVS; j++) vb[i][j] = uint4{0, 0, 0, 0};
                }
            }
            const float mt = max4(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])));
            if (__any(mt > m + kLazy || (m == -INFINITY && mt > m))) {
                const float nm = fmaxf(m, mt), f = m == nm ? 1.f : __builtin_amdgcn_exp2f(m - nm);
                l *= f;
                m = nm;
                float fr[4];
#pragma unroll
                for (int i = 0; i < 4; i++) fr[i] = __shfl(f, 4 * g + i);
#pragma unroll
                for (int t = 0; t < kVS * kE; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[t][i] *= fr[i];
            }
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = sc[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sc[i] - m);
            l += (w[0] + w[1]) + (w[2] + w[3]);
#pragma unroll
            for (int j = 0; j < 4; j++) {
#pragma unroll
                for (int i = 0; i < kVS; i++) {
                    float vf[8];
                    widen<T>(vb[j][i], vf);
#pragma unroll
                    for (int e = 0; e < kE; e++)
                        acc[i * kE + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[j], vf[e], acc[i * kE + e], 0, 0, 0);
                }
            }
            if (more) {
                load_v(off_next);
                off = off_next;
                valid = valid_next;
            }
        }
        // the four waves' parts: one maximum, then the sums pairwise through LDS
        l = sum4(l);
        if (g == 0) {
            s_m[wave][c] = m;
            s_l[wave][c] = l;
        }
        __syncthreads();
        float M[4], f[4], L[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int hh = 4 * g + i;
            M[i] = fmaxf(fmaxf(s_m[0][hh], s_m[1][hh]), fmaxf(s_m[2][hh], s_m[3][hh]));
            L[i] = 0.f;
            for (int w = 0; w < kWaves; w++) {
                const float mw = s_m[w][hh], fw = mw == M[i] ? 1.f : __builtin_amdgcn_exp2f(mw - M[i]);
                L[i] += s_l[w][hh] * fw;
                if (w == wave) f[i] = fw;
            }
        }
#pragma unroll
        for (int t = 0; t < kVS * kE; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[t][i] *= f[i];
#pragma unroll
        for (int step = 2; step; step >>= 1) {
            if (wave >= step && wave < 2 * step) {
#pragma unroll
                for (int t = 0; t < kVS * kE; t++) *(v4f *)&s_o[wave - step][(t * 64 + lane) * 4] = acc[t];
            }
            __syncthreads();
            if (wave < step) {
#pragma unroll
                for (int t = 0; t < kVS * kE; t++) acc[t] += *(const v4f *)&s_o[wave][(t * 64 + lane) * 4];
            }
            __syncthreads();
        }
        if (wave == 0) {
            const bool whole = c0 == 0 && c1 == nc;
            const long slot = 2L * blockIdx.x + (u == u0 ? 0 : 1);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int hh = 4 * g + i;
                if (hh >= hn) continue;
                float *dst = whole ? a.out + ((long)r * h.H + head + hh) * p.hd : a.part + (slot * kGroup + hh) * p.hd;
                const float *gt = a.gate ? a.gate + r * h.q_row + (head + hh) * h.q_head : nullptr;
                const float inv = cnt ? 1.f / L[i] : 0.f;
                if (!whole && c == 0) a.ml[slot * kGroup + hh] = make_float2(M[i], L[i]);
#pragma unroll
                for (int j = 0; j < kVS; j++) {
                    if (!(kExact && HD >= 16 * kE) && 16 * j + c >= pieces) continue;
                    float o[kE];
                    const int d0 = (16 * j + c) * kE;
#pragma unroll
                    for (int e = 0; e < kE; e++) {
                        o[e] = acc[j * kE + e][i];
                        if (whole) {
                            o[e] = cnt ? o[e] * inv : 0.f;
                            if (gt) o[e] /= 1.f + expf(-gt[d0 + e]);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < kE; e += 4) *(float4 *)(dst + d0 + e) = *(const float4 *)(o + e);
                }
            }
        }
        u += c1 - c0;
    }
}

// Block (j, hh): the (row, kv head) that the border between blocks j and j + 1 of attn_part
// cuts, when it is the first border inside it: head hh of its parts joined.
__global__ __launch_bounds__(kAttnThreads) void attn_join(PoolView p, HeadsView h, PagedArgs a, int nblocks) {
    __shared__ long s_base[kAttnThreads], s_wave[kWaves];
    const Line ln = line_up(p, a, nblocks, s_base, s_wave);
    const long u = (blockIdx.x + 1L) * ln.share;
    if (u >= ln.total) return;
    long first;
    const int r = row_of(p, a, ln, s_base, u, first);
    if (r >= a.n) return;
    int s;
    const int nc = chunks_of(row_count(p, a, r, s)), G = h.H / p.KH;
    const int hv = (int)((u - first) / nc), hh = blockIdx.y;
    const long from = first + (long)hv * nc, to = from + nc;   // its units
    if (from == u || from < u - ln.share) return;              // not cut here, or cut before
    const int h0 = (hv % a.groups) * kGroup;
    if (hh >= min(kGroup, G - h0)) return;
    const long head = (long)(hv / a.groups) * G + h0 + hh;
    const long b0 = from / ln.share, b1 = (to - 1) / ln.share;
    auto slot_of = [&](long b) { return (2 * b + (from <= b * ln.share ? 0 : 1)) * kGroup + hh; };
    float M = -INFINITY, L = 0.f;
    for (long b = b0; b <= b1; b++) M = fmaxf(M, a.ml[slot_of(b)].x);
    const int d = threadIdx.x;
    float o = 0.f;
    for (long b = b0; b <= b1; b++) {
        const float2 ml = a.ml[slot_of(b)];
        const float f = ml.x == M ? 1.f : __builtin_amdgcn_exp2f(ml.x - M);
        L += f * ml.y;
        if (d < p.hd) o += f * a.part[slot_of(b) * p.hd + d];
    }
    if (d >= p.hd) return;
    o /= L;
    if (a.gate) o /= 1.f + expf(-a.gate[r * h.q_row + head * h.q_head + d]);
    a.out[((long)r * h.H + head) * p.hd + d] = o;
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
    return launched("qk rope launch");
}

static size_t attn_work(const PoolView &pv) {
    return 2 * (size_t)kAttnBlocks * kGroup * (pv.hd * sizeof(float) + sizeof(float2));
}

template <int T>
static void attn_launch_t(const PoolView &pv, const HeadsView &hv, const PagedArgs &a, int blocks, hipStream_t st) {
    const dim3 g(blocks), t(kAttnThreads);
    switch (pv.hd) {
    case 64: hipLaunchKernelGGL((attn_part<T, 64, true>), g, t, 0, st, pv, hv, a); return;
    case 128: hipLaunchKernelGGL((attn_part<T, 128, true>), g, t, 0, st, pv, hv, a); return;
    case 256: hipLaunchKernelGGL((attn_part<T, 256, true>), g, t, 0, st, pv, hv, a); return;
    }
    if (pv.hd < 64)
        hipLaunchKernelGGL((attn_part<T, 64, false>), g, t, 0, st, pv, hv, a);
    else if (pv.hd < 128)
        hipLaunchKernelGGL((attn_part<T, 128, false>), g, t, 0, st, pv, hv, a);
    else
        hipLaunchKernelGGL((attn_part<T, 256, false>), g, t, 0, st, pv, hv, a);
}

static bool attn_launch(const PoolView &pv, const HeadsView &hv, int dtype, int layer, const float *q,
                        const float *gate, const int *seq, const int *pos, int n, int max_len, float *out, void *work,
                        hipStream_t st) {
    PagedArgs a;
    a.q = q, a.gate = gate, a.seq = seq, a.pos = pos, a.out = out, a.n = n, a.layer = layer;
    a.part = (float *)work;
    a.ml = (float2 *)(a.part + 2 * (size_t)kAttnBlocks * kGroup * pv.hd);
    const int G = hv.H / pv.KH;
    a.groups = (G + kGroup - 1) / kGroup;
    a.khv = pv.KH * a.groups;
    a.shift = 0;
    while ((1L << a.shift) < pv.page) a.shift++;
    a.magic = (unsigned)(((1ULL << 32) * ((1ULL << a.shift) - pv.page)) / pv.page + 1);
    const long cap = (long)pv.max_pages * pv.page, units = ((cap + kKeys - 1) / kKeys) * a.khv * (long)n;
    const int blocks = (int)(units < kAttnBlocks ? units : kAttnBlocks);
    switch (dtype) {
    case COLI_HIP_F32: attn_launch_t<COLI_HIP_F32>(pv, hv, a, blocks, st); break;
    case COLI_HIP_F16: attn_launch_t<COLI_HIP_F16>(pv, hv, a, blocks, st); break;
    default: attn_launch_t<COLI_HIP_BF16>(pv, hv, a, blocks, st);
    }
    if (blocks > 1)
        hipLaunchKernelGGL(attn_join, dim3(blocks - 1, G < kGroup ? G : kGroup), dim3(kAttnThreads), 0, st, pv, hv, a,
                           blocks);
    return launched("paged attention launch");
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
    return pool_view(p, pv) && heads_view(p, h, hv) ? attn_work(pv) : 0;
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
    return !n || attn_launch(pv, hv, p->dtype, layer, d_q, d_gate, d_seq, d_pos, n, max_len, d_out, d_work, st) ? 1 : 0;
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
        !attn_launch(pv, hv, p->dtype, layer, qn, gated ? q + hd : nullptr, d_seq, d_pos, n, max_len, ctx,
                     g_pw[P_WORK].p, st))
        return 0;
    return gemv(out_t, ctx, d_out, n, st) ? 1 : 0;
}
