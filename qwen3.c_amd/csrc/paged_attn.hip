// paged_attn.hip - attention of one query row per token over the pages of its sequence.
//
//   o = sum_t softmax_t(scale q . k_t) v_t over t <= pos, times sigmoid(gate)
//
// in one pass over K and V with a running maximum m and sum l per head (scores in units of
// log 2: the scale and log2 e are folded into q).
//
// A wave takes a tile of keys of one kv head with up to 16 of its query heads, and both
// products run on the matrix cores straight from the lanes' own loads:
//   scores [key][head] = K q^T: a lane's 16-byte pieces of key row l % 16 are the A operand; lane
//     l ends up with keys 4 (l / 16) + i of column l % 16.
//   out [row][column] += P V: the lane's own weights are the A operand (any order of the keys
//     does, the same on both sides), and B wants the lane's keys of one column: a lane loads
//     8 values of each of its keys' V rows and regroups them by column with one byte permute
//     per two values.  No transpose goes through LDS.
// Pages of f32 use v_mfma_f32_16x16x4_f32 as they are, 16 keys a tile.  Pages of 16 bits, 32
// keys a tile, use the 16-bit products (K and V are exact there), with q and the weights as a sum
// of pieces: 3 of bf16 (24 bits) or 2 of f16 (22 bits; q scaled by a power of two per head, the
// weights by 2^kUp).  The pieces are further rows of the same products: GS (4, 8 or 16) rows per
// piece, so 8 heads in f16 and 4 in bf16 cost one product, and the 16 rows are seldom idle.
// The f32 products they replace took 8 times the matrix cycles of one 16-bit product.
//   A piece times an infinity can be NaN where the product is infinite, and so can the zeros that q is
// padded with to the kernel's head dim (the keys' first columns are loaded again there): when a result
// is not finite, the block computes its part again in plain fp32 (slow_part), which gives what the
// formula gives.  Pages of f32 at the kernels' own head dims have no such zeros.
//
// Work: a unit is kKeys keys (a tile per wave) of a kv head, 64 KB or so; a (row, kv head) counts
// kSetup units more, about what its q, row offsets and sums cost beside the keys (200 ragged rows of
// 45 to 2900 keys, 8 kv heads: 156 us without, 125 with one).  The units of all rows in one line
// are cut into equal shares, one per block of four waves, whatever the lengths are.  A (row, kv head)
// that a border cuts goes through the workspace, and attn_join joins its parts.  Where the caller says
// that the rows are short, each (row, kv head) is a block's instead, of four waves or of one (whole_by):
// no lining up, no second launch.
//
// Bound by the bytes of K and V where there are many: two rows of 120000 keys (2 kv heads of 256,
// f16) 97 us, 5.1 TB/s (a large copy here moves 4.9, the library's GEMV reads 6.2); 48 rows of up to 16000
// keys 68 us, 4.4; the 200 rows above 121 us, 4.7.  Bound by a chain of latencies where there are few: one row of 600 keys
// 15 us, of which 4 are the join; one of 8 keys, whole, 8.4.  Tried and left out: 32-key tiles for
// heads of 256 (spills: 48 rows 121 us against 78), more blocks per CU for heads of 128 (154 us with two,
// 165 with three), blocks of eight waves for whole rows (one row of 600 keys 19.8 us with four, 21.5).
#include "paged.h"

#include <math.h>

namespace coli {

constexpr int kCUs = 256;         // of a whole card
constexpr int kGroup = 16;        // heads a wave takes
constexpr int kLaneRows = 8;      // rows of a lane while they are lined up: 512 rows or fewer
constexpr float kLazy = 8.f;      // the maximum moves when a score passes it by 2^8: weights stay below
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoKeys = -1.f;   // the sum of the weights of a part none of whose keys are there (others': 0 or more)

typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));

// A (row, kv head) that a border cuts: what attn_join needs of it.  Parts k > 0 are in slots
// 2 (block + k).
struct Cut {
    int row, head, heads, parts;   // first query head, heads, parts (0: not cut)
    int block, slot;               // of its first part
};

// Keys of a wave's tile, and waves of a SIMD (blocks of four waves a CU), which bounds their registers.  Four
// for 16-bit heads of 64 spill vector registers: 32 ragged rows of 2400 keys, 8 kv heads, 22.1 us with four, 17.0
// with three.  Blocks of one wave keep four though they spill 7 to 14 (500 rows of 32: 11.7 with four, 12.5 with
// three; no other shape was measured), and so do f32 pages (2 to 6; three was not measured).
constexpr int tile_of(int T, int HD) { return T == COLI_HIP_F32 || HD == 256 ? 16 : 32; }
constexpr int resident(int T, int HD, int W = 4) {
    return HD == 256 ? (T == COLI_HIP_F32 ? 1 : 2) : HD == 128 ? 2 : T == COLI_HIP_F32 || W == 1 ? 4 : 3;
}

struct PagedArgs {
    const float *q, *gate;
    const int *seq, *pos;
    float *out, *part;
    float2 *ml;
    Cut *cut;
    int stride;                  // heads of a part's place in the workspace
    int direct;                  // block (row, kv head) has all of it: no units, no cuts (always with W 1)
    int by_row;                  // cuts are listed by (row, kv head), else by the block they begin in
    int n, layer, groups, khv;   // head groups of kGroup per kv head, khv = KH * groups
    unsigned magic, shift;       // t / page = (umulhi(t, magic) + t) >> shift, t < 2^31
};

// The positions that row r sees (a row of no sequence: -1).
__device__ __forceinline__ int row_count(const PoolView &p, const PagedArgs &a, int r, int &s) {
    const int at = row_pos(p, a.seq, a.pos, r, s);
    return s < 0 ? -1 : at < -2 ? -3 - at : at < 0 ? 0 : at + 1;   // past the end: what is held
}
template <int kKeys>
__device__ __forceinline__ int chunks_of(int cnt) {   // an empty row has one
    return cnt < 1 ? 1 : (int)(((unsigned)cnt + kKeys - 1) / kKeys);
}
// the units of a row per kv head
template <int kKeys, int kSetup>
__device__ __forceinline__ int units_of(int cnt) {
    return cnt < 0 ? 0 : chunks_of<kKeys>(cnt) + kSetup;
}

// A value that every lane holds alike, in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ long uniform(long x) {
    return (long)(((unsigned long)(unsigned)uniform((int)(x >> 32)) << 32) | (unsigned)uniform((int)x));
}

__device__ __forceinline__ unsigned page_of(const PagedArgs &a, unsigned t) {
    return (__umulhi(t, a.magic) + t) >> a.shift;
}

template <int T>
struct Pieces;
template <>
struct Pieces<COLI_HIP_F32> {
    static constexpr int n = 1, up = 0;
};
template <>
struct Pieces<COLI_HIP_BF16> {
    static constexpr int n = 3, up = 0;
};
template <>
struct Pieces<COLI_HIP_F16> {
    static constexpr int n = 2, up = 6;   // weights of 2^6 at the maximum, 2^14 at most: small ones keep their bits
};

template <int T>
__device__ __forceinline__ float widen(unsigned word, int half) {
    if (T == COLI_HIP_F32) return __uint_as_float(word);
    if (T == COLI_HIP_BF16) return __uint_as_float(half ? word & 0xffff0000u : word << 16);
    return (float)__builtin_bit_cast(_Float16, (unsigned short)(half ? word >> 16 : word));
}
template <int T>
__device__ __forceinline__ unsigned pack(float x, float y) {   // to nearest, ties to even
    if (T == COLI_HIP_BF16) {
        typedef __bf16 v2b __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(unsigned, v2b{(__bf16)x, (__bf16)y});
    }
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, v2h{(_Float16)x, (_Float16)y});
}
// 16-bit products of 8 (4) values a lane: 32 (16) of the summed index
template <int T>
__device__ __forceinline__ v4f mfma16(v4u x, v4u y, v4f c) {
    if (T == COLI_HIP_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, x), __builtin_bit_cast(v8b, y), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, y), c, 0, 0, 0);
}
template <int T>
__device__ __forceinline__ v4f mfma16(v2u x, v2u y, v4f c) {
    if (T == COLI_HIP_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(v4s, x), __builtin_bit_cast(v4s, y), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(v4h, x), __builtin_bit_cast(v4h, y), c, 0, 0, 0);
}

// The values of lanes l ^ 16 and l ^ 32 beside the lane's own.
__device__ __forceinline__ float other16(float x) { return __shfl_xor(x, 16); }
__device__ __forceinline__ float other32(float x) { return __shfl_xor(x, 32); }
template <int N>   // the value n lanes further in the row of 16
__device__ __forceinline__ float ror(float x) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x120 + N, 0xf, 0xf, true));
}
// the sum over a head's columns (pieces) of a score
template <int GS>
__device__ __forceinline__ float sum_pieces(float x) {
    if (GS <= 8) x += ror<8>(x);
    if (GS <= 4) x += ror<4>(x);
    return x;
}

// N sums over the weights' sum (a row that has no keys: 0), times the gate.  The divisions, each a chain of ten
// instructions, and the gate's loads go side by side (one row of 128 keys, gated: 10.7 us one by one, 9.9 so).
template <int N>
__device__ __forceinline__ void finish(float *o, float l, int some, const float *gate, long at) {
#pragma unroll
    for (int i = 0; i < N; i++) o[i] = some ? o[i] / l : 0.f;
    if (!gate || !some) return;
    float w[N];
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = gate[at + i];
#pragma unroll
    for (int i = 0; i < N; i++) o[i] /= 1.f + expf(-w[i]);
}

// A part in plain fp32: keys [from, last) of the row, a key per wave at a time, four columns a
// lane, head by head.  Where no page of it is one, the row or part is empty: 0, or a sum of -1 for the join.
template <int T, int W>
__device__ void slow_part(const PoolView &p, const HeadsView &h, const PagedArgs &a, int r, int s, int kh, long head,
                          int hn, int from, int last, bool whole, long slot, float *s_o, float *s_ml) {
    constexpr int kUp = Pieces<T>::up, kWaves = W;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d0 = 4 * lane;
    const bool in = d0 < p.hd;
    const int *row = p.table + (size_t)s * p.max_pages;
    const char *base = p.data + (size_t)a.layer * p.layer_bytes + (size_t)kh * p.head_bytes;
    int seen = 0;
    for (int hh = 0; hh < hn; hh++) {
        float x[4] = {}, o[4] = {}, m = -INFINITY, l = 0.f;
        if (in)
            for (int i = 0; i < 4; i++) x[i] = a.q[((long)r * h.H + head + hh) * p.hd + d0 + i] * (h.scale * kLog2e);
        for (int t = from + wave; t < last; t += kWaves) {
            const unsigned j = page_of(a, t);
            const int pg = row[j];
            if (pg < 0 || pg >= p.n_pages) continue;
            seen = 1;
            const char *kr = base + (size_t)pg * p.page_bytes + (size_t)(t - j * p.page) * p.row_bytes;
            float k[4] = {}, v[4] = {}, dot = 0.f;
            if (in)
                for (int i = 0; i < 4; i++) {
                    const int d = d0 + i, w = T == COLI_HIP_F32 ? d : d / 2;
                    k[i] = widen<T>(((const unsigned *)kr)[w], d & 1);
                    v[i] = widen<T>(((const unsigned *)(kr + p.kv_bytes))[w], d & 1);
                    dot = fmaf(x[i], k[i], dot);
                }
            for (int sft = 32; sft; sft >>= 1) dot += __shfl_xor(dot, sft);
            const float nm = fmaxf(m, dot), f = m == nm ? 1.f : __builtin_amdgcn_exp2f(m - nm);
            const float w = dot == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(dot - nm + kUp);
            for (int i = 0; i < 4; i++) o[i] = fmaf(o[i], f, w * v[i]);
            l = fmaf(l, f, w);
            m = nm;
        }
        seen = __syncthreads_or(seen);
        if (in)
            for (int i = 0; i < 4; i++) s_o[wave * 256 + d0 + i] = o[i];
        if (lane == 0) s_ml[2 * wave] = m, s_ml[2 * wave + 1] = l;
        __syncthreads();
        float M = -INFINITY, L = 0.f, f[kWaves];
        for (int w = 0; w < kWaves; w++) M = fmaxf(M, s_ml[2 * w]);
        for (int w = 0; w < kWaves; w++) {
            f[w] = s_ml[2 * w] == M ? 1.f : __builtin_amdgcn_exp2f(s_ml[2 * w] - M);
            L += f[w] * s_ml[2 * w + 1];
        }
        for (int d = threadIdx.x; d < p.hd; d += 64 * W) {
            float t = 0.f;
            for (int w = 0; w < kWaves; w++) t += f[w] * s_o[w * 256 + d];
            if (whole) finish<1>(&t, L, seen, a.gate, r * h.q_row + (head + hh) * h.q_head + d);
            (whole ? a.out + ((long)r * h.H + head + hh) * p.hd : a.part + (slot * a.stride + hh) * p.hd)[d] = t;
        }
        if (!whole && threadIdx.x == 0) a.ml[slot * a.stride + hh] = make_float2(M, seen ? L : kNoKeys);
    }
    __syncthreads();
}

// HD: the head dim, or the next of 64, 128, 256 above it (kExact false).  GS: rows of a piece, at
// least the heads of a group.  W: waves of a block.
template <int T, int HD, bool kExact, int GS, int W>
__global__ __launch_bounds__(64 * W, resident(T, HD, W)) void attn_part(PoolView p, HeadsView h, PagedArgs a) {
    constexpr int kWaves = W, kThreads = 64 * W;
    constexpr int kWindow = W == 1 ? 128 : 1024;   // keys whose row offsets are in LDS at a time
    constexpr bool kWide = T == COLI_HIP_F32;
    constexpr int kTile = tile_of(T, HD), kSub = kTile / 16, kKeys = kWaves * kTile;
    constexpr int kPieces = Pieces<T>::n, kUp = Pieces<T>::up, kNT = kWide ? 1 : (kPieces * GS + 15) / 16;
    constexpr int kKE = kWide ? 4 : 8, kKC = HD / (4 * kKE);                       // K: values of a piece, pieces of a lane
    constexpr int kVE = HD >= 16 * kKE ? kKE : HD / 16, kVS = HD / (16 * kVE);     // V alike
    constexpr int kVW = kWide ? kVE : kVE / 2, kVK = kTile / 4;                    // words of a V piece, keys of a lane
    constexpr int kUnit = kKeys * HD * (kWide ? 8 : 4), kSetup = kUnit >= 65536 ? 1 : 65536 / kUnit;
    static_assert(kSetup <= 8, "the host counts a row's units with 8");
    constexpr int kPad = kKeys + kTile;                                            // offsets read past the last key
    constexpr int kQRow = kWide ? HD + 4 : HD / 2 + 4;                             // words of a q row in LDS
    constexpr int kQWords = kNT * 16 * kQRow, kOffWords = 2 * (kWindow + kPad), kSum = HD * 16;
    // q and the offsets of the keys' rows, then the waves' sums
    __shared__ __attribute__((aligned(16))) unsigned s_mem[kQWords + kOffWords > kWaves * kSum ? kQWords + kOffWords : kWaves * kSum];
    __shared__ int s_cnt[64 * kLaneRows], s_wave[kWaves], s_row, s_first;
    __shared__ float s_inv[kGroup], s_m[kWaves][kGroup], s_l[kWaves][kGroup];
    unsigned *const s_q = s_mem;
    long *const s_off = (long *)(s_mem + kQWords);
    float *const s_o = (float *)s_mem;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), c = lane & 15, g = lane >> 4;
    const int G = h.H / p.KH;

    // The units of all rows in one line: a thread has `per` rows; up to 64 kLaneRows rows every wave
    // lines up for itself.
    auto units = [&](int cnt) { return units_of<kKeys, kSetup>(cnt) * a.khv; };
    auto none = [&](int r) {   // no block has this row
        if (a.by_row && !blockIdx.x)
            for (int k = 0; k < a.khv; k++) a.cut[r * a.khv + k].parts = 0;
    };
    const bool direct = W == 1 || a.direct, few = !direct && a.n <= 64 * kLaneRows;
    int r, first, s, cnt, u0, end, share = 1;
    if (direct) {
        r = uniform((int)(blockIdx.x / (unsigned)a.khv));
        cnt = row_count(p, a, r, s);
        if (cnt < 0) return;
        const int nu = units_of<kKeys, kSetup>(cnt);
        first = 0, u0 = ((int)blockIdx.x - r * a.khv) * nu, end = u0 + nu;
    } else {
        const int per = few ? (a.n + 63) / 64 : (a.n + kThreads - 1) / kThreads, t0 = (few ? lane : tid) * per;
        int mine = 0, total = 0;
#pragma unroll 4
        for (int i = 0; i < per; i++) {
            int s;
            const int r = t0 + i, cnt = r < a.n ? row_count(p, a, r, s) : -1;
            if (few) s_cnt[r] = cnt;   // every wave the same
            if (r < a.n && cnt < 0) none(r);
            mine += units(cnt);
        }
        int x = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        int before = x - mine;
        if (few) {
            total = __builtin_amdgcn_readlane(x, 63);
        } else {
            if (lane == 63) s_wave[wave] = x;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                before += w < wave ? s_wave[w] : 0;
                total += s_wave[w];
            }
            total = uniform(total);
        }
        share = uniform((int)((unsigned)(total + gridDim.x - 1) / gridDim.x));
        u0 = min(total, (int)blockIdx.x * share), end = min(total, u0 + share);
        if (u0 >= end) {
            if (tid == 0 && !a.by_row) a.cut[blockIdx.x].parts = 0;
            return;
        }
        // the row of unit u0, and the units before it
        const bool mine0 = before <= u0 && u0 < before + mine;
        if (few) {
            const int l = __ffsll((unsigned long long)__ballot(mine0)) - 1;
            r = l * per;
            first = __builtin_amdgcn_readlane(before, l);
            cnt = uniform(s_cnt[r]);
            for (int i = 1; i < per; i++) {
                const int k = units(cnt);
                if (first + k > u0) break;
                first += k;
                cnt = uniform(s_cnt[++r]);
            }
            s = a.seq[r];
        } else {
            if (mine0) {
                int k = t0;
                for (int i = 1; i < per; i++) {
                    int s;
                    const int c = units(row_count(p, a, k, s));
                    if (before + c > u0) break;
                    before += c;
                    k++;
                }
                s_row = k;
                s_first = before;
            }
            __syncthreads();
            r = uniform(s_row);
            first = uniform(s_first);
            cnt = row_count(p, a, r, s);
        }
    }
    s = uniform(s);
    cnt = uniform(cnt);
    Cut cut = {};
    int done = 0;   // whether the block has had a part before

    for (int u = u0; u < end;) {
        const int nc = chunks_of<kKeys>(cnt), nu = units_of<kKeys, kSetup>(cnt);
        const int xx = u - first;
        if (xx >= nu * a.khv) {   // this row is done (or has none)
            first += nu * a.khv;
            if (++r >= a.n) break;
            cnt = uniform(few ? s_cnt[r] : row_count(p, a, r, s));
            s = uniform(a.seq[r]);
            continue;
        }
        const int hv = uniform((int)((unsigned)xx / (unsigned)nu)), x0 = xx - hv * nu;
        const int x1 = min(nu, x0 + (end - u)), c0 = max(x0 - kSetup, 0), c1 = x1 - kSetup;
        u += x1 - x0;
        if (c1 <= c0) continue;   // the keys are the next block's
        const int kh = uniform(hv / a.groups), h0 = (hv - kh * a.groups) * kGroup, hn = min(kGroup, G - h0);
        const long head = (long)kh * G + h0;   // the first query head
        const int from = c0 * kKeys, last = min(cnt, c1 * kKeys);
        const int *row = p.table + (size_t)s * p.max_pages;
        const long fix = a.layer * p.layer_bytes + kh * p.head_bytes;

        // q in units of log 2, in pieces; a wave takes every W-th head
        float qx[GS / kWaves][HD / 64];
#pragma unroll
        for (int k = 0; k < GS / kWaves; k++)
#pragma unroll
            for (int i = 0; i < HD / 64; i++) {
                const int hh = wave + kWaves * k, d = lane + 64 * i;
                qx[k][i] = hh < hn && (kExact || d < p.hd) ? a.q[((long)r * h.H + head + hh) * p.hd + d] : 0.f;
            }
        if (!kWide)   // rows of q past the last piece
            for (int i = kPieces * GS * kQRow + tid; i < kQWords; i += kThreads) s_q[i] = 0;
        // where the keys' rows lie (-1: no such key)
        auto fill = [&](int w0, int nk) {
            for (int i = tid; i < nk + kPad; i += kThreads) {
                long off = -1;
                if (i < nk) {
                    const unsigned t = w0 + i, j = page_of(a, t);
                    const int pg = row[j];
                    if (pg >= 0 && pg < p.n_pages)
                        off = pg * p.page_bytes + fix + (long)(t - j * p.page) * p.row_bytes;
                    else
                        atomicOr(&p.state[kStErr], kPgPage);
                }
                s_off[i] = off;
            }
        };
        fill(from, min(last - from, kWindow));
        lds_barrier();
        // a row that is always there, for the loads of keys that are not
        long hot = 0;
        v4u kb[kSub][kKC];
        unsigned vb[kVK][kVS][kVW];
        unsigned vm[kSub], vm_next[kSub];
        auto load_k = [&](int i0) {
#pragma unroll
            for (int t = 0; t < kSub; t++) {
                const long o = s_off[i0 + 16 * t + c];
                vm_next[t] = (unsigned)__ballot(o >= 0) & 0xffffu;
                const v4u *k = (const v4u *)(p.data + (o >= 0 ? o : hot));
#pragma unroll
                for (int i = 0; i < kKC; i++) {
                    const int at = 4 * i + g;
                    kb[t][i] = k[kExact || at * kKE < p.hd ? at : 0];
                }
            }
        };
        auto load_v = [&](int i0) {
#pragma unroll
            for (int j = 0; j < kVK; j++) {
                const long o = s_off[i0 + 16 * (j / 4) + 4 * g + j % 4];
                const char *v = p.data + p.kv_bytes + (o >= 0 ? o : hot);
#pragma unroll
                for (int i = 0; i < kVS; i++) {
                    int d = (16 * i + c) * kVE;
                    if (!kExact && d >= p.hd) d = 0;
                    if (kVW == 4)
                        *(uint4 *)vb[j][i] = *(const uint4 *)(v + d * (kWide ? 4 : 2));
                    else
                        *(uint2 *)vb[j][i] = *(const uint2 *)(v + d * (kWide ? 4 : 2));
                }
            }
        };
        auto start = [&] {   // the first tile of a window
            hot = uniform(max(s_off[0], 0L));
            load_k(wave * kTile);
            __builtin_amdgcn_sched_barrier(0);
            load_v(wave * kTile);
            __builtin_amdgcn_sched_barrier(0);
        };
        start();   // on their way while q is cut into its pieces
#pragma unroll
        for (int k = 0; k < GS / kWaves; k++) {
            const int hh = wave + kWaves * k;
            float big = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 64; i++) {
                qx[k][i] *= h.scale * kLog2e;
                big = fmaxf(big, fabsf(qx[k][i]));
            }
            if (T == COLI_HIP_F16) {   // the largest of a head in [2^14, 2^15)
#pragma unroll
                for (int o = 32; o; o >>= 1) big = fmaxf(big, __shfl_xor(big, o));
                const int e = big > 0.f && big < INFINITY ? min(14 - ilogbf(big), 100) : 0;
#pragma unroll
                for (int i = 0; i < HD / 64; i++) qx[k][i] = ldexpf(qx[k][i], e);
                if (lane == 0) s_inv[hh] = ldexpf(1.f, -e);
            }
#pragma unroll
            for (int i = 0; i < HD / 64; i++) {
                const int d = lane + 64 * i;
                if (kWide) {
                    s_q[hh * kQRow + d] = __float_as_uint(qx[k][i]);
                } else {
                    float rest = qx[k][i];
#pragma unroll
                    for (int e = 0; e < kPieces; e++) {
                        const unsigned w = pack<T>(rest, 0.f);
                        ((unsigned short *)s_q)[(e * GS + hh) * 2 * kQRow + d] = (unsigned short)w;
                        rest -= widen<T>(w, 0);
                    }
                }
            }
        }
        lds_barrier();   // the loads stay in flight
        const float inv = T == COLI_HIP_F16 ? s_inv[c % GS] : 1.f;

        v4f acc[kVS][kVE];
#pragma unroll
        for (int i = 0; i < kVS; i++)
#pragma unroll
            for (int e = 0; e < kVE; e++) acc[i][e] = v4f{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;

        for (int w0 = from; w0 < last; w0 += kWindow) {
            const int nk = min(last - w0, kWindow);
            if (w0 != from) {
                lds_barrier();
                fill(w0, nk);
                lds_barrier();
                start();
            }
            for (int i0 = wave * kTile; i0 < nk; i0 += kKeys) {
                unsigned all = 0xffffu;
#pragma unroll
                for (int t = 0; t < kSub; t++) all &= vm[t] = vm_next[t];
                // scores
                v4f sc[kSub];
                {
                    v4f d[kSub][kWide ? 2 : kNT];
#pragma unroll
                    for (int t = 0; t < kSub; t++)
#pragma unroll
                        for (int e = 0; e < (kWide ? 2 : kNT); e++) d[t][e] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < kKC; i++) {
                        if constexpr (kWide) {
                            const v4u qv = *(const v4u *)&s_q[c * kQRow + (4 * i + g) * 4];
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                d[0][e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                    __uint_as_float(kb[0][i][e]), __uint_as_float(qv[e]), d[0][e & 1], 0, 0, 0);
                        } else {
#pragma unroll
                            for (int e = 0; e < kNT; e++) {
                                const v4u qv = *(const v4u *)&s_q[(16 * e + c) * kQRow + (4 * i + g) * 4];
#pragma unroll
                                for (int t = 0; t < kSub; t++) d[t][e] = mfma16<T>(kb[t][i], qv, d[t][e]);
                            }
                        }
                    }
#pragma unroll
                    for (int t = 0; t < kSub; t++) {
                        sc[t] = d[t][0];
#pragma unroll
                        for (int e = 1; e < (kWide ? 2 : kNT); e++) sc[t] += d[t][e];
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                // blocks of four do not ask for the tile past the last: its registers are waited for (8 rows of
                // 4000 keys 23.5 -> 23.0 us, 200 ragged rows 123.0 -> 121.5); blocks of one lose by the branch (500
                // rows of 100 48.6 -> 49.5)
                if (W == 1 || i0 + kKeys < nk) load_k(i0 + kKeys);
                __builtin_amdgcn_sched_barrier(0);
                float mt = -INFINITY;
#pragma unroll
                for (int t = 0; t < kSub; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (!kWide) sc[t][i] = sum_pieces<GS>(sc[t][i]);
                        if (T == COLI_HIP_F16) sc[t][i] *= inv;
                    }
                if (all != 0xffffu) {   // keys that are not there: no score, and nothing of V
#pragma unroll
                    for (int j = 0; j < kVK; j++) {
                        if (vm[j / 4] >> (4 * g + j % 4) & 1) continue;
                        sc[j / 4][j % 4] = -INFINITY;
#pragma unroll
                        for (int i = 0; i < kVS; i++)
#pragma unroll
                            for (int w = 0; w < kVW; w++) vb[j][i][w] = 0;
                    }
                }
#pragma unroll
                for (int t = 0; t < kSub; t++) mt = fmaxf(mt, fmaxf(fmaxf(sc[t][0], sc[t][1]), fmaxf(sc[t][2], sc[t][3])));
                mt = fmaxf(mt, other16(mt));
                mt = fmaxf(mt, other32(mt));
                if (__any(mt > m + kLazy)) {
                    const float nm = fmaxf(m, mt), f = m == nm ? 1.f : __builtin_amdgcn_exp2f(m - nm);
                    l *= f;
                    m = nm;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float fr = __shfl(f, 4 * g + i);
#pragma unroll
                        for (int t = 0; t < kVS; t++)
#pragma unroll
                            for (int e = 0; e < kVE; e++) acc[t][e][i] *= fr;
                    }
                }
                float w[kVK];
#pragma unroll
                for (int j = 0; j < kVK; j++) {
                    const float x = sc[j / 4][j % 4];
                    w[j] = x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x - m + kUp);
                    l += w[j];
                }
                // out += P V
                if constexpr (kWide) {
#pragma unroll
                    for (int j = 0; j < kVK; j++)
#pragma unroll
                        for (int i = 0; i < kVS; i++)
#pragma unroll
                            for (int e = 0; e < kVE; e++)
                                acc[i][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[j], __uint_as_float(vb[j][i][e]),
                                                                                 acc[i][e], 0, 0, 0);
                } else {
                    constexpr int kPW = kVK / 2;   // words of a lane's weights
                    typedef unsigned vp __attribute__((ext_vector_type(kPW)));
                    vp pw[kPieces], pa[kNT];
#pragma unroll
                    for (int e = 0; e < kPieces; e++)
#pragma unroll
                        for (int j = 0; j < kPW; j++) {
                            pw[e][j] = pack<T>(w[2 * j], w[2 * j + 1]);
                            w[2 * j] -= widen<T>(pw[e][j], 0);
                            w[2 * j + 1] -= widen<T>(pw[e][j], 1);
                        }
#pragma unroll
                    for (int e = 0; e < kNT; e++) {   // row c of product e is piece (16 e + c) / GS
#pragma unroll
                        for (int j = 0; j < kPW; j++) pa[e][j] = 0;
#pragma unroll
                        for (int k = 0; k < kPieces; k++) {
                            if ((k + 1) * GS <= 16 * e || k * GS >= 16 * e + 16) continue;
                            const bool is = (16 * e + c) / GS == k;
#pragma unroll
                            for (int j = 0; j < kPW; j++) pa[e][j] = is ? pw[k][j] : pa[e][j];
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kVS; i++)
#pragma unroll
                        for (int x = 0; x < kVE; x++) {
                            vp b;
#pragma unroll
                            for (int j = 0; j < kPW; j++)
                                b[j] = __builtin_amdgcn_perm(vb[2 * j + 1][i][x / 2], vb[2 * j][i][x / 2],
                                                             x & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                            for (int e = 0; e < kNT; e++) acc[i][x] = mfma16<T>(pa[e], b, acc[i][x]);
                        }
                }
                __builtin_amdgcn_sched_barrier(0);
                if (W == 1 || i0 + kKeys < nk) load_v(i0 + kKeys);
                __builtin_amdgcn_sched_barrier(0);
            }
        }

        const bool whole = c0 == 0 && c1 == nc;
        const long slot = 2L * blockIdx.x + done;
        // the four waves' parts
        l += other16(l);
        l += other32(l);
        if (g == 0) {
            s_m[wave][c] = m;
            s_l[wave][c] = l;
        }
        lds_barrier();   // the last loads, of no keys, need not have come
        float z = 0.f;   // NaN when a result of this thread's is not finite, 1 when a row's weights are all 0
        {
            float *so = s_o + wave * kSum + 4 * lane;
#pragma unroll
            for (int t = 0; t < kVS * kVE; t++) *(v4f *)(so + 256 * t) = acc[t / kVE][t % kVE];
            lds_barrier();
            // a thread: head hh's kVE columns from d0.  Rows of one head's pieces are GS apart.
            for (int i = tid; i < GS * kVS * 16; i += kThreads) {
                const int hh = i / 16 % GS, t = i / 16 / GS, d0 = (16 * t + (i & 15)) * kVE;
                if (hh >= hn || (!kExact && d0 >= p.hd)) continue;
                float f[kWaves], M = -INFINITY, L = 0.f, o[kVE];
#pragma unroll
                for (int w = 0; w < kWaves; w++) M = fmaxf(M, f[w] = s_m[w][hh]);
#pragma unroll
                for (int w = 0; w < kWaves; w++) {
                    f[w] = f[w] == M ? 1.f : __builtin_amdgcn_exp2f(f[w] - M);
                    L = fmaf(s_l[w][hh], f[w], L);
                }
#pragma unroll
                for (int e = 0; e < kVE; e++) o[e] = 0.f;
#pragma unroll
                for (int k = 0; k < (kWide ? 1 : 16 / GS); k++) {
                    const int row = hh + k * GS;
                    const float *at = s_o + 256 * kVE * t + (row / 4 * 16 + (i & 15)) * 4 + row % 4;
#pragma unroll
                    for (int e = 0; e < kVE; e++)
#pragma unroll
                        for (int w = 0; w < kWaves; w++) o[e] = fmaf(at[w * kSum + 256 * e], f[w], o[e]);
                }
#pragma unroll
                for (int e = 0; e < kVE; e++)
                    if (!(kWide && kExact)) z = fmaf(o[e] + L, 0.f, z);
                if (L == 0.f && cnt) z += 1.f;
                float *dst = a.part + (slot * a.stride + hh) * p.hd + d0;
                if (whole) {
                    dst = a.out + ((long)r * h.H + head + hh) * p.hd + d0;
                    finish<kVE>(o, L, cnt, a.gate, r * h.q_row + (head + hh) * h.q_head + d0);
                } else if (d0 == 0) {
                    a.ml[slot * a.stride + hh] = make_float2(M, L);
                }
#pragma unroll
                for (int e = 0; e < kVE; e += 4) *(float4 *)(dst + e) = *(const float4 *)(o + e);
            }
        }
        // the sums' place is the next part's q; products that met an infinity or NaN: again, where pieces or
        // the zeros of q past the head dim may have made a NaN of what is none.  And where no key had a weight,
        // to tell scores of -inf (NaN) from pages that are none (0).
        if (__syncthreads_or(z != 0.f))
            slow_part<T, W>(p, h, a, r, s, kh, head, hn, from, last, whole, slot, s_o, &s_m[0][0]);
        if (c0 == 0 && !direct) {   // u is behind its unit c1
            cut = Cut{};
            if (c1 < nc) {
                const int parts = (int)((unsigned)(u + (nc - c1) - 1) / (unsigned)share) - (int)blockIdx.x + 1;
                cut = Cut{r, (int)head, hn, parts, (int)blockIdx.x, (int)slot};
            }
            if (a.by_row && tid == 0) a.cut[r * a.khv + hv] = cut;
        }
        done = 1;
    }
    if (tid == 0 && !direct && !a.by_row) a.cut[blockIdx.x] = cut;   // only the last part can go on
}

// Block (i, hh, z): columns z * cols.. of head hh of cut i.  A thread has four columns of every
// ks-th part; the first kAhead parts are on their way while the weights are found.
constexpr int kAhead = 8, kJoin = 256;
constexpr int kJoinW = kCUs * 4;   // parts whose weights are kept: a launch's blocks (max_blocks) at most
__global__ __launch_bounds__(kJoin) void attn_join(PoolView p, HeadsView h, PagedArgs a, int cols) {
    __shared__ float s_w[kJoinW], s_red[kJoin / 64];
    __shared__ v4f s_o[kJoin];
    const Cut cut = a.cut[blockIdx.x];
    const int hh = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = cut.parts;
    if (!n || hh >= cut.heads) return;
    const int wide = cols / 4, d = blockIdx.z * cols + tid % wide * 4, k0 = tid / wide, ks = kJoin / wide;
    const bool in = d < p.hd;
    auto at = [&](int k) { return (k ? 2L * (cut.block + k) : (long)cut.slot) * a.stride + hh; };
    v4f x[kAhead], o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
        const int k = k0 + j * ks;
        x[j] = k < n && in ? *(const v4f *)(a.part + at(k) * p.hd + d) : o;
    }
    float m = -INFINITY, l = 0.f;
    for (int k = tid; k < n; k += kJoin) {
        const float2 ml = a.ml[at(k)];
        m = fmaxf(m, ml.x);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (lane == 0) s_red[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    __syncthreads();
    for (int k = tid; k < n; k += kJoin) {
        const float2 ml = a.ml[at(k)];
        const float f = ml.x == m ? 1.f : __builtin_amdgcn_exp2f(ml.x - m);
        s_w[k] = f;
        l += f * ml.y;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o);
    if (lane == 0) s_red[wave] = l;
    __syncthreads();
    l = (s_red[0] + s_red[1]) + (s_red[2] + s_red[3]);
    const bool some = m != -INFINITY || l != n * kNoKeys;   // parts of no keys count with any other part's 0 at most
    if (m == -INFINITY) l = 0.f;                            // every score is -inf
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
        const int k = k0 + j * ks;
        if (k < n) o += s_w[k] * x[j];
    }
    if (in) {
#pragma unroll 8
        for (int k = k0 + kAhead * ks; k < n; k += ks) o += s_w[k] * *(const v4f *)(a.part + at(k) * p.hd + d);
    }
    s_o[tid] = o;
    __syncthreads();
    if (k0 || !in) return;
    for (int k = 1; k < ks; k++) o += s_o[tid + k * wide];
    float y[4] = {o[0], o[1], o[2], o[3]};
    finish<4>(y, l, some, a.gate, cut.row * h.q_row + (cut.head + hh) * h.q_head + d);
    o = v4f{y[0], y[1], y[2], y[3]};
    *(v4f *)(a.out + ((long)cut.row * h.H + cut.head + hh) * p.hd + d) = o;
}

// Blocks of a launch: on a card's 256 CUs all of them are resident, so that equal shares end together (on a
// partition of fewer CUs they take their turns).  A constant: the workspace's size is asked for without a device.
static int max_blocks(int T, int HD) { return kCUs * resident(T, HD); }
static_assert(kJoinW >= kCUs * resident(COLI_HIP_F32, 64) && kJoinW >= kCUs * resident(COLI_HIP_F16, 64),
              "the join keeps a weight for every block of a launch");
static int head_dim(int hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }

// Waves of the blocks where each has a (row, kv head) to itself, or 0: units in equal shares.  us with
// whole rows / shares, ragged rows of up to so many keys where there are several:
//   few (row, kv head)s, up to 300 KB of K and V each; 2 kv heads of 256, bf16: one row of 128 keys 9.9 / 15.5,
//   300 13.7 / 14.7, 600 19.5 / 14.8; 8 of 128: 128 7.3 / 10.3, 600 11.7 / 13.4, 1200 18.5 / 13.4; 8 of 64, f32:
//   300 9.9 / 12.5, 600 14.2 / 12.6
//   from 128 on, where shares are cut oftener, up to 450 KB; 128 rows, 2 kv heads of 256: 300 15.9 / 20.8, 600
//   22.1 / 22.0, 1200 35 / 27; 8 of 128, f32: 300 30.5 / 32.8, 1200 77 / 63
//   from 512 on up to 640 KB; 2 kv heads of 256, 260 to 400 rows of 600 all alike 79 to 105 / 83 to 116, ragged
//   27 to 42 / 33 to 49; 8 of 128, 65 and 150 rows of 1200 75, 136 / 73, 145, ragged 29, 54 / 26, 56
// One wave instead of four where not all blocks of four are resident and the rows are short for that (us
// with 1 / 4; 8 heads of 128, bf16: 128 rows of 128 10 / 15.6, 600 27.4 / 23.7; 500 of 300 42 / 65; f32: 128 of 32
// 9.8 / 16.4, 300 34 / 30.5; 500 rows, 2 heads of 256: 128 22.9 / 24.4, 300 36 / 32), and, 16 bits and heads up to
// 128, for rows of a tile (6.3 / 7.0).
static int whole_by(int T, int HD, long row_heads, int max_len) {
    const long bytes = 2L * max_len * HD * (T == COLI_HIP_F32 ? 4 : 2), blocks = max_blocks(T, HD);
    if (max_len <= 0 || bytes > (row_heads < 128 ? 300L : row_heads < 512 ? 450L : 640L) << 10) return 0;
    if (T != COLI_HIP_F32 && HD <= 128 && max_len <= tile_of(T, HD)) return 1;
    return row_heads > blocks && max_len * blocks <= 5 * tile_of(T, HD) * row_heads ? 1 : 4;
}

// Two parts a block, each of up to 16 heads.
size_t attn_paged_work(const PoolView &p) {
    const int T = p.es == 4 ? COLI_HIP_F32 : COLI_HIP_F16, HD = head_dim(p.hd);
    const size_t blocks = max_blocks(T, HD);
    return 2 * blocks * kGroup * (p.hd * sizeof(float) + sizeof(float2)) + blocks * sizeof(Cut);
}

template <int T, int GS, int W>
static void launch(const PoolView &pv, const HeadsView &hv, const PagedArgs &a, int blocks, hipStream_t st) {
    const dim3 g(blocks), t(64 * W);
    switch (pv.hd) {
    case 64: hipLaunchKernelGGL((attn_part<T, 64, true, GS, W>), g, t, 0, st, pv, hv, a); return;
    case 128: hipLaunchKernelGGL((attn_part<T, 128, true, GS, W>), g, t, 0, st, pv, hv, a); return;
    case 256: hipLaunchKernelGGL((attn_part<T, 256, true, GS, W>), g, t, 0, st, pv, hv, a); return;
    }
    if (pv.hd < 64)
        hipLaunchKernelGGL((attn_part<T, 64, false, GS, W>), g, t, 0, st, pv, hv, a);
    else if (pv.hd < 128)
        hipLaunchKernelGGL((attn_part<T, 128, false, GS, W>), g, t, 0, st, pv, hv, a);
    else
        hipLaunchKernelGGL((attn_part<T, 256, false, GS, W>), g, t, 0, st, pv, hv, a);
}

template <int T, int W>
static void launch_heads(const PoolView &pv, const HeadsView &hv, const PagedArgs &a, int blocks, hipStream_t st) {
    if constexpr (T != COLI_HIP_F32) {
        if (a.stride == 8) return launch<T, 8, W>(pv, hv, a, blocks, st);
        if (a.stride == 4) return launch<T, 4, W>(pv, hv, a, blocks, st);
    }
    launch<T, 16, W>(pv, hv, a, blocks, st);
}

template <int W>
static void launch_type(const PoolView &pv, const HeadsView &hv, int dtype, const PagedArgs &a, int blocks, hipStream_t st) {
    switch (dtype) {
    case COLI_HIP_F32: launch_heads<COLI_HIP_F32, W>(pv, hv, a, blocks, st); break;
    case COLI_HIP_F16: launch_heads<COLI_HIP_F16, W>(pv, hv, a, blocks, st); break;
    default: launch_heads<COLI_HIP_BF16, W>(pv, hv, a, blocks, st);
    }
}

bool attn_paged(const PoolView &pv, const HeadsView &hv, int dtype, int layer, const float *q, const float *gate,
                const int *seq, const int *pos, int n, int max_len, float *out, void *work, hipStream_t st) {
    const int G = hv.H / pv.KH, HD = head_dim(pv.hd), GS = dtype == COLI_HIP_F32 || G > 8 ? 16 : G > 4 ? 8 : 4;
    const int most = max_blocks(dtype, HD), keys = 4 * tile_of(dtype, HD), groups = (G + kGroup - 1) / kGroup;
    PagedArgs a;
    a.q = q, a.gate = gate, a.seq = seq, a.pos = pos, a.out = out, a.n = n, a.layer = layer;
    a.part = (float *)work;
    a.ml = (float2 *)(a.part + 2 * (size_t)most * GS * pv.hd);
    a.cut = (Cut *)(a.ml + 2 * (size_t)most * GS);
    a.stride = GS;
    a.groups = groups;
    a.khv = pv.KH * a.groups;
    a.shift = 0;
    while ((1L << a.shift) < pv.page) a.shift++;
    a.magic = (unsigned)(((1ULL << 32) * ((1ULL << a.shift) - pv.page)) / pv.page + 1);
    const long cap = (long)pv.max_pages * pv.page, len = max_len > 0 && max_len < cap ? max_len : cap;
    // the units of a launch's rows are counted in 31 bits: more rows go in several launches
    const long row = ((cap + keys - 1) / keys + 8) * a.khv;   // kSetup is 8 at most
    if (row >= 1L << 30) return paged_refuse("a sequence of more than 2^30 units");
    const long row_heads = (long)n * a.khv;
    const int whole = row < 1L << 28 && row_heads <= 1L << 22 ? whole_by(dtype, HD, row_heads, max_len) : 0;
    a.direct = whole != 0;
    if (whole) {
        a.n = n;
        if (whole == 1)
            launch_type<1>(pv, hv, dtype, a, (int)row_heads, st);
        else
            launch_type<4>(pv, hv, dtype, a, (int)row_heads, st);
        return paged_launched("paged attention launch");
    }
    const int rows = (int)min((long)n, (1L << 30) / row);
    for (int r = 0; r < n; r += rows) {
        a.n = min(rows, n - r);
        const long units = ((len + keys - 1) / keys) * a.khv * (long)a.n;   // more blocks would cut setups only
        const int blocks = (int)(units < most ? units : most);
        a.by_row = a.n * (long)a.khv <= blocks;
        launch_type<4>(pv, hv, dtype, a, blocks, st);
        if (blocks > 1) {
            // few cuts: blocks of 64 columns (16 parts at a time); else of a whole head
            const int cuts = a.by_row ? a.n * a.khv : blocks, heads = G < kGroup ? G : kGroup;
            const int cols = cuts * heads <= 512 ? 64 : pv.hd <= 64 ? 64 : pv.hd <= 128 ? 128 : 256;
            hipLaunchKernelGGL(attn_join, dim3(cuts, heads, (pv.hd + cols - 1) / cols), dim3(kJoin), 0, st, pv, hv, a,
                               cols);
        }
        a.q += (size_t)a.n * hv.H * pv.hd;
        a.out += (size_t)a.n * hv.H * pv.hd;
        a.seq += a.n;
        if (a.pos) a.pos += a.n;
        if (a.gate) a.gate += a.n * hv.q_row;
    }
    return paged_launched("paged attention launch");
}

}  // namespace coli
