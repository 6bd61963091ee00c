// pages.hip - the pages of a key-value cache that serves many sequences: taking pages for new
// positions, forking and freeing sequences, closing up the pool.  No counterpart in the
// reference, whose cache is one dense row per position of one sequence.
//
// Everything a decode loop changes lives on the device (tables, lengths, reference counts, the
// bitmap of pages in use), so a step needs no host decision and can be captured.  Nothing
// depends on the order of atomics: pages are taken lowest free one first in the order of the
// call, counts are integers, and a page's bit falls with the count that reaches 0.  A page that
// is not full belongs to one sequence alone (fork copies it), so a new position never lands in
// a shared page; a step whose append was refused has no position to write, and the sequences'
// words (paged.h) tell the rotation so.
//
// The copies are bound by their bytes: 20 of 40 sequences replaced with the pool closed up, 530 MB
// moved, 227 us for the four launches (the move 197 us, 5.4 TB/s); six sequences copied whole, 209 MB,
// 103 us (the copy 89).  60 forks that share their full pages: 16 us, three launches of 3 to 7 us.
#include "paged.h"

#include <stdio.h>
#include <stdlib.h>

namespace coli {

constexpr int kPgThreads = 1024;     // the bookkeeping block
constexpr int kTakeN = 4;            // sequences of a thread of pages_take
constexpr int kPgMaxN = kTakeN * kPgThreads;   // of a call
constexpr int kCopyThreads = 256;
constexpr long kCopyPiece = 16384;   // bytes of a page that one block copies at a time

bool paged_refuse(const char *why) {
    fprintf(stderr, "[HIP] paged cache call refused: %s\n", why);
    return false;
}

bool pool_view(const ColiHipPages *p, PoolView &v) {
    if (!p || !p->data || !p->table || !p->lens || !p->refs || !p->used || !p->state || !p->work)
        return paged_refuse("a pool pointer is NULL");
    if (p->dtype != COLI_HIP_F32 && p->dtype != COLI_HIP_F16 && p->dtype != COLI_HIP_BF16)
        return paged_refuse("page type");
    if (p->hd < 8 || p->hd > 256 || p->hd % 8) return paged_refuse("head dim not a multiple of 8 in 8..256");
    if (p->page < 1 || p->page > 4096) return paged_refuse("page size not in 1..4096");
    if (p->KH < 1 || p->KH > 1024 || p->n_layers < 1 || p->n_layers > 4096) return paged_refuse("heads or layers");
    if (p->n_pages < 1 || p->n_seqs < 1 || p->max_pages < 1) return paged_refuse("empty pool");
    if ((long)p->max_pages * p->page > 1L << 30 || p->n_pages > 1 << 30) return paged_refuse("pool too large");
    if ((uintptr_t)p->data % 16) return paged_refuse("pool data not aligned to 16 bytes");
    v.data = (char *)p->data;
    v.table = p->table, v.lens = p->lens, v.refs = p->refs, v.used = p->used, v.state = p->state, v.work = p->work;
    v.es = p->dtype == COLI_HIP_F32 ? 4 : 2;
    v.n_layers = p->n_layers, v.KH = p->KH, v.hd = p->hd, v.page = p->page;
    v.n_pages = p->n_pages, v.n_seqs = p->n_seqs, v.max_pages = p->max_pages;
    v.row_bytes = (long)p->hd * v.es;
    v.head_bytes = v.row_bytes * p->page;
    v.kv_bytes = v.head_bytes * p->KH;
    v.layer_bytes = 2 * v.kv_bytes;
    v.page_bytes = v.layer_bytes * p->n_layers;
    return v.page_bytes < 1L << 34 || paged_refuse("page of 16 GiB or more");
}

bool paged_stream(void *stream_, hipStream_t &st) {
    if (!ok()) return false;
    int dev = -1;
    if (hipGetDevice(&dev) != hipSuccess || dev != 0) return paged_refuse("the library's device is not current");
    st = stream_ ? (hipStream_t)stream_ : stream();
    return true;
}

bool paged_launched(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess || fail(what, e);
}

// ---------------------------------------------------------------- block helpers
// Exclusive prefix sum of v over the block's threads, the total in *total.
__device__ __forceinline__ int block_scan(int v, int *s_wave, int *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    if (lane == 63) s_wave[wave] = x;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kPgThreads / 64; w++) {
        const int t = s_wave[w];
        before += w < wave ? t : 0;
        all += t;
    }
    __syncthreads();
    *total = all;
    return before + x - v;
}

// The pages of word w that are in use; those past the pool's end count as used.
__device__ __forceinline__ unsigned used_word(const PoolView &p, int w) {
    unsigned u = p.used[w];
    const int left = p.n_pages - w * 32;
    if (left < 32) u |= ~0u << left;
    return u;
}

__device__ __forceinline__ int pages_of(int len, int page) { return (int)(((long)len + page - 1) / page); }

// ---------------------------------------------------------------- taking pages
enum { kTakeAppend = 0, kTakeShare = 1, kTakeCopy = 2 };

// One block.  Append: sequence b[i] grows by count[i] positions (NULL: 1).  Fork: b[i] becomes
// as long as a[i]; its new pages are the last, partly filled one (share) or all of them (copy).
// Nothing changes unless the whole call can be done.
// A chain of latencies (names, lengths, table) with three barriers: the scan that places the needs
// also ranks the free pages of the first T words of the bitmap.  T = 512 where four words a
// thread cover the pool, 1024 otherwise (60 forks in a pool of 13000 pages: 6.2 us with 512 threads, 7.7
// with 1024; 20 sequences of 2200 pages in all: 11.0 both, 13.5 with 256).
template <int T>
__global__ __launch_bounds__(T) void pages_take(PoolView p, const int *__restrict__ a, const int *__restrict__ b,
                                                const int *__restrict__ count, int n, int mode) {
    constexpr int kMax = kTakeN * T, kHash = 2 * kMax, kW = T / 64;
    __shared__ int s_off[kMax + 1];    // sequence i's new pages: [s_off[i], s_off[i + 1])
    __shared__ int s_first[kMax];      // and its first new table entry
    __shared__ int s_list[kMax];       // the new pages, where they are that few
    __shared__ int s_hash[kHash];      // the sequences named so far
    __shared__ long s_need[kW];
    __shared__ int s_free[kW], s_more[kW], s_err[kW];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, words = (p.n_pages + 31) / 32;
    const unsigned fr0 = tid < words ? ~used_word(p, tid) : 0u;
    for (int i = tid; i < kHash; i += T) s_hash[i] = -1;
    int more = 0;   // free pages past the first T words
    for (int w = tid + T; w < words; w += T) more += __popc(~used_word(p, w));
    const long most = (long)p.max_pages * p.page;
    // what each needs: a thread has kTakeN neighbours
    int s[kTakeN], need[kTakeN], grown[kTakeN], first[kTakeN], err = 0;
#pragma unroll
    for (int k = 0; k < kTakeN; k++) {
        const int i = tid * kTakeN + k;
        s[k] = -1, need[k] = grown[k] = first[k] = 0;
        if (i >= n) continue;
        const int to = b[i], from = mode == kTakeAppend ? to : a[i];
        if (to < -1 || to >= p.n_seqs || from < -1 || from >= p.n_seqs) {
            err |= kPgIndex;
        } else if (to >= 0 && from >= 0) {
            s[k] = to;
            const int len = p.lens[to];
            if (len < 0 || len > most) err |= kPgIndex;
            if (mode == kTakeAppend) {
                const int c = count ? count[i] : 1;
                if (c < 0) {
                    err |= kPgIndex;
                } else if ((long)len + c > most) {
                    err |= kPgRow;
                } else {
                    grown[k] = len + c;
                    first[k] = pages_of(len, p.page);
                    need[k] = pages_of(len + c, p.page) - first[k];
                }
            } else {
                grown[k] = p.lens[from];
                if (len != 0 || to == from) err |= kPgTwice;
                if (grown[k] < 0 || grown[k] > most) err |= kPgIndex;
                first[k] = mode == kTakeCopy ? 0 : grown[k] / p.page;
                need[k] = pages_of(grown[k], p.page) - first[k];
            }
        }
    }
    __syncthreads();
    long mine = 0;
#pragma unroll
    for (int k = 0; k < kTakeN; k++) {
        mine += need[k];
        if (s[k] < 0) continue;
        unsigned at = (unsigned)s[k] * 2654435761u % kHash;
        for (;;) {   // ends: twice as many places as sequences
            const int old = atomicCAS(&s_hash[at], -1, s[k]);
            if (old == s[k]) err |= kPgTwice;
            if (old == -1 || old == s[k]) break;
            at = (at + 1) % kHash;
        }
    }
    long x = mine;
    int f = __popc(fr0);
    const int f0 = f;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long y = __shfl_up(x, o);
        const int g = __shfl_up(f, o);
        if (lane >= o) x += y, f += g;
        more += __shfl_xor(more, o);
        err |= __shfl_xor(err, o);
    }
    if (lane == 63) s_need[wave] = x, s_free[wave] = f, s_more[wave] = more, s_err[wave] = err;
    __syncthreads();
    long total = 0, off = x - mine;
    int found = 0, rank = f - f0, rest = 0;
    err = 0;
    for (int w = 0; w < kW; w++) {
        off += w < wave ? s_need[w] : 0;
        rank += w < wave ? s_free[w] : 0;
        total += s_need[w], found += s_free[w], rest += s_more[w], err |= s_err[w];
    }
    if (!err && total > (long)found + rest) err = kPgFull;
    if (err) {
        if (mode == kTakeAppend)
#pragma unroll
            for (int k = 0; k < kTakeN; k++)
                if (s[k] >= 0 && (!count || count[tid * kTakeN + k])) grow_word(p, s[k]) = refused_at(p.lens[s[k]]);
        if (tid == 0) {
            atomicOr(&p.state[kStErr], err);
            p.state[kStGo] = 0;
        }
        return;
    }
    // the lengths (all were read before the barrier: a fork's source may be another's target)
#pragma unroll
    for (int k = 0; k < kTakeN; k++) {
        const int i = tid * kTakeN + k;
        if (i < n) s_off[i] = (int)off, s_first[i] = first[k];
        off += need[k];
        if (s[k] < 0) continue;
        p.lens[s[k]] = grown[k];
        if (mode != kTakeAppend || !count || count[i]) grow_word(p, s[k]) = 0;
    }
    if (tid == 0) s_off[n] = (int)total, p.state[kStGo] = 1;
    // the lowest `total` free pages, in order, into the list
    int *list = total <= kMax ? s_list : p.work;
    unsigned fr = fr0;
    for (int w0 = 0, base = 0;;) {
        const int w = w0 + tid;
        unsigned taken = 0;
        while (fr && rank < total) {
            const int bit = __ffs(fr) - 1;
            list[rank++] = w * 32 + bit;
            taken |= 1u << bit;
            fr &= fr - 1;
        }
        if (taken) p.used[w] |= taken;
        base += found;
        w0 += T;
        if (base >= total || w0 >= words) break;   // alike in every thread
        fr = w0 + tid < words ? ~used_word(p, w0 + tid) : 0u;
        f = __popc(fr);
        rank = f;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int g = __shfl_up(rank, o);
            if (lane >= o) rank += g;
        }
        __syncthreads();
        if (lane == 63) s_free[wave] = rank;
        __syncthreads();
        rank += base - f;
        found = 0;
        for (int v = 0; v < kW; v++) {
            rank += v < wave ? s_free[v] : 0;
            found += s_free[v];
        }
    }
    __syncthreads();
    // each page to its table entry
    for (int r = tid; r < (int)total; r += T) {
        int lo = 0, hi = n;   // the last i with s_off[i] <= r
        while (hi - lo > 1) {
            const int m = (lo + hi) / 2;
            if (s_off[m] <= r)
                lo = m;
            else
                hi = m;
        }
        const int pg = list[r];
        p.table[(size_t)b[lo] * p.max_pages + s_first[lo] + r - s_off[lo]] = pg;
        p.refs[pg] = 1;
    }
}

// ---------------------------------------------------------------- copying
typedef unsigned v4u __attribute__((ext_vector_type(4)));
// The first `held` rows of every head plane of page `from` to page `to`, piece of pieces.
__device__ __forceinline__ void copy_page(const PoolView &p, int from, int to, int held, int piece, int pieces) {
    const v4u *src = (const v4u *)(p.data + (size_t)from * p.page_bytes);
    v4u *dst = (v4u *)(p.data + (size_t)to * p.page_bytes);
    // 16-byte units of a plane held, and from plane to plane
    const unsigned plane = held * (unsigned)(p.row_bytes / 16), stride = (unsigned)(p.head_bytes / 16);
    const unsigned n = plane * (unsigned)(p.n_layers * 2 * p.KH), per = (n + pieces - 1) / pieces;
    const unsigned end = min(n, (piece + 1) * per);
    auto place = [&](unsigned w) { return plane == stride ? w : w / plane * stride + w % plane; };
    unsigned u = piece * per + threadIdx.x;
    for (; u + 3 * kCopyThreads < end; u += 4 * kCopyThreads) {   // four loads before the first store
        v4u x[4];
        unsigned at[4];
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = src[at[i] = place(u + i * kCopyThreads)];
#pragma unroll
        for (int i = 0; i < 4; i++) dst[at[i]] = x[i];
    }
    for (; u < end; u += kCopyThreads) {
        const unsigned at = place(u);
        dst[at] = src[at];
    }
}

static int pieces_of(const PoolView &p) {
    const long n = (p.page_bytes + kCopyPiece - 1) / kCopyPiece;
    return (int)(n < 1 ? 1 : n > 4096 ? 4096 : n);
}

// Behind pages_take: the shared entries of the table with their counts, and the rows of the
// new pages.  Block (i, y) takes every gridDim.y-th piece of pair i.
__global__ __launch_bounds__(kCopyThreads) void pages_fork_copy(PoolView p, const int *__restrict__ a,
                                                                const int *__restrict__ b, int share, int pieces) {
    const int s = b[blockIdx.x], f = a[blockIdx.x];
    if (!p.state[kStGo] || s < 0 || f < 0) return;
    const int len = p.lens[s], full = len / p.page, np = pages_of(len, p.page);
    const int *from = p.table + (size_t)f * p.max_pages;
    int *to = p.table + (size_t)s * p.max_pages;
    if (share)
        for (int j = blockIdx.y * kCopyThreads + threadIdx.x; j < full; j += gridDim.y * kCopyThreads) {
            const int pg = from[j];
            to[j] = pg;
            if (pg >= 0 && pg < p.n_pages)
                atomicAdd(&p.refs[pg], 1);
            else
                atomicOr(&p.state[kStErr], kPgPage);
        }
    const int j0 = share ? full : 0;
    const long tasks = (long)(np - j0) * pieces;
    for (long t = blockIdx.y; t < tasks; t += gridDim.y) {
        const int j = j0 + (int)(t / pieces), src = from[j], dst = to[j];
        if (src < 0 || src >= p.n_pages || dst < 0 || dst >= p.n_pages) {
            atomicOr(&p.state[kStErr], kPgPage);
            continue;
        }
        copy_page(p, src, dst, min(p.page, len - j * p.page), (int)(t % pieces), pieces);
    }
}

// ---------------------------------------------------------------- freeing
// Block i ends sequence seq[i]: the length is taken atomically, so a sequence named twice (or
// an empty one) is freed once.
__global__ __launch_bounds__(kCopyThreads) void pages_drop(PoolView p, const int *__restrict__ seq) {
    __shared__ int s_len;
    const int s = seq[blockIdx.x];
    if (s < 0 || s >= p.n_seqs) {
        if (s != -1 && threadIdx.x == 0) atomicOr(&p.state[kStErr], kPgIndex);
        return;
    }
    int *row = p.table + (size_t)s * p.max_pages, next = -1;
    if (threadIdx.x == 0) {
        s_len = atomicExch(&p.lens[s], 0);
        grow_word(p, s) = 0;
    }
    if (threadIdx.x < p.max_pages) next = row[threadIdx.x];
    __syncthreads();
    const int np = min(pages_of(s_len, p.page), p.max_pages);
    for (int j = threadIdx.x; j < np; j += kCopyThreads) {
        const int pg = next;
        if (j + kCopyThreads < np) next = row[j + kCopyThreads];
        row[j] = -1;
        if (pg < 0 || pg >= p.n_pages) {
            atomicOr(&p.state[kStErr], kPgPage);
            continue;
        }
        if (atomicSub(&p.refs[pg], 1) == 1) atomicAnd(&p.used[pg >> 5], ~(1u << (pg & 31)));
    }
}

// ---------------------------------------------------------------- closing up
// One block: with L pages in use, the k-th used page at or past L (a mover) goes into the k-th
// free page below L (a hole).  work holds the holes, the movers, and for each page past L its
// new place.
__global__ __launch_bounds__(kPgThreads) void pages_plan(PoolView p) {
    __shared__ int s_wave[kPgThreads / 64];
    const int tid = threadIdx.x, words = (p.n_pages + 31) / 32;
    int n = 0, live;
    for (int w = tid; w < words; w += kPgThreads) n += 32 - __popc(used_word(p, w));
    block_scan(n, s_wave, &live);
    live = p.n_pages - live;
    int *hole = p.work, *mover = hole + (p.n_pages + 1) / 2 + 1, *to = hole + p.n_pages + 4;
    int nh = 0, nm = 0;
    for (int w0 = 0; w0 < words; w0 += kPgThreads) {
        const int w = w0 + tid;
        const unsigned u = w < words ? used_word(p, w) : 0u;
        const int below = live - w * 32;   // this word's pages below L
        const unsigned low = below >= 32 ? ~0u : below <= 0 ? 0u : (1u << below) - 1u;
        unsigned h = w < words ? ~u & low : 0u, m = u & ~low;
        const int left = p.n_pages - w * 32;   // the last word's bits past the end are no pages
        if (left < 32) m &= left <= 0 ? 0u : (1u << left) - 1u;
        int got;
        int r = nh + block_scan(__popc(h), s_wave, &got);
        nh += got;
        while (h) {
            hole[r++] = w * 32 + __ffs(h) - 1;
            h &= h - 1;
        }
        r = nm + block_scan(__popc(m), s_wave, &got);
        nm += got;
        while (m) {
            mover[r++] = w * 32 + __ffs(m) - 1;
            m &= m - 1;
        }
        if (w < words) p.used[w] = low;
    }
    __syncthreads();
    for (int k = tid; k < nm; k += kPgThreads) {
        const int h = hole[k], m = mover[k];
        to[m - live] = h;
        p.refs[h] = p.refs[m];
        p.refs[m] = 0;
    }
    if (tid == 0) {
        p.state[kStMove] = nm;
        p.state[kStLive] = live;
    }
}

__global__ __launch_bounds__(kCopyThreads) void pages_move(PoolView p, int pieces) {
    const int moved = p.state[kStMove], live = p.state[kStLive];
    if (!moved) return;
    const int *hole = p.work, *mover = hole + (p.n_pages + 1) / 2 + 1, *to = hole + p.n_pages + 4;
    const long tasks = (long)moved * pieces;
    for (long t = blockIdx.x; t < tasks; t += gridDim.x) {
        const int k = (int)(t / pieces);
        copy_page(p, mover[k], hole[k], p.page, (int)(t % pieces), pieces);
    }
    for (int s = blockIdx.x; s < p.n_seqs; s += gridDim.x) {
        const int np = min(pages_of(p.lens[s], p.page), p.max_pages);
        int *row = p.table + (size_t)s * p.max_pages;
        for (int j = threadIdx.x; j < np; j += kCopyThreads) {
            const int pg = row[j];
            if (pg >= p.n_pages || pg < 0)
                atomicOr(&p.state[kStErr], kPgPage);
            else if (pg >= live)
                row[j] = to[pg - live];
        }
    }
}

// ---------------------------------------------------------------- a new pool
__global__ __launch_bounds__(256) void pages_clear(PoolView p) {
    const size_t i0 = blockIdx.x * 256 + threadIdx.x, step = (size_t)gridDim.x * 256;
    for (size_t i = i0; i < (size_t)p.n_seqs * p.max_pages; i += step) p.table[i] = -1;
    for (size_t i = i0; i < (size_t)p.n_seqs; i += step) p.lens[i] = grow_word(p, (int)i) = 0;
    for (size_t i = i0; i < (size_t)p.n_pages; i += step) p.refs[i] = 0;
    for (size_t i = i0; i < (size_t)(p.n_pages + 31) / 32; i += step) p.used[i] = 0;
    for (size_t i = i0; i < COLI_HIP_PAGES_STATE; i += step) p.state[i] = 0;
}

// The error bits, taken in one step: attention on another stream may be setting more.
__global__ void pages_errors(PoolView p) { p.state[kStSeen] = atomicExch(&p.state[kStErr], 0); }

}  // namespace coli

using namespace coli;

COLI_API int coli_hip_pages_check(const ColiHipPages *p) {
    PoolView v;
    return pool_view(p, v) ? 1 : 0;
}

COLI_API size_t coli_hip_pages_work(const ColiHipPages *p) {
    return p && p->n_pages > 0 ? work_ints(p->n_pages) + (p->n_seqs > 0 ? p->n_seqs : 0) : 0;
}

COLI_API int coli_hip_pages_init(const ColiHipPages *p, void *stream_) {
    PoolView v;
    hipStream_t st;
    if (!pool_view(p, v) || !paged_stream(stream_, st)) return 0;
    const size_t most = (size_t)v.n_seqs * v.max_pages, all = most > (size_t)v.n_pages ? most : v.n_pages;
    const unsigned grid = (unsigned)(all / 256 + 1 < 2048 ? all / 256 + 1 : 2048);
    hipLaunchKernelGGL(pages_clear, dim3(grid), dim3(256), 0, st, v);
    return paged_launched("pages init") ? 1 : 0;
}

static bool take_args(const ColiHipPages *p, PoolView &v, const void *seq, int n) {
    if (!pool_view(p, v)) return false;
    if (n < 0 || n > kPgMaxN) return paged_refuse("more than 4096 sequences in a call");
    return !n || seq || paged_refuse("NULL sequence list");
}

static void take(const PoolView &v, const int *a, const int *b, const int *count, int n, int mode, hipStream_t st) {
    if (n <= kTakeN * 512 && v.n_pages <= 512 * 32 * 4)
        hipLaunchKernelGGL(pages_take<512>, dim3(1), dim3(512), 0, st, v, a, b, count, n, mode);
    else
        hipLaunchKernelGGL(pages_take<kPgThreads>, dim3(1), dim3(kPgThreads), 0, st, v, a, b, count, n, mode);
}

COLI_API int coli_hip_pages_append(const ColiHipPages *p, const int *d_seq, const int *d_count, int n, void *stream_) {
    PoolView v;
    hipStream_t st;
    if (!take_args(p, v, d_seq, n) || !paged_stream(stream_, st)) return 0;
    if (!n) return 1;
    take(v, d_seq, d_seq, d_count, n, kTakeAppend, st);
    return paged_launched("pages append") ? 1 : 0;
}

COLI_API int coli_hip_pages_fork(const ColiHipPages *p, const int *d_src, const int *d_dst, int n, int share,
                                 void *stream_) {
    PoolView v;
    hipStream_t st;
    if (!take_args(p, v, d_src && d_dst ? d_src : nullptr, n) || !paged_stream(stream_, st)) return 0;
    if (!n) return 1;
    take(v, d_src, d_dst, nullptr, n, share ? kTakeShare : kTakeCopy, st);
    const int pieces = pieces_of(v);
    // share: a page's pieces; copy: enough blocks for the whole card
    const long most = (65536 + n - 1) / n, want = share ? pieces : (8L * n_cu() + n - 1) / n, y = want < most ? want : most;
    hipLaunchKernelGGL(pages_fork_copy, dim3(n, (unsigned)y), dim3(kCopyThreads), 0, st, v, d_src, d_dst, share ? 1 : 0,
                       pieces);
    return paged_launched("pages fork") ? 1 : 0;
}

COLI_API int coli_hip_pages_free(const ColiHipPages *p, const int *d_seq, int n, void *stream_) {
    PoolView v;
    hipStream_t st;
    if (!take_args(p, v, d_seq, n) || !paged_stream(stream_, st)) return 0;
    if (!n) return 1;
    hipLaunchKernelGGL(pages_drop, dim3(n), dim3(kCopyThreads), 0, st, v, d_seq);
    return paged_launched("pages free") ? 1 : 0;
}

COLI_API int coli_hip_pages_compact(const ColiHipPages *p, void *stream_) {
    PoolView v;
    hipStream_t st;
    if (!pool_view(p, v) || !paged_stream(stream_, st)) return 0;
    hipLaunchKernelGGL(pages_plan, dim3(1), dim3(kPgThreads), 0, st, v);
    hipLaunchKernelGGL(pages_move, dim3(8 * n_cu()), dim3(kCopyThreads), 0, st, v, pieces_of(v));
    return paged_launched("pages compact") ? 1 : 0;
}

COLI_API int coli_hip_pages_status(const ColiHipPages *p, int *n_free, int *errors, void *stream_) {
    PoolView v;
    hipStream_t st;
    if (!pool_view(p, v) || !paged_stream(stream_, st)) return 0;
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(st, &cap) != hipSuccess || cap != hipStreamCaptureStatusNone)
        return paged_refuse("a status read in a captured stream") ? 1 : 0;
    const int words = (v.n_pages + 31) / 32;
    unsigned *h = (unsigned *)malloc((size_t)words * 4);
    if (!h) return 0;
    int err = 0;
    hipLaunchKernelGGL(pages_errors, dim3(1), dim3(1), 0, st, v);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess) e = hipMemcpyAsync(h, v.used, (size_t)words * 4, hipMemcpyDeviceToHost, st);
    if (e == hipSuccess) e = hipMemcpyAsync(&err, v.state + kStSeen, 4, hipMemcpyDeviceToHost, st);
    if (e == hipSuccess) e = hipStreamSynchronize(st);
    int fr = 0;
    for (int w = 0; e == hipSuccess && w < words; w++) {
        const int left = v.n_pages - w * 32;
        fr += __builtin_popcount(~h[w] & (left < 32 ? (1u << left) - 1u : ~0u));
    }
    free(h);
    if (e != hipSuccess) return fail("pages status", e) ? 1 : 0;
    if (n_free) *n_free = fr;
    if (errors) *errors = err;
    return 1;
}
