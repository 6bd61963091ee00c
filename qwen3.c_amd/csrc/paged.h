// paged.h - the paged key-value cache as its kernels see it (pages.hip, paged.hip).
#pragma once

#include "../../include/coli_hip.h"
#include "internal.h"

namespace coli {

// Error bits of a pool, gathered in state[kStErr] until coli_hip_pages_status reads them.
enum {
    kPgFull = 1,      // not enough free pages
    kPgRow = 2,       // a sequence longer than its table row
    kPgIndex = 4,     // a sequence number or count out of range
    kPgTwice = 8,     // a sequence twice in one call, or a fork into one that is not empty
    kPgPos = 16,      // a position past the sequence's end
    kPgPage = 32,     // a table entry that is no page
};
// Words of the pool's state: the error bits; what a bookkeeping kernel leaves to the copy
// kernel behind it on the stream (go; pages to move, pages in use); the error bits that a status call took.
enum { kStErr = 0, kStGo = 1, kStMove = 2, kStLive = 3, kStSeen = 4 };

// ColiHipPages with its derived strides, by value to every kernel.
struct PoolView {
    char *data;
    int *table, *lens, *refs;
    unsigned *used;
    int *state, *work;
    int es;                       // bytes of a value
    int n_layers, KH, hd, page, n_pages, n_seqs, max_pages;
    long row_bytes, head_bytes, kv_bytes, layer_bytes, page_bytes;
};

// ColiHipHeads as the kernels take it.
struct HeadsView {
    int H, rot, interleaved;
    long q_row, q_head, kv_row;
    float eps, mag, scale;
    const float *qn, *kn, *freq;
};

// Scratch of `work` in ints; behind it a word per sequence.  The word is refused_at(len) after a call that
// was to grow the sequence at that length and was refused; no other call leaves that value for a length it
// gives the sequence.
constexpr size_t work_ints(int n_pages) { return 2 * (size_t)n_pages + 64; }
__device__ __forceinline__ int refused_at(int len) { return len ^ (int)0xA5C35A3Cu; }
__device__ __forceinline__ int &grow_word(const PoolView &p, int s) { return p.work[work_ints(p.n_pages) + s]; }

// The last position that row n sees (-1: none), and its sequence (-1: no row).  kNew: the row brings that
// position's keys and values; without pos it has none (-2) when its sequence was refused the place for it.
template <bool kNew = false>
__device__ __forceinline__ int row_pos(const PoolView &p, const int *seq, const int *pos, int n, int &s) {
    s = seq[n];
    if (s < 0 || s >= p.n_seqs) {
        if (s != -1) atomicOr(&p.state[kStErr], kPgIndex);
        s = -1;
        return -1;
    }
    const int word = kNew && !pos ? grow_word(p, s) : 0;
    const int len = min(max(p.lens[s], 0), p.max_pages * p.page), at = pos ? pos[n] : len - 1;
    if (kNew && !pos && word == refused_at(len)) {
        atomicOr(&p.state[kStErr], kPgPos);
        return -2;
    }
    if (at < len && at >= -1) return at;
    atomicOr(&p.state[kStErr], at < -1 ? kPgIndex : kPgPos);
    return at < -1 ? -2 : -3 - len;   // -2: no position; -3 - len: past the end
}

// Workgroup barrier for LDS alone: __syncthreads() also waits for every load in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// What the wave's lanes wrote to LDS is there for its other lanes.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
}

// false, with a message, when the description is outside what the kernels take (host only)
bool pool_view(const ColiHipPages *p, PoolView &v);
// the stream of a call and whether it can run: device usable and current
bool paged_stream(void *stream, hipStream_t &st);
bool paged_refuse(const char *why);
bool paged_launched(const char *what);   // no error of the launches before it

// The attention of n rows (paged_attn.hip) on device pointers, and the bytes of its workspace.
size_t attn_paged_work(const PoolView &p);
bool attn_paged(const PoolView &p, const HeadsView &h, int dtype, int layer, const float *q, const float *gate,
                const int *seq, const int *pos, int n, int max_len, float *out, void *work, hipStream_t st);

}  // namespace coli
