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
// kernel behind it on the stream (go; pages to move, pages in use).
enum { kStErr = 0, kStGo = 1, kStMove = 2, kStLive = 3 };

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

// false, with a message, when the description is outside what the kernels take (host only)
bool pool_view(const ColiHipPages *p, PoolView &v);
// the stream of a call and whether it can run: device usable and current
bool paged_stream(void *stream, hipStream_t &st);
bool paged_refuse(const char *why);

}  // namespace coli
