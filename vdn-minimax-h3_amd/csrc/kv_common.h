// What the kernels of the 8-bit key/value cache share: the cache and batch arguments, which
// sequence a unit of work belongs to, and the scales' exponents.
#pragma once

#include <stdint.h>

#include "vdn_common.h"

namespace vdn {

constexpr int kPage = VDN_FP8_KV_PAGE;

// Exponents of a page's scale. The least one is what a page of zeros gets: far enough below
// every real scale, and such that 2^100 times a page's sum of weights stays in binary32.
constexpr int kLeastScale = -100, kMostScale = 120;

struct KvCacheArgs {
    uint8_t* k;          // e4m3 [pages, heads, 64, d]
    uint8_t* v;          // e4m3 [pages, heads, d, 64]
    uint8_t* k_scale;    // e8m0 [pages, heads]
    uint8_t* v_scale;
    uint16_t* k_mean;    // bf16 [pages, heads, d] or NULL
    int64_t pages;
    int heads, d;
};

struct KvBatchArgs {
    const int32_t* table;      // [batch, width], row stride ldtable
    int64_t ldtable;
    int width;                 // pages of the longest sequence the table holds
    const int32_t* lengths;    // [batch], the call's tokens included
    const int32_t* q_start;    // [batch + 1] or NULL: tokens / batch each
    int batch;
    int64_t tokens;            // < 2^31
    int each;                  // tokens of every sequence, where q_start is NULL
};

// Sequence b of the batch: its rows [start, start + n) of the call (clamped into it), the position
// of the first of them (negative where the sequence is shorter than its rows), and its tokens in the
// cache, no more than its table holds.
struct KvSequence {
    int64_t start, first;
    int n, length;
};

__device__ __forceinline__ KvSequence kv_sequence(const KvBatchArgs& p, int b)
{
    KvSequence s;
    if (p.q_start) {
        const int64_t lo = min(max((int64_t)p.q_start[b], (int64_t)0), p.tokens);
        const int64_t hi = min(max((int64_t)p.q_start[b + 1], lo), p.tokens);
        s.start = lo;
        s.n = (int)(hi - lo);
    } else {
        s.n = p.each;
        s.start = (int64_t)b * p.each;
    }
    const int64_t length = max((int64_t)p.lengths[b], (int64_t)0);
    s.first = length - s.n;
    s.length = (int)min(length, (int64_t)p.width * kPage);
    return s;
}

// Work is handed out in units of `size` rows of one sequence (`mult` rows a token), and the host
// knows the tokens of the call alone, not those of each sequence. Unit numbers are spread so that
// sequence b's begin at floor(mult start / size) + more b: n tokens take at most
// floor(mult n / size) + 1 units of rows (more = 1), or that many + 1 where the rows begin inside a
// unit, as the pages of a cache do (more = 2), so they never reach the next sequence's, and all fit
// mult tokens / size + more batch. Without q_start every sequence has `each` units. The host keeps
// tokens * mult and the units below 2^31.
struct KvUnits {
    uint32_t size, each;
    int mult, more;
};

__device__ __forceinline__ uint32_t kv_first_unit(const KvBatchArgs& p, const KvUnits& u, int b)
{
    return (uint32_t)(min(max(p.q_start[b], 0), (int)p.tokens) * u.mult) / u.size + (uint32_t)(u.more * b);
}

// The sequence that a unit belongs to, and its number `at` within it; with q_start, the batch's
// size stands for the rows behind the last sequence.
__device__ __forceinline__ int kv_locate(const KvBatchArgs& p, const KvUnits& u, uint32_t unit, uint32_t& at)
{
    if (!p.q_start) {
        const uint32_t b = unit / u.each;
        at = unit - b * u.each;
        return (int)b;
    }
    // The sequences that do not begin behind the unit, counted 64 at a time by the wave (all of it is here).
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int b0 = 0; b0 <= p.batch; b0 += 64) {
        const int b = b0 + lane;
        const uint64_t before = __ballot(b <= p.batch && kv_first_unit(p, u, min(b, p.batch)) <= unit);
        n += __builtin_popcountll(before);
        if (before != ~0ull) break;
    }
    const int b = max(n - 1, 0);
    at = unit - kv_first_unit(p, u, b);
    return b;
}

inline int64_t kv_unit_count(const KvBatchArgs& p, const KvUnits& u)
{
    return p.q_start ? p.tokens * u.mult / u.size + (int64_t)u.more * p.batch : (int64_t)u.each * p.batch;
}

// The pool page of page w of sequence b, -1 where the table's entry is outside the pool.
__device__ __forceinline__ int kv_page(const KvBatchArgs& p, const KvCacheArgs& c, int b, int w)
{
    const int page = p.table[(int64_t)b * p.ldtable + w];
    return page >= 0 && page < c.pages ? page : -1;
}

// Host: the checks that every entry point makes, and the two argument structs. Returns a status.
int kv_arguments(const char* what, const vdn_fp8_kv_cache* c, const vdn_fp8_kv_batch* b, KvCacheArgs& cache, KvBatchArgs& batch);

}  // namespace vdn
