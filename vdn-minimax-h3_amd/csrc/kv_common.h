// What the kernels of the 8-bit key/value cache share: the cache and batch arguments, which
// sequence a unit of work belongs to, and the scales' exponents.
#pragma once

#include <stdint.h>

#include "vdn_common.h"

namespace vdn {

constexpr int kPage = VDN_FP8_KV_PAGE;

// Exponents of a page's scale. The least one is what a page of zeros gets: far enough below every real scale.
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

__device__ __forceinline__ KvSequence kv_sequence(const KvBatchArgs& p, int64_t start, int n, int length)
{
    const int64_t kept = max((int64_t)length, (int64_t)0);
    return KvSequence{start, kept - n, n, (int)min(kept, (int64_t)p.width * kPage)};
}

__device__ __forceinline__ int kv_start(const KvBatchArgs& p, int b) { return min(max(p.q_start[b], 0), (int)p.tokens); }

__device__ __forceinline__ KvSequence kv_sequence(const KvBatchArgs& p, int b)
{
    if (!p.q_start) return kv_sequence(p, (int64_t)b * p.each, p.each, p.lengths[b]);
    const int lo = kv_start(p, b), hi = max(kv_start(p, b + 1), lo);
    return kv_sequence(p, lo, hi - lo, p.lengths[b]);
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

__device__ __forceinline__ uint32_t kv_first_unit(const KvUnits& u, int start, int b) { return (uint32_t)(start * u.mult) / u.size + (uint32_t)(u.more * b); }

__device__ __forceinline__ uint32_t kv_first_unit(const KvBatchArgs& p, const KvUnits& u, int b) { return kv_first_unit(u, kv_start(p, b), b); }

// The sequence s that a unit belongs to, its number, and the unit's number `at` within it; with q_start, the
// batch's size stands for the rows behind the last sequence (and s for none).
__device__ __forceinline__ int kv_locate(const KvBatchArgs& p, const KvUnits& u, uint32_t unit, uint32_t& at, KvSequence& s)
{
    if (!p.q_start) {
        const int b = (int)(unit / u.each);
        at = unit - (uint32_t)b * u.each;
        s = kv_sequence(p, b);
        return b;
    }
    // The sequences that do not begin behind the unit, counted 64 at a time by the wave (all of it is here). The
    // last of them is at hand as a rule, its end in the next lane: one trip to memory instead of two.
    const int lane = threadIdx.x & 63;
    for (int b0 = 0;; b0 += 64) {
        const int own = min(b0 + lane, p.batch), start = kv_start(p, own), length = p.lengths[min(own, p.batch - 1)];
        const uint64_t before = __ballot(b0 + lane <= p.batch && kv_first_unit(u, start, own) <= unit);
        const int count = __builtin_popcountll(before);
        if (count == 64 && b0 + 64 <= p.batch) continue;
        const int b = max(b0 + count - 1, 0);
        if (count > 0 && count < 64) {
            const int lo = __builtin_amdgcn_readlane(start, count - 1), hi = max(__builtin_amdgcn_readlane(start, count), lo);
            at = unit - kv_first_unit(u, lo, b);
            s = kv_sequence(p, lo, hi - lo, __builtin_amdgcn_readlane(length, count - 1));
        } else {
            at = unit - kv_first_unit(p, u, b);
            if (b < p.batch) s = kv_sequence(p, b);
        }
        return b;
    }
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
