// Choosing the cache pages that a block of queries attends to.
//
// For each block of queries of a sequence and each key/value head, with s = the sum of the block's
// queries (tokens and heads of the group) rounded to binary32 once:
//   score[w] = s . k_mean[page w]
// and the `top` best pages, ties to the lower one, a few first and last ones in any case.
//
// A choice is a whole number: two programs that sum in different orders must still take the same
// pages. So everything up to the comparison is exact or nearly so: the query sum runs in binary64
// (bf16 terms of like size add exactly there), its products with bf16 means (24 + 8 bits) are exact in
// binary64, and their sum is off by 2^-50 or so. That costs nothing here: d products a page are four to
// five orders below the attention that follows, and the matrix cores take binary64.
//
// What bounds it: at many queries the query sum's bytes (each query read once); at single tokens the
// page means' bytes (2 d a page and head, 1/64 of the cache) and the latency of three launches.
//   k_kv_query_sum   one workgroup per block and head
//   k_kv_scores      one wave per 16 pages, all blocks of the sequence, 16 at a time
//   k_kv_top         one workgroup per block and head: radix selection on the scores' bits,
//                    eight bits a pass, until what is left of a digit is wanted as a whole
#include <stdint.h>

#include "kv_common.h"
#include "vdn_common.h"

namespace vdn {
namespace {

typedef double f64x4_t __attribute__((ext_vector_type(4)));
constexpr int kThreads = 256;
constexpr int kHeld = 8;              // scores that a thread of k_kv_top holds in registers

struct KvSelectArgs {
    KvCacheArgs c;
    KvBatchArgs b;
    KvUnits listed;
    int64_t rows;        // of the block list
    const uint16_t* q;
    int64_t ldq;
    int group, causal, query_block;
    int top, first, last;
    int32_t* blocks;     // [rows, heads, top]
    double* score;       // [rows, heads, width]
    float* sum;          // [rows, heads, d]
};

// Row `row` of the list: its sequence, the tokens [from, to) of it that make the block. False: none.
__device__ __forceinline__ bool block_of(const KvSelectArgs& p, int64_t row, int& b, KvSequence& s, int& from, int& to)
{
    int64_t at;
    b = kv_locate(p.b, p.listed, row, at);
    if (b == p.b.batch) return false;
    s = kv_sequence(p.b, b);
    if (at * p.query_block >= s.n) return false;
    from = (int)at * p.query_block;
    to = min(from + p.query_block, s.n);
    return true;
}

template <bool F16>
__global__ __launch_bounds__(kThreads) void k_kv_query_sum(KvSelectArgs p)
{
    __shared__ double part[kThreads * 8];
    const int d = p.c.d, chunks = d / 8, tid = threadIdx.x;
    const int64_t row = blockIdx.x / (uint32_t)p.c.heads;
    const int h = (int)(blockIdx.x % (uint32_t)p.c.heads);
    int b, from, to;
    KvSequence s;
    if (!block_of(p, row, b, s, from, to)) return;
    const int ch = tid % chunks, lanes = kThreads / chunks, n = (to - from) * p.group;
    double sum[8] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
    for (int i = tid / chunks; i < n; i += lanes) {
        const int64_t token = s.start + from + i / p.group;
        const uint4 v = *reinterpret_cast<const uint4*>(p.q + token * p.ldq + (int64_t)(h * p.group + i % p.group) * d + 8 * ch);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (F16) {
                sum[2 * e] += (double)(float)__builtin_bit_cast(_Float16, (uint16_t)w[e]);
                sum[2 * e + 1] += (double)(float)__builtin_bit_cast(_Float16, (uint16_t)(w[e] >> 16));
            } else {
                sum[2 * e] += (double)bf16_lo(w[e]);
                sum[2 * e + 1] += (double)bf16_hi(w[e]);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) part[e * kThreads + tid] = sum[e];
    __syncthreads();
    for (int i = tid; i < d; i += kThreads) {
        double total = 0.0;
        for (int g = 0; g < lanes; ++g) total += part[(i % 8) * kThreads + g * chunks + i / 8];
        p.sum[(row * p.c.heads + h) * d + i] = (float)total;
    }
}

// One wave: 16 pages of one sequence and head, against all of its blocks. The matrix instruction's
// inner index runs over four lane groups; group g takes elements [g d / 4, (g + 1) d / 4), so that a lane
// reads them contiguously.
template <int D>
__global__ __launch_bounds__(kThreads) void k_kv_scores(KvSelectArgs p)
{
    constexpr int E = D / 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = blockIdx.z, h = blockIdx.y;
    const KvSequence s = kv_sequence(p.b, b);
    const int have = (s.length + kPage - 1) / kPage;
    const int w0 = (blockIdx.x * 4 + wave) * 16;
    if (w0 >= have || s.n == 0) return;
    const int w = w0 + lane % 16, g = lane / 16;
    const int page = w < have ? kv_page(p.b, p.c, b, w) : -1;
    uint32_t mean[E / 2];
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (page >= 0) v = *reinterpret_cast<const uint4*>(p.c.k_mean + ((int64_t)page * p.c.heads + h) * D + g * E + 8 * i);
        mean[4 * i] = v.x, mean[4 * i + 1] = v.y, mean[4 * i + 2] = v.z, mean[4 * i + 3] = v.w;
    }
    const int blocks = (s.n + p.query_block - 1) / p.query_block;
    const int64_t row0 = p.b.q_start ? kv_first_unit(p.b, p.listed, b) : (int64_t)b * p.listed.each;
    for (int r0 = 0; r0 < blocks; r0 += 16) {
        const int r = min(r0 + lane % 16, blocks - 1);
        const float4* const src = reinterpret_cast<const float4*>(p.sum + ((row0 + r) * p.c.heads + h) * D + g * E);
        f64x4_t acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
            const float4 q = src[i];
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)q.x, (double)bf16_lo(mean[2 * i]), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)q.y, (double)bf16_hi(mean[2 * i]), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)q.z, (double)bf16_lo(mean[2 * i + 1]), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)q.w, (double)bf16_hi(mean[2 * i + 1]), acc, 0, 0, 0);
        }
        // acc[i]: block row 4 i + lane / 16, page lane % 16
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = r0 + 4 * i + lane / 16;
            if (at < blocks && w < have) p.score[((row0 + at) * p.c.heads + h) * p.b.width + w] = acc[i];
        }
    }
}

// A score's bits, ordered as the scores are, above 0; NaN as -inf.
__device__ __forceinline__ uint64_t score_key(double v)
{
    if (v != v) v = -__builtin_inf();
    const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);   // -0 and 0 are one
    return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}

template <bool HELD>
__global__ __launch_bounds__(kThreads) void k_kv_top(KvSelectArgs p)
{
    __shared__ uint32_t hist[256];
    __shared__ uint32_t wave_sum[4];
    __shared__ uint32_t picked[3];   // digit, how many of it are wanted, how many it has
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / (uint32_t)p.c.heads;
    const int h = (int)(blockIdx.x % (uint32_t)p.c.heads);
    int32_t* const out = p.blocks + (row * p.c.heads + h) * p.top;
    int b, from, to;
    KvSequence s;
    int have = 0;
    if (block_of(p, row, b, s, from, to)) {
        const int seen = p.causal ? (int)min(max(s.first + to, (int64_t)0), (int64_t)s.length) : s.length;
        have = (seen + kPage - 1) / kPage;
    }
    const double* const score = p.score + (row * p.c.heads + h) * p.b.width;
    const int turns = (have + kThreads - 1) / kThreads;
    auto key_at = [&](int w) -> uint64_t {
        if (w >= have || kv_page(p.b, p.c, b, w) < 0) return 0;
        if (w < p.first || w >= have - p.last) return ~0ull;
        return score_key(score[w]);
    };
    uint64_t held[HELD ? kHeld : 1];
    if (HELD)
#pragma unroll
        for (int j = 0; j < kHeld; ++j) held[j] = j < turns ? key_at(tid + j * kThreads) : 0;
    // (a thread's scores: pages tid, tid + 256, ...)
    auto each = [&](auto f) {
        if (HELD) {
#pragma unroll
            for (int j = 0; j < kHeld; ++j)
                if (j < turns) f(held[j], j);
        } else {
            for (int j = 0; j < turns; ++j) f(key_at(tid + j * kThreads), j);
        }
    };
    // sum over the workgroup of what comes before this thread's value, and in all
    auto prefix = [&](uint32_t v, uint32_t& all) {
        uint32_t run = v;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t t = __shfl_up(run, off, 64);
            if (lane >= off) run += t;
        }
        __syncthreads();
        if (lane == 63) wave_sum[wave] = run;
        __syncthreads();
        uint32_t before = run - v;
        all = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i < wave) before += wave_sum[i];
            all += wave_sum[i];
        }
        return before;
    };

    uint32_t candidates = 0;
    {
        uint32_t mine = 0;
        each([&](uint64_t k, int) { mine += k != 0; });
        prefix(mine, candidates);
    }
    // The least key that is taken (`least`), and how many of those equal to it: all but at the end.
    uint64_t least = 1;
    uint32_t equal = ~0u, wanted = (uint32_t)p.top;
    if (candidates > wanted) {
        uint64_t high = 0;
        for (int shift = 56;; shift -= 8) {
            hist[tid] = 0;
            __syncthreads();
            const uint64_t mask = shift == 56 ? 0 : ~0ull << (shift + 8);
            each([&](uint64_t k, int) {
                if (k != 0 && (k & mask) == high) atomicAdd(&hist[(k >> shift) & 255], 1u);
            });
            __syncthreads();
            // thread t: digit 255 - t, so that what comes before it is what is larger
            const uint32_t own = hist[255 - tid];
            uint32_t all;
            const uint32_t before = prefix(own, all);
            if (before < wanted && before + own >= wanted) picked[0] = 255 - tid, picked[1] = wanted - before, picked[2] = own;
            __syncthreads();
            high |= (uint64_t)picked[0] << shift;
            wanted = picked[1];
            const bool whole = picked[2] == wanted;
            __syncthreads();
            if (whole || shift == 0) {
                least = high;
                equal = whole ? ~0u : wanted;   // (at shift 0: the first `wanted` of the equal ones)
                break;
            }
        }
    }
    // In ascending order: pages of a turn come before those of the next.
    uint32_t taken = 0, equal_before = 0;
    auto turn = [&](uint64_t k, int j) {
        const bool same = equal != ~0u && k == least;
        uint32_t all;
        uint32_t n = 0;
        if (equal != ~0u) {   // (uniform)
            n = equal_before + prefix(same, all);
            equal_before += all;
        }
        const bool take = k != 0 && (equal == ~0u ? k >= least : k > least || (same && n < equal));
        const uint32_t at = taken + prefix(take, all);
        taken += all;
        if (take && at < (uint32_t)p.top) out[at] = tid + j * kThreads;
    };
    each(turn);
    for (int i = (int)taken + tid; i < p.top; i += kThreads) out[i] = -1;
}

int select_arguments(const vdn_fp8_kv_cache* cache, const vdn_fp8_kv_batch* batch, int64_t q_heads, int64_t query_block, KvSelectArgs& p,
                     int64_t& bytes)
{
    const int st = kv_arguments("kv_select", cache, batch, p.c, p.b);
    if (st != VDN_FP8_OK) return st;
    if (q_heads < 1 || q_heads > (1 << 16) || q_heads % p.c.heads)
        return set_error(VDN_FP8_EINVAL, "kv_select: %lld query heads for %d key/value heads", (long long)q_heads, p.c.heads);
    p.group = (int)(q_heads / p.c.heads);
    if (query_block < 1 || query_block > (1 << 20) || (query_block > 1 && query_block * p.group % 128))
        return set_error(VDN_FP8_EINVAL, "kv_select: query_block must be 1, or such that query_block * group is a multiple of 128 "
                         "(got %lld with groups of %d)", (long long)query_block, p.group);
    if (p.b.batch > 65535) return set_error(VDN_FP8_EINVAL, "kv_select: batch above 65535");
    p.query_block = (int)query_block;
    const int64_t n = p.b.batch > 0 ? p.b.tokens / p.b.batch : 0;
    p.listed = KvUnits{query_block, (n + query_block - 1) / query_block, 1, query_block == 1 ? 0 : 1};
    p.rows = p.b.tokens == 0 ? 0 : kv_unit_count(p.b, p.listed);
    if (p.rows * p.c.heads >= (1 << 24)) return set_error(VDN_FP8_EINVAL, "kv_select: %lld blocks of queries and heads, 2^24 at most", (long long)(p.rows * p.c.heads));
    if ((p.b.width + 63ll) / 64 * p.c.heads * p.b.batch >= (1 << 24))
        return set_error(VDN_FP8_EINVAL, "kv_select: 2^30 pages and heads of the page table at most");
    bytes = p.rows * p.c.heads * (8 * (int64_t)p.b.width + 4 * p.c.d);
    return VDN_FP8_OK;
}

}  // namespace
}  // namespace vdn

using namespace vdn;

extern "C" int vdn_fp8_kv_select_workspace_size(const vdn_fp8_kv_cache* cache, const vdn_fp8_kv_batch* batch, int64_t q_heads,
                                                int64_t query_block, int64_t* bytes)
{
    KvSelectArgs p{};
    if (!bytes) return set_error(VDN_FP8_EINVAL, "kv_select_workspace_size: null pointer");
    *bytes = 0;
    return select_arguments(cache, batch, q_heads, query_block, p, *bytes);
}

extern "C" int vdn_fp8_kv_select(const vdn_fp8_kv_cache* cache, const vdn_fp8_kv_batch* batch, const void* query, int dtype, int64_t q_heads,
                                 int64_t ldq, int causal, int64_t top, int64_t first, int64_t last, int64_t query_block, int32_t* blocks,
                                 void* workspace, int64_t workspace_bytes, hipStream_t stream)
{
    KvSelectArgs p{};
    int64_t bytes = 0;
    if (dtype != VDN_FP8_DTYPE_BF16 && dtype != VDN_FP8_DTYPE_F16) return set_error(VDN_FP8_EINVAL, "kv_select: dtype must be bf16 or binary16");
    const int st = select_arguments(cache, batch, q_heads, query_block, p, bytes);
    if (st != VDN_FP8_OK || p.rows == 0) return st;
    if (!query || !blocks) return set_error(VDN_FP8_EINVAL, "kv_select: null pointer");
    if (p.c.pages > 0 && !p.c.k_mean) return set_error(VDN_FP8_EINVAL, "kv_select: the cache keeps no k_mean");
    if (top < 1 || top > (1 << 24) || first < 0 || last < 0 || first + last > top)
        return set_error(VDN_FP8_EINVAL, "kv_select: need top >= 1, first and last >= 0, first + last <= top");
    if (ldq % 8 || ldq < q_heads * p.c.d) return set_error(VDN_FP8_EINVAL, "kv_select: need ldq a multiple of 8 and >= q_heads * head_dim");
    if (!aligned(query, 16) || !aligned(blocks, 4) || !aligned(workspace, 16))
        return set_error(VDN_FP8_EINVAL, "kv_select: misaligned pointer (query, workspace 16 B; blocks 4 B)");
    if (bytes > 0 && (!workspace || workspace_bytes < bytes))
        return set_error(VDN_FP8_EINVAL, "kv_select: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)bytes);
    p.q = (const uint16_t*)query, p.ldq = ldq, p.causal = causal != 0;
    p.top = (int)top, p.first = (int)first, p.last = (int)last, p.blocks = blocks;
    p.sum = (float*)workspace;   // (a multiple of 256 bytes)
    p.score = (double*)(p.sum + p.rows * p.c.heads * p.c.d);
    const dim3 block(kThreads), per_row((unsigned)(p.rows * p.c.heads));
    if (p.b.width > 0) {
        if (dtype == VDN_FP8_DTYPE_F16) hipLaunchKernelGGL((k_kv_query_sum<true>), per_row, block, 0, stream, p);
        else hipLaunchKernelGGL((k_kv_query_sum<false>), per_row, block, 0, stream, p);
        int launched = check_launch("kv_select query sum");
        if (launched != VDN_FP8_OK) return launched;
        const dim3 grid((unsigned)((p.b.width + 63) / 64), (unsigned)p.c.heads, (unsigned)p.b.batch);
        switch (p.c.d) {
            case 64: hipLaunchKernelGGL((k_kv_scores<64>), grid, block, 0, stream, p); break;
            case 128: hipLaunchKernelGGL((k_kv_scores<128>), grid, block, 0, stream, p); break;
            default: hipLaunchKernelGGL((k_kv_scores<256>), grid, block, 0, stream, p); break;
        }
        launched = check_launch("kv_select scores");
        if (launched != VDN_FP8_OK) return launched;
    }
    if (p.b.width <= kHeld * kThreads) hipLaunchKernelGGL((k_kv_top<true>), per_row, block, 0, stream, p);
    else hipLaunchKernelGGL((k_kv_top<false>), per_row, block, 0, stream, p);
    return check_launch("kv_select top");
}
