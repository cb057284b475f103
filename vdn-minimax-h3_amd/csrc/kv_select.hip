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
// page means' bytes (2 d a page and head, 1/64 of the cache) and the latency of two launches. 3120 queries in
// blocks of 128 over 512 pages, 40 heads of 128: 8.3 + 7.5 + 7.8 us; eight single queries of 40 heads over
// up to 2048 pages of 8: 9.2 + 6.6 us.
//   k_kv_query_sum   one workgroup per block and head
//   k_kv_scores      one wave per 16 pages, all blocks of the sequence, 16 at a time
//   k_kv_scores_step both of these where each query has its own pages
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
    int row_turns;       // workgroups of k_kv_scores that share the blocks of a sequence
    int32_t* blocks;     // [rows, heads, top]
    double* score;       // [rows, heads, width]
    float* sum;          // [rows, heads, d]
};

// Row `row` of the list: its sequence, the tokens [from, to) of it that make the block. False: none.
__device__ __forceinline__ bool block_of(const KvSelectArgs& p, int64_t row, int& b, KvSequence& s, int& from, int& to)
{
    uint32_t at;
    b = kv_locate(p.b, p.listed, (uint32_t)row, at, s);
    if (b == p.b.batch) return false;
    if ((int64_t)at * p.query_block >= s.n) return false;
    from = (int)at * p.query_block;
    to = min(from + p.query_block, s.n);
    return true;
}

// Lane exchanges of binary64 within rows of 16 lanes.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v)
{
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = dpp_u32<CTRL>((uint32_t)u), hi = dpp_u32<CTRL>((uint32_t)(u >> 32));
    return __longlong_as_double((int64_t)((uint64_t)hi << 32 | lo));
}

// Sum of the lanes up to and including this one, over the wave: within rows of 16 lanes by shifts, then the
// last lanes of the rows before.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v)
{
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);   // row_shr 1
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);   // 2
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);   // 4
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);   // 8
    const uint32_t r0 = __builtin_amdgcn_readlane(v, 15), r1 = __builtin_amdgcn_readlane(v, 31), r2 = __builtin_amdgcn_readlane(v, 47);
    const int row = (threadIdx.x & 63) / 16;
    return v + (row > 0 ? r0 : 0) + (row > 1 ? r1 : 0) + (row > 2 ? r2 : 0);
}

// Adds eight elements.
template <bool F16>
__device__ __forceinline__ void add8(uint4 v, double sum[8])
{
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
        add8<F16>(*reinterpret_cast<const uint4*>(p.q + token * p.ldq + (int64_t)(h * p.group + i % p.group) * d + 8 * ch), sum);
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
    const int b = blockIdx.z / p.row_turns, h = blockIdx.y;
    const KvSequence s = kv_sequence(p.b, b);
    const int have = (s.length + kPage - 1) / kPage;
    const int w0 = (blockIdx.x * 4 + wave) * 16;
    if (w0 >= have || s.n == 0) return;
    const int w = w0 + lane % 16, g = lane / 16;
    // (a page that is not there: any page's mean, as k_kv_top passes it over)
    const int page = max(kv_page(p.b, p.c, b, min(w, have - 1)), 0);
    uint32_t mean[E / 2];
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
        const uint4 v = *reinterpret_cast<const uint4*>(p.c.k_mean + ((int64_t)page * p.c.heads + h) * D + g * E + 8 * i);
        mean[4 * i] = v.x, mean[4 * i + 1] = v.y, mean[4 * i + 2] = v.z, mean[4 * i + 3] = v.w;
    }
    const int blocks = (s.n + p.query_block - 1) / p.query_block;
    const int64_t row0 = p.b.q_start ? (int64_t)kv_first_unit(p.b, p.listed, b) : (int64_t)b * p.listed.each;
    for (int r0 = 16 * (blockIdx.z % p.row_turns); r0 < blocks; r0 += 16 * p.row_turns) {
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

// One query (its group's heads) against all pages of its sequence, where each query has its own pages: 16
// lanes a page, eight elements each. The matrix instruction would use one of its 16 rows: 64 cycles for four
// products of 16 pages, where four fma here take 16 for four pages.
template <int D, bool F16>
__global__ __launch_bounds__(kThreads) void k_kv_scores_step(KvSelectArgs p)
{
    constexpr int L = D / 8, kPages = 64 / L, kSweeps = 4;   // lanes of a page, pages of a sweep, sweeps of a wave
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = blockIdx.y;
    const int64_t row = blockIdx.z;   // the query
    int b, from, to;
    KvSequence s;
    if (!block_of(p, row, b, s, from, to)) return;
    const int have = (s.length + kPage - 1) / kPage;
    const int w0 = (blockIdx.x * 4 + wave) * (kPages * kSweeps) + lane / L, i0 = 8 * (lane % L);
    if (w0 - lane / L >= have) return;
    // (every load before any use, and none under a condition: each of its own would be a round trip to memory)
    const uint16_t* const src = p.q + (s.start + from) * p.ldq + (int64_t)h * p.group * D + i0;
    uint4 q0[8];
#pragma unroll
    for (int g = 0; g < 8; ++g) q0[g] = *reinterpret_cast<const uint4*>(src + (int64_t)min(g, p.group - 1) * D);
    int page[kSweeps];
#pragma unroll
    for (int j = 0; j < kSweeps; ++j) page[j] = max(kv_page(p.b, p.c, b, min(w0 + j * kPages, have - 1)), 0);
    uint4 mean[kSweeps];
#pragma unroll
    for (int j = 0; j < kSweeps; ++j)
        mean[j] = *reinterpret_cast<const uint4*>(p.c.k_mean + ((int64_t)page[j] * p.c.heads + h) * D + i0);
    double q[8] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int g = 0; g < 8; ++g)
        if (g < p.group) add8<F16>(q0[g], q);
    for (int g = 8; g < p.group; ++g) add8<F16>(*reinterpret_cast<const uint4*>(src + (int64_t)g * D), q);
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = (double)(float)q[e];
#pragma unroll
    for (int j = 0; j < kSweeps; ++j) {
        const uint32_t m[4] = {mean[j].x, mean[j].y, mean[j].z, mean[j].w};
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            sum = __builtin_fma(q[2 * e], (double)bf16_lo(m[e]), sum);
            sum = __builtin_fma(q[2 * e + 1], (double)bf16_hi(m[e]), sum);
        }
        sum += dpp_f64<kDppXor1>(sum);
        sum += dpp_f64<kDppXor2>(sum);
        sum += dpp_f64<kDppHalfMirror>(sum);
        if (L >= 16) sum += dpp_f64<kDppMirror>(sum);
        if (L == 32) sum += __shfl_xor(sum, 16, 64);
        const int w = w0 + j * kPages;
        if (lane % L == 0 && w < have) p.score[(row * p.c.heads + h) * p.b.width + w] = sum;
    }
}

// A score's bits, ordered as the scores are, above 0; NaN as -inf.
__device__ __forceinline__ uint64_t score_key(double v)
{
    if (v != v) v = -__builtin_inf();
    const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);   // -0 and 0 are one
    return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}

// HELD: at most kHeld * 256 pages, whose keys stay in registers; else they are read again in every pass.
// A pass counts one digit of the keys that share the digits before it, in LDS; the first wave finds the
// digit in which the last wanted key lies. What is taken then goes through bitmaps, whose bits in
// order are the pages in order.
template <bool HELD>
__global__ __launch_bounds__(kThreads) void k_kv_top(KvSelectArgs p)
{
    constexpr int kWords = kHeld * kThreads / 32;   // of a bitmap, one lane each
    static_assert(kWords == 64, "a wave reads a bitmap at once");
    __shared__ __attribute__((aligned(16))) uint32_t hist[8][256];
    __shared__ uint32_t picked[4];   // digit, how many of it are wanted, how many it has, keys counted in all
    __shared__ uint32_t above[kWords], same[kWords];
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
    auto key_of = [&](int w, int page, double v) -> uint64_t {   // 0: not to be taken
        return w >= have || page < 0 ? 0 : w < p.first || w >= have - p.last ? ~0ull : score_key(v);
    };
    auto key_at = [&](int w) {
        const int at = min(w, have - 1);
        return key_of(w, kv_page(p.b, p.c, b, at), score[at]);
    };
    const int turns = (have + kThreads - 1) / kThreads;
    uint64_t held[HELD ? kHeld : 1];
    if (HELD && have > 0) {   // (all loads before their uses)
        int page[kHeld];
        double v[kHeld];
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int at = min(tid + j * kThreads, have - 1);
            page[j] = kv_page(p.b, p.c, b, at), v[j] = score[at];
        }
#pragma unroll
        for (int j = 0; j < kHeld; ++j) held[j] = key_of(tid + j * kThreads, page[j], v[j]);
    }
    auto each = [&](auto f) {
        if (HELD) {
#pragma unroll
            for (int j = 0; j < kHeld; ++j)
                if (j < turns) f(held[j]);
        } else {
            for (int j = 0; j < turns; ++j) f(key_at(tid + j * kThreads));
        }
    };
#pragma unroll
    for (int i = 0; i < 8; ++i) hist[i][tid] = 0;
    __syncthreads();

    // Taken: the keys above `least`, and of those equal to it the first `equal`.
    uint64_t least = 0;
    uint32_t equal = 0, wanted = (uint32_t)p.top;
    uint64_t high = 0;
    for (int pass = 0; pass < 8; ++pass) {
        const int shift = 56 - 8 * pass;
        each([&](uint64_t k) {
            if (k != 0 && (pass == 0 || (k >> (shift + 8)) == (high >> (shift + 8)))) atomicAdd(&hist[pass][(k >> shift) & 255], 1u);
        });
        __syncthreads();
        if (wave == 0) {
            // lane l: digits 255 - 4 l and the three below it; what comes before them is what is larger
            const uint4 v = *reinterpret_cast<const uint4*>(&hist[pass][252 - 4 * lane]);
            const uint32_t n[4] = {v.w, v.z, v.y, v.x}, own = n[0] + n[1] + n[2] + n[3];
            const uint32_t run = wave_scan(own);
            uint32_t before = run - own;
            if (before < wanted && run >= wanted)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (before < wanted && before + n[i] >= wanted) picked[0] = 255 - 4 * lane - i, picked[1] = wanted - before, picked[2] = n[i];
                    before += n[i];
                }
            if (lane == 63) picked[3] = run;
        }
        __syncthreads();
        if (pass == 0 && picked[3] <= wanted) break;   // all that there are: least = 0
        high |= (uint64_t)picked[0] << shift;
        wanted = picked[1];
        least = high, equal = wanted;
        if (picked[2] == wanted) {   // the whole digit: every key from its least one on
            least = high - 1;
            equal = 0;
            break;
        }
    }
    // (high > 0 where the loop went past its first test, since every key counted has a bit of it or
    // more: 0 itself is no key)

    uint32_t taken = 0, equal_left = equal;
    for (int w0 = 0; w0 < have; w0 += kWords * 32) {
        if (w0) __syncthreads();   // the bitmaps before have been read
        if (tid < kWords) above[tid] = same[tid] = 0;
        __syncthreads();
        auto mark = [&](uint64_t k, int j) {
            const uint64_t more = __ballot(k > least), alike = __ballot(k == least && k != 0);
            // this wave's 64 pages of the turn: two words
            if (lane < 2) {
                above[8 * j + 2 * wave + lane] = (uint32_t)(more >> (32 * lane));
                same[8 * j + 2 * wave + lane] = (uint32_t)(alike >> (32 * lane));
            }
        };
        if (HELD) {
#pragma unroll
            for (int j = 0; j < kHeld; ++j)
                if (j < turns) mark(held[j], j);
        } else {
            for (int j = 0; j < kHeld && w0 + j * kThreads < have; ++j) mark(key_at(w0 + tid + j * kThreads), j);
        }
        __syncthreads();
        if (wave == 0) {
            uint32_t alike = same[lane], bits = above[lane], run = __builtin_popcount(alike);
            if (equal_left > 0) {   // (uniform)
                const uint32_t own = run;
                run = wave_scan(own);
                uint32_t room = equal_left > run - own ? equal_left - (run - own) : 0;   // of this word's
                while (alike && room) {
                    bits |= alike & (0u - alike);
                    alike &= alike - 1;
                    --room;
                }
                const uint32_t all = __builtin_amdgcn_readlane(run, 63);
                equal_left = equal_left > all ? equal_left - all : 0;
            }
            const uint32_t own = __builtin_popcount(bits);
            run = wave_scan(own);
            uint32_t at = taken + run - own;
            while (bits) {
                if (at < (uint32_t)p.top) out[at] = w0 + 32 * lane + __builtin_ctz(bits);
                bits &= bits - 1;
                ++at;
            }
            taken += __builtin_amdgcn_readlane(run, 63);
        }
    }
    if (wave == 0)
        for (int i = (int)taken + lane; i < p.top; i += 64) out[i] = -1;
}

// The list of a call without tokens.
__global__ __launch_bounds__(kThreads) void k_kv_no_blocks(KvSelectArgs p)
{
    for (int i = threadIdx.x; i < p.top; i += kThreads) p.blocks[(int64_t)blockIdx.x * p.top + i] = -1;
}

int select_arguments(const vdn_fp8_kv_cache* cache, const vdn_fp8_kv_batch* batch, int64_t q_heads, int64_t query_block, KvSelectArgs& p,
                     int64_t& bytes)
{
    const int st = kv_arguments("kv_select", cache, batch, p.c, p.b);
    if (st != VDN_FP8_OK) return st;
    if (q_heads < 1 || q_heads > (1 << 16) || q_heads % p.c.heads)
        return set_error(VDN_FP8_EINVAL, "kv_select: %lld query heads for %d key/value heads", (long long)q_heads, p.c.heads);
    p.group = (int)(q_heads / p.c.heads);
    if (p.b.tokens * q_heads >= ((int64_t)1 << 30))
        return set_error(VDN_FP8_EINVAL, "kv_select: %lld tokens of %lld heads, 2^30 rows at most", (long long)p.b.tokens, (long long)q_heads);
    if (query_block < 1 || query_block > (1 << 20) || (query_block > 1 && query_block * p.group % 128))
        return set_error(VDN_FP8_EINVAL, "kv_select: query_block must be 1, or such that query_block * group is a multiple of 128 "
                         "(got %lld with groups of %d)", (long long)query_block, p.group);
    if (p.b.batch > 65535) return set_error(VDN_FP8_EINVAL, "kv_select: batch above 65535");
    p.query_block = (int)query_block;
    const int64_t n = p.b.batch > 0 ? p.b.tokens / p.b.batch : 0;
    p.listed = KvUnits{(uint32_t)query_block, (uint32_t)((n + query_block - 1) / query_block), 1, query_block == 1 ? 0 : 1};
    p.rows = kv_unit_count(p.b, p.listed);   // (of a call without tokens too, where q_start gives each sequence one)
    if (p.rows * p.c.heads >= (1 << 24)) return set_error(VDN_FP8_EINVAL, "kv_select: %lld blocks of queries and heads, 2^24 at most", (long long)(p.rows * p.c.heads));
    if ((p.b.width + 63ll) / 64 * p.c.heads * p.b.batch >= (1 << 21))
        return set_error(VDN_FP8_EINVAL, "kv_select: 2^27 pages and heads of the page table at most");
    bytes = p.b.tokens == 0 ? 0 : p.rows * p.c.heads * (8 * (int64_t)p.b.width + 4 * p.c.d);
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
    if ((!query && p.b.tokens > 0) || !blocks) return set_error(VDN_FP8_EINVAL, "kv_select: null pointer");
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
    if (p.b.tokens == 0) {
        hipLaunchKernelGGL(k_kv_no_blocks, per_row, block, 0, stream, p);
        return check_launch("kv_select");
    }
    const bool f16 = dtype == VDN_FP8_DTYPE_F16;
    const int64_t step_pages = 4 * 4 * (64 / (p.c.d / 8)), step_groups = (p.b.width + step_pages - 1) / step_pages;   // of k_kv_scores_step
    if (p.b.width > 0 && p.query_block == 1 && p.rows <= 65535 && step_groups * p.c.heads * p.rows < (1 << 24)) {
        const dim3 grid((unsigned)step_groups, (unsigned)p.c.heads, (unsigned)p.rows);
#define VDN_STEP(n)                                                                                         \
    case n:                                                                                                 \
        if (f16) hipLaunchKernelGGL((k_kv_scores_step<n, true>), grid, block, 0, stream, p);                \
        else hipLaunchKernelGGL((k_kv_scores_step<n, false>), grid, block, 0, stream, p);                   \
        break;
        switch (p.c.d) { VDN_STEP(64) VDN_STEP(128) VDN_STEP(256) }
#undef VDN_STEP
        const int launched = check_launch("kv_select scores");
        if (launched != VDN_FP8_OK) return launched;
    } else if (p.b.width > 0) {
        if (f16) hipLaunchKernelGGL((k_kv_query_sum<true>), per_row, block, 0, stream, p);
        else hipLaunchKernelGGL((k_kv_query_sum<false>), per_row, block, 0, stream, p);
        int launched = check_launch("kv_select query sum");
        if (launched != VDN_FP8_OK) return launched;
        const int64_t tiles = ((p.b.q_start ? p.b.tokens / query_block : (int64_t)p.listed.each) + 15) / 16, most = 65535 / p.b.batch;
        p.row_turns = (int)(tiles < 1 ? 1 : tiles < 8 ? tiles : 8);
        if (p.row_turns > most) p.row_turns = (int)most;
        const dim3 grid((unsigned)((p.b.width + 63) / 64), (unsigned)p.c.heads, (unsigned)(p.b.batch * p.row_turns));
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
