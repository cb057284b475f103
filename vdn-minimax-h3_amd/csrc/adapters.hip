// Low-rank adapters of many requests beside a shared projection:
//
//   out[t][n] = round(base[t][n] + scale[i] * sum_r h[t][r] B[i][n][r]),   h[t][r] = sum_k x[t][k] A[i][r][k],   i = index[t]
//   out[t]    = base[t] where index[t] is outside [0, L)
//
// in two launches: k_shrink_* write h, binary32, in S parts summed over disjoint ranges of k; k_expand_* add the parts and
// the second product to the base. A step of few tokens is one launch (k_few). All are bound by memory (2 R operations for
// each element of x and of base, R <= 128), so the matrix cores have time to spare: h is not rounded to 16 bits between the
// products but goes in as two of them, a high and a low part, which lose 2^-17 of it at most and cost the second product twice over
// (1 us of 79 at 6470 tokens, 5376 -> 7168, rank 128).
//
// On the card: 32760 tokens, 5120 -> 15360, rank 64: 72 + 377 us, 5.2 TB/s of the bytes that it cannot do without (a large copy
// reaches 5.1); 6470 tokens of six requests, 5376 -> 7168, rank 128: 32 + 53 us, 3.3 TB/s; 32 tokens of 12 adapters, 5120 -> 7168, rank 32:
// 14 us; one token of rank 16, 5120 -> 5120: 4.6 us.
//
// Which tokens share an adapter. A tile is 64 consecutive tokens; a wave holds their adapters one a lane and finds the distinct
// ones by ballots, so nothing is sorted, nothing is read back to the host, and a call can be captured into a graph and replayed
// with another index. The tokens of one adapter in a tile are packed into columns of matrix products, 16 at a time. A batch whose
// requests are runs of tokens has one or two adapters a tile; in a step of single tokens the adapters of a tile are dealt out to
// `slots` workgroups.
#include <stdint.h>

#include "eight.h"
#include "vdn_common.h"

namespace vdn {
namespace {

constexpr int kLanes = 64;
constexpr int kTile = 64;         // tokens of a tile: a lane's each
constexpr int kMostRank = 128;
constexpr uint32_t kDies = 8;     // of the card, each with an L2 of its own
constexpr uint32_t kOutside = 0xfffffff0u;   // an offset outside every buffer: reads zero, stores nothing

typedef float f32x4_t __attribute__((ext_vector_type(4)));

template <int TYPE>
struct Mma;
template <>
struct Mma<kBf16> {
    typedef __bf16 Vec __attribute__((ext_vector_type(8)));
    __device__ __forceinline__ static f32x4_t mma(uint4 a, uint4 b, f32x4_t c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Vec, a), __builtin_bit_cast(Vec, b), c, 0, 0, 0);
    }
};
template <>
struct Mma<kF16> {
    typedef _Float16 Vec __attribute__((ext_vector_type(8)));
    __device__ __forceinline__ static f32x4_t mma(uint4 a, uint4 b, f32x4_t c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(Vec, a), __builtin_bit_cast(Vec, b), c, 0, 0, 0);
    }
};

struct AdapterArgs {
    const uint8_t* x;
    int64_t ldx;               // elements, as every stride
    const uint8_t* base;
    int64_t ldbase;
    uint8_t* out;
    int64_t ldo;
    const uint8_t* a;          // [L, R, K]
    const uint8_t* b;          // [L, N, R]
    const float* scale;        // [L]
    const int32_t* index;      // [T]
    int64_t T;
    int K, N, L, R;
    float* part;               // [tiles, S, 64, R]
    int S;                     // parts of h
    int slots;                 // workgroups that the adapters of a tile are dealt out to
    int blocks;                // ranges of k (k_shrink) or of n (k_expand) of a tile
    int span;                  // k of a part (k_shrink), or columns of a workgroup (k_expand)
    int copy;                  // out is not base: tokens without an adapter are copied
    int once;                  // out is so large that it only passes through the caches
};

template <int POL = 0>
__device__ __forceinline__ uint4 load16(__amdgpu_buffer_rsrc_t buffer, uint32_t off)
{
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(buffer, off, 0, POL));
}

// The adapters of a tile, one after the other, as the masks of their tokens.
struct Groups {
    int mine;            // this lane's token's adapter, or -1
    uint64_t left;
    uint64_t mask;
    int adapter;
    __device__ __forceinline__ Groups(const AdapterArgs& p, int64_t tile)
    {
        const int64_t t = tile * kTile + (threadIdx.x & (kLanes - 1));
        const int i = t < p.T ? p.index[t] : -1;
        mine = i >= 0 && i < p.L ? i : -1;
        left = __ballot(mine >= 0);
    }
    __device__ __forceinline__ bool next()
    {
        if (!left) return false;
        adapter = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
        mask = __ballot(mine == adapter);
        left &= ~mask;
        return true;
    }
};

// The tokens of a mask in order: list[i] is the i-th one's place in the tile. The list is the wave's own.
__device__ __forceinline__ int list_tokens(uint64_t mask, int* list)
{
    const int lane = threadIdx.x & (kLanes - 1);
    __builtin_amdgcn_wave_barrier();
    if (mask >> lane & 1) list[__builtin_popcountll(mask & ((1ull << lane) - 1))] = lane;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    return __builtin_popcountll(mask);
}

// ---------------------------------------------------------------------------
// h = x A^T
// ---------------------------------------------------------------------------

// One step of 64 k, 128 bytes of each row: a lane's 16 bytes of it for each of two products.
template <int RF, int TF>
struct ShrinkStep {
    uint4 a[RF][2], x[TF][2];
};

template <int RF, int TF>
__device__ __forceinline__ void load_step(ShrinkStep<RF, TF>& s, __amdgpu_buffer_rsrc_t ar, __amdgpu_buffer_rsrc_t xr, const uint32_t (&arow)[RF],
                                          const uint32_t (&xrow)[TF], int k, int end)
{
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        // (a row's last chunks may lie past the range: both read zero there)
        const int at = k + 32 * h;
        const bool in = at < end;
#pragma unroll
        for (int f = 0; f < TF; ++f) s.x[f][h] = load16(xr, in && xrow[f] != kOutside ? xrow[f] + 2u * at : kOutside);
#pragma unroll
        for (int r = 0; r < RF; ++r) s.a[r][h] = load16(ar, in && arow[r] != kOutside ? arow[r] + 2u * at : kOutside);
    }
}

// The sums of 16 RF ranks from `rank` on for the tokens [16 f0, 16 (f0 + TF)) of the list, over k from k0 to end.
template <int TYPE, int RF, int TF>
__device__ __forceinline__ void shrink_tokens(const AdapterArgs& p, int64_t tile, int adapter, const int* list, int count, int f0, int rank, int k0,
                                              int end, f32x4_t (&acc)[RF][2])
{
    const int lane = threadIdx.x & (kLanes - 1), col = lane & 15, quad = lane >> 4;
    const int64_t rows = min(p.T - tile * kTile, (int64_t)kTile);
    const __amdgpu_buffer_rsrc_t xr = row_buffer(p.x + tile * kTile * p.ldx * 2, ((rows - 1) * p.ldx + p.K) * 2);
    const __amdgpu_buffer_rsrc_t ar = row_buffer(p.a + (int64_t)adapter * p.R * p.K * 2, (int64_t)p.R * p.K * 2);
    uint32_t arow[RF], xrow[TF];
#pragma unroll
    for (int r = 0; r < RF; ++r) {
        const int at = rank + 16 * r + col;
        arow[r] = at < p.R ? (uint32_t)at * (uint32_t)p.K * 2u : kOutside;
    }
#pragma unroll
    for (int f = 0; f < TF; ++f) {
        const int at = 16 * (f0 + f) + col;
        xrow[f] = at < count ? (uint32_t)list[at] * (uint32_t)p.ldx * 2u : kOutside;
    }
    auto use = [&](const ShrinkStep<RF, TF>& s) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < RF; ++r)
#pragma unroll
                for (int f = 0; f < TF; ++f) acc[r][f] = Mma<TYPE>::mma(s.a[r][h], s.x[f][h], acc[r][f]);
    };
    ShrinkStep<RF, TF> even, odd;
    int k = k0 + 8 * quad;
    const int steps = (end - k0 + 63) / 64;
    load_step<RF, TF>(even, ar, xr, arow, xrow, k, end);
    for (int i = 0; i < steps; i += 2) {
        load_step<RF, TF>(odd, ar, xr, arow, xrow, k + 64, end);
        use(even);
        load_step<RF, TF>(even, ar, xr, arow, xrow, k + 128, end);
        use(odd);
        k += 128;
    }
}

// A step of single tokens: WK waves share the tokens and take other ranges of the workgroup's k, and their sums meet in LDS: the
// upper half of them hands its sums to the lower half until one is left.
template <int TYPE, int RF, int WK>
__global__ __launch_bounds__(WK * kLanes) void k_shrink_step(AdapterArgs p)
{
    __shared__ int lists[WK][kTile];
    __shared__ f32x4_t sums[WK / 2][RF][2][kLanes];
    const int wk = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const int lane = threadIdx.x & (kLanes - 1), col = lane & 15, quad = lane >> 4;
    const uint32_t block = blockIdx.x / (uint32_t)p.blocks, part = blockIdx.x % (uint32_t)p.blocks;
    const int64_t tile = block / (uint32_t)p.slots;
    const int slot = (int)(block % (uint32_t)p.slots);
    const int own = p.span / WK;
    const int k0 = (int)part * p.span + wk * own, end = min(p.K, k0 + own);
    const int rank = blockIdx.y * 16 * RF;
    int* list = lists[wk];
    Groups groups(p, tile);
    for (int g = 0; groups.next(); ++g) {
        if (g % p.slots != slot) continue;
        const int count = list_tokens(groups.mask, list);
        for (int f = 0; f * 16 < count; f += 2) {   // (the same rounds in every wave)
            f32x4_t acc[RF][2];
#pragma unroll
            for (int r = 0; r < RF; ++r) acc[r][0] = acc[r][1] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (f * 16 + 16 < count) shrink_tokens<TYPE, RF, 2>(p, tile, groups.adapter, list, count, f, rank, k0, end, acc);
            else shrink_tokens<TYPE, RF, 1>(p, tile, groups.adapter, list, count, f, rank, k0, end, acc);
#pragma unroll
            for (int w = WK / 2; w > 0; w /= 2) {
                if (wk >= w && wk < 2 * w)
#pragma unroll
                    for (int r = 0; r < RF; ++r)
#pragma unroll
                        for (int t = 0; t < 2; ++t) sums[wk - w][r][t][lane] = acc[r][t];
                __syncthreads();
                if (wk < w)
#pragma unroll
                    for (int r = 0; r < RF; ++r)
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const f32x4_t v = sums[wk][r][t][lane];
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[r][t][e] += v[e];
                        }
                __syncthreads();
            }
            if (wk > 0) continue;
            // column = token, rows 4 quad .. 4 quad + 3 = ranks
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int at = 16 * (f + t) + col;
                if (at >= count) continue;
                float* h = p.part + ((tile * p.S + part) * kTile + list[at]) * p.R + rank + 4 * quad;
#pragma unroll
                for (int r = 0; r < RF; ++r)
                    if (rank + 16 * r < p.R) *reinterpret_cast<f32x4_t*>(h + 16 * r) = acc[r][t];
            }
            settle_stores();
        }
    }
}

// Many tokens: a workgroup of four waves takes a tile, 16 tokens a wave and all ranks (R = 16 RF). A matrix operand has 16 rows in 16 neighbouring
// lanes, and read from memory like that every lane of a quarter wave touches a line of its own (the step's kernels, which read so, take two to five times as
// long: figures at kStepTokens). So both go through LDS: kBk consecutive k of 64 tokens and of R ranks are loaded
// as whole lines into registers, one step ahead. Chunk c of 16
// bytes of a row lies at c ^ (row % 16): rows' writes and columns' reads both spread over all banks.
constexpr int kWaves = 4;
constexpr int kBk = 128;
constexpr int kRowChunks = kBk / 8;

template <int TYPE, int RF>
__global__ __launch_bounds__(kWaves * kLanes) void k_shrink_tile(AdapterArgs p)
{
    constexpr int kRows = kTile + 16 * RF, kEach = kRows / 16;   // a thread's loads
    __shared__ int lists[kWaves][kTile];
    __shared__ uint4 buffer[kRows][kRowChunks];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const int lane = threadIdx.x & (kLanes - 1), col = lane & 15, quad = lane >> 4;
    const int64_t tile = blockIdx.x / (uint32_t)p.blocks;
    const int part = (int)(blockIdx.x % (uint32_t)p.blocks);
    const int k0 = part * p.span, end = min(p.K, k0 + p.span);
    const int steps = (end - k0 + kBk - 1) / kBk;
    int* list = lists[wave];
    const int64_t rows = min(p.T - tile * kTile, (int64_t)kTile);
    const __amdgpu_buffer_rsrc_t xr = row_buffer(p.x + tile * kTile * p.ldx * 2, ((rows - 1) * p.ldx + p.K) * 2);
    // this thread's chunks: rows threadIdx / kRowChunks + 16 i, all at one place of the row
    const int mine = threadIdx.x % kRowChunks, row0 = threadIdx.x / kRowChunks;
    Groups groups(p, tile);
    for (int g = 0; groups.next(); ++g) {
        if (g % p.slots != (int)blockIdx.y) continue;
        const int count = list_tokens(groups.mask, list);
        const __amdgpu_buffer_rsrc_t ar = row_buffer(p.a + (int64_t)groups.adapter * p.R * p.K * 2, (int64_t)p.R * p.K * 2);
        uint32_t from[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int row = row0 + 16 * i;
            if (16 * i < kTile) from[i] = row < count ? (uint32_t)list[row] * (uint32_t)p.ldx * 2u : kOutside;
            else from[i] = (uint32_t)(row - kTile) * (uint32_t)p.K * 2u;
        }
        uint4 held[kEach];
        auto load = [&](int step) {
            const int k = k0 + step * kBk + 8 * mine;
#pragma unroll
            for (int i = 0; i < kEach; ++i) held[i] = 16 * i < kTile ? load16<2>(xr, k < end && from[i] != kOutside ? from[i] + 2u * k : kOutside) : load16(ar, k < end && from[i] != kOutside ? from[i] + 2u * k : kOutside);
        };
        auto store = [&]() {
#pragma unroll
            for (int i = 0; i < kEach; ++i) buffer[row0 + 16 * i][mine ^ row0] = held[i];
        };
        f32x4_t acc[RF];
#pragma unroll
        for (int r = 0; r < RF; ++r) acc[r] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        __syncthreads();   // (the buffer's rows of the tile's adapter before)
        load(0);
        store();
        __syncthreads();
        for (int step = 0; step < steps; ++step) {
            load(step + 1);   // (past the end: zeros, not used)
            if (16 * wave < count) {
#pragma unroll
                for (int s = 0; s < kRowChunks / 4; ++s) {
                    const uint4 x = buffer[16 * wave + col][(4 * s + quad) ^ col];
#pragma unroll
                    for (int r = 0; r < RF; ++r) acc[r] = Mma<TYPE>::mma(buffer[kTile + 16 * r + col][(4 * s + quad) ^ col], x, acc[r]);
                }
            }
            __syncthreads();
            store();
            __syncthreads();
        }
        const int at = 16 * wave + col;
        if (at < count) {
            float* h = p.part + ((tile * p.S + part) * kTile + list[at]) * p.R + 4 * quad;
#pragma unroll
            for (int r = 0; r < RF; ++r) *reinterpret_cast<f32x4_t*>(h + 16 * r) = acc[r];
        }
        settle_stores();
    }
}

// ---------------------------------------------------------------------------
// out = base + scale h B^T
// ---------------------------------------------------------------------------

constexpr float kMostBf16 = 0x1.fep127f;

// Eight ranks of h as two operands of eight 16-bit values, high and low part. bf16: h rounded to nearest and what that leaves, 2^-8 of
// it at most, rounded likewise: 2^-17 of h is lost at most (a high part of truncated words would leave 2^-7, and lose 2^-16).
// float16: relative to the power of two 2^e above the token's largest, e back in the result, so that no h is too large
// for it; 2^-24 of that power of two is lost at most, whatever the size of h.
template <int TYPE>
__device__ __forceinline__ void split8(const float (&h)[8], float down, uint4& high, uint4& low)
{
    uint32_t a[4], b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (TYPE == kBf16) {
            const float v0 = h[2 * e], v1 = h[2 * e + 1];
            const bool in0 = __builtin_isfinite(v0), in1 = __builtin_isfinite(v1);
            // (what would round to infinity takes bf16's largest; an infinity leaves nothing: the difference would be NaN)
            a[e] = pack_bf16x2(in0 ? fminf(fmaxf(v0, -kMostBf16), kMostBf16) : v0, in1 ? fminf(fmaxf(v1, -kMostBf16), kMostBf16) : v1);
            b[e] = pack_bf16x2(in0 ? v0 - bf16_lo(a[e]) : 0.0f, in1 ? v1 - bf16_hi(a[e]) : 0.0f);
        } else {
            f16x2_t hi, lo;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float v = h[2 * e + i], s = v * down;
                // (beside an infinity the others keep to float16's range, for their signs)
                hi[i] = (_Float16)(__builtin_isfinite(v) ? fminf(fmaxf(s, -65504.0f), 65504.0f) : v);
                lo[i] = __builtin_isfinite((float)hi[i]) ? (_Float16)(fminf(fmaxf(s, -65504.0f), 65504.0f) - (float)hi[i]) : (_Float16)0.0f;
            }
            a[e] = __builtin_bit_cast(uint32_t, hi);
            b[e] = __builtin_bit_cast(uint32_t, lo);
        }
    }
    high = make_uint4(a[0], a[1], a[2], a[3]);
    low = make_uint4(b[0], b[1], b[2], b[3]);
}

// h of a token (its ranks 32 r + 8 (lane / 16) .. + 7 in this lane) as operands; up: what the products have to be multiplied by (float16).
template <int TYPE, int RK>
__device__ __forceinline__ void split_h(const float (&h)[RK][8], uint4 (&high)[RK], uint4 (&low)[RK], float& up)
{
    float down = 1.0f;
    up = 1.0f;
    if (TYPE == kF16) {
        float most = 0.0f;
#pragma unroll
        for (int r = 0; r < RK; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) most = __builtin_fmaxf(most, __builtin_fabsf(h[r][e]));
        most = __builtin_fmaxf(most, __shfl_xor(most, 16, kLanes));
        most = __builtin_fmaxf(most, __shfl_xor(most, 32, kLanes));
        // 2^e above the largest, e in the range in which 2^-e and 2^e are normal
        const int e = most > 0.0f && __builtin_isfinite(most) ? min(max((int)(__float_as_uint(most) >> 23) - 126, -120), 120) : 0;
        down = __uint_as_float((uint32_t)(127 - e) << 23);
        up = __uint_as_float((uint32_t)(127 + e) << 23);
    }
#pragma unroll
    for (int r = 0; r < RK; ++r) split8<TYPE>(h[r], down, high[r], low[r]);
}

// Part s of the h of a tile's tokens.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t part_buffer(const AdapterArgs& p, int64_t tile, int s)
{
    return row_buffer(p.part + (tile * p.S + s) * kTile * p.R, (int64_t)kTile * p.R * 4);
}

// The same of a tile's token (-1: zeros) from memory, its parts added.
template <int TYPE, int RK>
__device__ __forceinline__ void load_h(const AdapterArgs& p, int64_t tile, int token, uint4 (&high)[RK], uint4 (&low)[RK], float& up)
{
    const int quad = (threadIdx.x & (kLanes - 1)) >> 4;
    float h[RK][8];
    uint32_t from[RK];
#pragma unroll
    for (int r = 0; r < RK; ++r) {
        const int rank = 32 * r + 8 * quad;
        from[r] = token >= 0 && rank < p.R ? ((uint32_t)token * (uint32_t)p.R + rank) * 4u : kOutside;
#pragma unroll
        for (int e = 0; e < 8; ++e) h[r][e] = 0.0f;
    }
    // (two parts at a time, all their loads ahead of the first sum)
    for (int s = 0; s < p.S; s += 2) {
        const __amdgpu_buffer_rsrc_t part[2] = {part_buffer(p, tile, s), part_buffer(p, tile, s + 1 < p.S ? s + 1 : s)};
        uint4 v[2][RK][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < RK; ++r) {
                const bool in = from[r] != kOutside && s + i < p.S;
                v[i][r][0] = load16(part[i], in ? from[r] : kOutside);
                v[i][r][1] = load16(part[i], in ? from[r] + 16u : kOutside);
            }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < RK; ++r)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const f32x4_t u = __builtin_bit_cast(f32x4_t, v[i][r][half]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) h[r][4 * half + e] += u[e];
                }
    }
    split_h<TYPE, RK>(h, high, low, up);
}

// A step of 64 columns: both halves of a 128-byte line of a token's row.
template <int RK, int TF>
struct ExpandStep {
    uint4 b[2][2][RK], base[2][TF];
};

// RK: steps of 32 ranks.
template <int TYPE, int RK, int TF>
__device__ __forceinline__ void expand_tokens(const AdapterArgs& p, int64_t tile, int adapter, const int* list, int count, int f0, int n0, int end)
{
    const int lane = threadIdx.x & (kLanes - 1), col = lane & 15, quad = lane >> 4;
    const int64_t rows = min(p.T - tile * kTile, (int64_t)kTile);
    const __amdgpu_buffer_rsrc_t baser = row_buffer(p.base + tile * kTile * p.ldbase * 2, ((rows - 1) * p.ldbase + p.N) * 2);
    const __amdgpu_buffer_rsrc_t outr = row_buffer(p.out + tile * kTile * p.ldo * 2, ((rows - 1) * p.ldo + p.N) * 2);
    const __amdgpu_buffer_rsrc_t br = row_buffer(p.b + (int64_t)adapter * p.N * p.R * 2, (int64_t)p.N * p.R * 2);
    const float scale = p.scale[adapter];
    uint32_t baserow[TF], outrow[TF];
    int token[TF];
#pragma unroll
    for (int f = 0; f < TF; ++f) {
        const int at = 16 * (f0 + f) + col;
        token[f] = at < count ? list[at] : -1;
        baserow[f] = token[f] >= 0 ? (uint32_t)token[f] * (uint32_t)p.ldbase * 2u : kOutside;
        outrow[f] = token[f] >= 0 ? (uint32_t)token[f] * (uint32_t)p.ldo * 2u : kOutside;
    }
    // B's rows as the first operand, so that a column of the result is a token; row i of product h is column
    // n + 8 (i / 4) + 4 h + i % 4: a lane holds eight consecutive columns of its token.
    const uint32_t brow = (uint32_t)(8 * (col / 4) + col % 4) * (uint32_t)p.R * 2u + 16u * quad;
    auto load = [&](ExpandStep<RK, TF>& s, int n) {
#pragma unroll
        for (int f = 0; f < TF; ++f)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int at = n + 32 * c + 8 * quad;
                s.base[c][f] = load16(baser, at < end && token[f] >= 0 ? baserow[f] + 2u * at : kOutside);
            }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < RK; ++r)
                    s.b[c][h][r] = load16(br, 32 * r + 8 * quad < p.R && n + 32 * c < end ? brow + (uint32_t)(n + 32 * c + 4 * h) * (uint32_t)p.R * 2u + 64u * r : kOutside);
    };
    ExpandStep<RK, TF> step;
    load(step, n0);   // (in flight while h is fetched)

    uint4 high[TF][RK], low[TF][RK];
    float up[TF];
#pragma unroll
    for (int f = 0; f < TF; ++f) load_h<TYPE, RK>(p, tile, token[f], high[f], low[f], up[f]);
    auto use = [&](const ExpandStep<RK, TF>& s, int n) {
#pragma unroll
        for (int f = 0; f < TF; ++f) {
            i32x4_t o[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                f32x4_t acc[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    acc[h] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int r = 0; r < RK; ++r) {
                        acc[h] = Mma<TYPE>::mma(s.b[c][h][r], high[f][r], acc[h]);
                        acc[h] = Mma<TYPE>::mma(s.b[c][h][r], low[f][r], acc[h]);
                    }
                }
                float v[8];
                Eight<TYPE> e8;
                e8.w[0] = s.base[c][f];
                decode8<TYPE>(e8, v);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[4 * h + e] = __builtin_fmaf(TYPE == kF16 ? acc[h][e] * up[f] : acc[h][e], scale, v[4 * h + e]);
                o[c] = __builtin_bit_cast(i32x4_t, encode8<TYPE>(v).w[0]);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int at = n + 32 * c + 8 * quad;
                __builtin_amdgcn_raw_buffer_store_b128(o[c], outr, at < end && token[f] >= 0 ? outrow[f] + 2u * at : kOutside, 0, 0);
            }
            settle_stores();
        }
    };
    for (int n = n0; n < end; n += 64) {
        use(step, n);
        load(step, n + 64);
    }
}

// The rows of a mask's tokens, columns n0 to end, by one wave of `waves`.
__device__ __forceinline__ void copy_tokens(const AdapterArgs& p, int64_t tile, const int* list, int count, int wave, int waves, int n0, int end)
{
    const int lane = threadIdx.x & (kLanes - 1);
    for (int i = wave; i < count; i += waves) {
        const int64_t t = tile * kTile + __builtin_amdgcn_readfirstlane(list[i]);
        const __amdgpu_buffer_rsrc_t from = row_buffer(p.base + t * p.ldbase * 2, (int64_t)end * 2), to = row_buffer(p.out + t * p.ldo * 2, (int64_t)end * 2);
        for (int n = n0 + 8 * lane; n < end; n += 8 * kLanes) store_b128_settled<0>(__builtin_bit_cast(i32x4_t, load16(from, 2u * n)), to, 2u * n, 0);
    }
}

// A step of single tokens: each of the waves takes its own columns of the tile's tokens.
template <int TYPE, int RK>
__global__ __launch_bounds__(kWaves * kLanes) void k_expand_step(AdapterArgs p)
{
    __shared__ int lists[kWaves][kTile];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes), lane = threadIdx.x & (kLanes - 1);
    const uint32_t block = blockIdx.x / (uint32_t)p.blocks, range = blockIdx.x % (uint32_t)p.blocks;
    const int64_t tile = block / (uint32_t)p.slots;
    const int slot = (int)(block % (uint32_t)p.slots);
    const int own = p.span / kWaves;
    const int n0 = (int)range * p.span + wave * own, end = min(p.N, n0 + own);
    Groups groups(p, tile);
    const uint64_t none = __ballot(tile * kTile + lane < p.T && groups.mine < 0);
    int g = 0;
    for (; groups.next(); ++g) {
        if (g % p.slots != slot) continue;
        const int count = list_tokens(groups.mask, lists[wave]);
        for (int f = 0; f * 16 < count; f += 2) {
            if (f * 16 + 16 < count) expand_tokens<TYPE, RK, 2>(p, tile, groups.adapter, lists[wave], count, f, n0, end);
            else expand_tokens<TYPE, RK, 1>(p, tile, groups.adapter, lists[wave], count, f, n0, end);
        }
    }
    if (p.copy && none && g % p.slots == slot) {
        const int count = list_tokens(none, lists[wave]);
        copy_tokens(p, tile, lists[wave], count, 0, 1, n0, end);
    }
}

// Many tokens: a workgroup takes a tile, 16 tokens a wave, 128 columns a step. h is the first operand here (a row of the result is a token)
// and B the second, column j of product f being column 8 j + f: a lane has eight consecutive columns of a token and 16 neighbouring
// lanes 256 consecutive bytes of its row, so that base and out are read and written as whole lines. B's 128 rows go through LDS, loaded as whole
// lines one step ahead: chunk c of row n lies at 17 (n % 8) + n / 8 of the plane of chunk c, the order in which product n % 8 reads it,
// planes being spaced so that the writes, rows of neighbouring lanes, spread over the banks as well. (Conflicts are 0.38 to 0.48 of the LDS's
// cycles all the same, and those 0.2 of the time.)
constexpr int kBn = 128;
// An out of at least this many bytes, the last-level cache's, is stored non-temporally (32760 x 15360, rank 64: 442 us a call against 463).
constexpr int64_t kOnceBytes = 256ll << 20;

// h of 16 tokens of a wave, its parts added, rows of neighbouring lanes: binary32, a row padded by a chunk.
template <int RF>
__device__ __forceinline__ void gather_h(const AdapterArgs& p, int64_t tile, const int* list, int count, int row0, f32x4_t* to)
{
    constexpr int kChunks = 4 * RF;
    const int lane = threadIdx.x & (kLanes - 1);
    f32x4_t sum[RF];
    uint32_t from[RF];
#pragma unroll
    for (int i = 0; i < RF; ++i) {
        const int row = (lane + kLanes * i) / kChunks, c = (lane + kLanes * i) % kChunks;
        sum[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        from[i] = row0 + row < count ? ((uint32_t)list[row0 + row] * (uint32_t)p.R + 4u * c) * 4u : kOutside;
    }
    // (two parts at a time, all their loads ahead of the first sum: left to itself the compiler may wait for each)
    for (int s = 0; s < p.S; s += 2) {
        const __amdgpu_buffer_rsrc_t part = part_buffer(p, tile, s), other = part_buffer(p, tile, s + 1 < p.S ? s + 1 : s);
        uint4 v[2][RF];
#pragma unroll
        for (int i = 0; i < RF; ++i) {
            v[0][i] = load16(part, from[i]);
            v[1][i] = load16(other, s + 1 < p.S ? from[i] : kOutside);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < RF; ++i) {
            sum[i] += __builtin_bit_cast(f32x4_t, v[0][i]);
            sum[i] += __builtin_bit_cast(f32x4_t, v[1][i]);
        }
    }
#pragma unroll
    for (int i = 0; i < RF; ++i) to[(lane + kLanes * i) / kChunks * (kChunks + 1) + (lane + kLanes * i) % kChunks] = sum[i];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// RF: 16 ranks each.
template <int TYPE, int RF>
__global__ __launch_bounds__(kWaves * kLanes) void k_expand_tile(AdapterArgs p)
{
    constexpr int RK = (RF + 1) / 2, kChunks = 2 * RF;                        // products of 32 ranks; 16-byte chunks of a row of B
    constexpr int kApart = kChunks == 2 ? 8 : kChunks == 4 ? 4 : kChunks == 8 ? 2 : 1;
    constexpr int kPlane = 8 * 17 + (kApart + 8) % 16;
    constexpr int kEach = kBn * kChunks / (kWaves * kLanes);                  // chunks of a thread
    constexpr int kHeld = 16 * (4 * RF + 1);                                  // of a wave's h
    constexpr int kSize = kWaves * kHeld > kChunks * kPlane ? kWaves * kHeld : kChunks * kPlane;
    __shared__ int lists[kWaves][kTile];
    __shared__ uint4 buffer[kSize];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const int lane = threadIdx.x & (kLanes - 1), col = lane & 15, quad = lane >> 4;
    // workgroups go to the eight dies in turn: those of one tile to the same die, whose L2 then reads the tile's h once
    const uint32_t turn = blockIdx.x / kDies;
    const int64_t tile = (int64_t)(turn / (uint32_t)p.blocks) * kDies + blockIdx.x % kDies;
    const int n0 = (int)(turn % (uint32_t)p.blocks) * p.span, end = min(p.N, n0 + p.span);
    if (tile * kTile >= p.T) return;
    const int steps = (end - n0 + kBn - 1) / kBn;
    int* list = lists[wave];
    const int64_t rows = min(p.T - tile * kTile, (int64_t)kTile);
    const __amdgpu_buffer_rsrc_t baser = row_buffer(p.base + tile * kTile * p.ldbase * 2, ((rows - 1) * p.ldbase + p.N) * 2);
    const __amdgpu_buffer_rsrc_t outr = row_buffer(p.out + tile * kTile * p.ldo * 2, ((rows - 1) * p.ldo + p.N) * 2);
    Groups groups(p, tile);
    const uint64_t none = __ballot(tile * kTile + lane < p.T && groups.mine < 0);
    int g = 0;
    for (; groups.next(); ++g) {
        if (g % p.slots != (int)blockIdx.y) continue;
        const int count = list_tokens(groups.mask, list);
        const __amdgpu_buffer_rsrc_t br = row_buffer(p.b + (int64_t)groups.adapter * p.N * p.R * 2, (int64_t)p.N * p.R * 2);
        const float scale = p.scale[groups.adapter];
        uint4 held[kEach];
        auto load_b = [&](int n) {   // (rows past the end are those of columns that are not stored)
#pragma unroll
            for (int i = 0; i < kEach; ++i) held[i] = load16(br, (uint32_t)n * (uint32_t)p.R * 2u + 16u * (threadIdx.x + kWaves * kLanes * i));
        };
        auto store_b = [&]() {
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int at = threadIdx.x + kWaves * kLanes * i, row = at / kChunks, c = at % kChunks;
                buffer[c * kPlane + (row % 8) * 17 + row / 8] = held[i];
            }
        };
        // the result's rows: tokens 4 quad + e of the wave's 16
        uint32_t brow[4], orow[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int at = 16 * wave + 4 * quad + e, token = at < count ? list[at] : -1;
            brow[e] = token >= 0 ? (uint32_t)token * (uint32_t)p.ldbase * 2u + 16u * col : kOutside;
            orow[e] = token >= 0 ? (uint32_t)token * (uint32_t)p.ldo * 2u + 16u * col : kOutside;
        }
        uint4 base[4];
        auto load_base = [&](int n) {
            const bool in = n + 8 * col < end;
#pragma unroll
            for (int e = 0; e < 4; ++e) base[e] = load16<kBufferLoadOnce>(baser, in && brow[e] != kOutside ? brow[e] + 2u * n : kOutside);
        };
        load_b(n0);
        load_base(n0);
        __syncthreads();   // (the buffer's rows of the tile's adapter before)
        f32x4_t* mine = reinterpret_cast<f32x4_t*>(buffer) + wave * kHeld;
        gather_h<RF>(p, tile, list, count, 16 * wave, mine);
        uint4 high[RK], low[RK];
        float up_row;
        {
            float h[RK][8];
#pragma unroll
            for (int r = 0; r < RK; ++r) {
                // (an odd number of 16 ranks: nothing in the last product's upper half)
                const bool in = 32 * r + 8 * quad < 16 * RF;
                const f32x4_t lo = mine[col * (4 * RF + 1) + (in ? 8 * r + 2 * quad : 0)], hi = mine[col * (4 * RF + 1) + (in ? 8 * r + 2 * quad + 1 : 0)];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    h[r][e] = in ? lo[e] : 0.0f;
                    h[r][4 + e] = in ? hi[e] : 0.0f;
                }
            }
            split_h<TYPE, RK>(h, high, low, up_row);
        }
        float up[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) up[e] = TYPE == kF16 ? __shfl(up_row, 4 * quad + e, kLanes) : 1.0f;
        __syncthreads();
        store_b();
        __syncthreads();
        for (int step = 0; step < steps; ++step) {
            const int n = n0 + step * kBn;
            load_b(n + kBn);
            if (16 * wave < count) {
                f32x4_t acc[8];
#pragma unroll
                for (int f = 0; f < 8; ++f) acc[f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
                // (columns of the next product under this one's: left to itself the compiler reads all eight ahead, 1% of a call's
                // time)
                uint4 v[2][RK];
                auto read = [&](uint4 (&to)[RK], int f) {
#pragma unroll
                    for (int r = 0; r < RK; ++r) {
                        const bool in = 4 * r + quad < kChunks;   // (constant but for the last product of an odd number of 16 ranks: zeros beside zeros)
                        to[r] = buffer[(in ? 4 * r + quad : 0) * kPlane + f * 17 + col];
                        if (RF % 2 && r == RK - 1 && !in) to[r] = make_uint4(0, 0, 0, 0);
                    }
                };
                read(v[0], 0);
#pragma unroll
                for (int f = 0; f < 8; ++f) {
                    if (f < 7) read(v[(f + 1) % 2], f + 1);
#pragma unroll
                    for (int r = 0; r < RK; ++r) {
                        acc[f] = Mma<TYPE>::mma(high[r], v[f % 2][r], acc[f]);
                        acc[f] = Mma<TYPE>::mma(low[r], v[f % 2][r], acc[f]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                i32x4_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    Eight<TYPE> e8;
                    e8.w[0] = base[e];
                    float v[8];
                    decode8<TYPE>(e8, v);
#pragma unroll
                    for (int f = 0; f < 8; ++f) v[f] = __builtin_fmaf(TYPE == kF16 ? acc[f][e] * up[e] : acc[f][e], scale, v[f]);
                    o[e] = __builtin_bit_cast(i32x4_t, encode8<TYPE>(v).w[0]);
                }
                load_base(n + kBn);
                const bool in = n + 8 * col < end;
                uint32_t to[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) to[e] = in && orow[e] != kOutside ? orow[e] + 2u * n : kOutside;
                if (p.once)
#pragma unroll
                    for (int e = 0; e < 4; ++e) __builtin_amdgcn_raw_buffer_store_b128(o[e], outr, to[e], 0, kBufferLoadOnce);
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e) __builtin_amdgcn_raw_buffer_store_b128(o[e], outr, to[e], 0, 0);
                settle_stores();
            }
            __syncthreads();
            store_b();
            __syncthreads();
        }
    }
    if (p.copy && none && g % p.slots == (int)blockIdx.y) {
        const int count = list_tokens(none, list);
        copy_tokens(p, tile, list, count, wave, kWaves, n0, end);
    }
}

// ---------------------------------------------------------------------------
// A step with few tokens of each adapter: both products in one launch
// ---------------------------------------------------------------------------

// A workgroup of 16 waves takes an adapter of the tile and 512 columns, and computes all of h for them again: A is at hand in the L2,
// and reading it (R K 2 bytes a workgroup) takes less than a second launch and h's way through memory. Up to eight tokens at a time, no
// matrix cores: with a few rows a product is bound by reading the other operand, and read along k by neighbouring lanes
// A comes as whole lines (as matrix operands, 16 rows in 16 lanes, it took four times as long). The tokens' x lie in
// LDS; a wave takes a rank at a time, sums in its lanes and then over them. B's rows are fetched at the start and put beside.
constexpr int kFewWaves = 16, kFewColumns = 512;
constexpr int kFewRank = 64, kFewK = 7168;              // (LDS: 8 tokens' x and 512 rows of B of 32 ranks, or 4 tokens' and 64)
constexpr int few_tokens(int rank_frags) { return rank_frags <= 2 ? 8 : 4; }

// acc + the products of eight elements. (binary16 by conversions and single fma: one token of rank 32 6.5 us against bf16's 6.3, eight of
// one adapter 18.4 against 12.9.)
template <int TYPE>
__device__ __forceinline__ float dot8(uint4 a, uint4 b, float acc)
{
    const uint32_t u[4] = {a.x, a.y, a.z, a.w}, v[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (TYPE == kBf16) {
            acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, u[e]), __builtin_bit_cast(bf16x2_t, v[e]), acc, false);
        } else {
            const f16x2_t p = __builtin_bit_cast(f16x2_t, u[e]), q = __builtin_bit_cast(f16x2_t, v[e]);
            acc = __builtin_fmaf((float)p[0], (float)q[0], acc);
            acc = __builtin_fmaf((float)p[1], (float)q[1], acc);
        }
    }
    return acc;
}

template <int TYPE>
__device__ __forceinline__ float to_float(uint16_t v)
{
    return TYPE == kBf16 ? bf16_to_f32(v) : (float)__builtin_bit_cast(_Float16, v);
}

template <int TYPE>
__device__ __forceinline__ uint16_t from_float(float v)
{
    return TYPE == kBf16 ? (uint16_t)pack_bf16x2(v, 0.0f) : __builtin_bit_cast(uint16_t, (_Float16)v);
}

// The sums of four values over the wave's 64 lanes: row 0 of 16 lanes gets v[0]'s, row 1 v[2]'s, row 2 v[1]'s, row 3 v[3]'s, each by the
// same tree. (Halves and rows are exchanged two values at a time, so four take one value's steps within the rows.)
__device__ __forceinline__ float sum_four(const float (&v)[4])
{
    auto add_swapped32 = [](float a, float b) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    };
    const float a = add_swapped32(v[0], v[1]), b = add_swapped32(v[2], v[3]);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    float s = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    s += __uint_as_float(dpp_u32<kDppXor1>(__float_as_uint(s)));
    s += __uint_as_float(dpp_u32<kDppXor2>(__float_as_uint(s)));
    s += __uint_as_float(dpp_u32<kDppHalfMirror>(__float_as_uint(s)));
    s += __uint_as_float(dpp_u32<kDppMirror>(__float_as_uint(s)));
    return s;
}

// h of TK tokens, whose x lie in LDS: this wave's ranks. (Two chunks of A in flight, and the code short: a workgroup runs each
// instruction a few times and waits for every line of them. With five or eight ahead the kernel took a fifth longer.)
template <int TYPE, int RF, int TK>
__device__ __forceinline__ void few_h(__amdgpu_buffer_rsrc_t ar, const uint4* x, int chunks, int wave, float (*h)[16 * RF])
{
    constexpr int kValues = (RF * TK + 3) / 4 * 4;
    const int lane = threadIdx.x & (kLanes - 1);
    float sum[kValues];
#pragma unroll
    for (int i = 0; i < kValues; ++i) sum[i] = 0.0f;
#pragma unroll 2
    for (int c = lane; c < chunks; c += kLanes) {
        uint4 a[RF];
#pragma unroll
        for (int r = 0; r < RF; ++r) a[r] = load16(ar, ((uint32_t)(wave + kFewWaves * r) * chunks + c) * 16u);
#pragma unroll
        for (int t = 0; t < TK; ++t) {
            const uint4 v = x[t * chunks + c];
#pragma unroll
            for (int r = 0; r < RF; ++r) sum[r * TK + t] = dot8<TYPE>(a[r], v, sum[r * TK + t]);
        }
    }
#pragma unroll
    for (int i = 0; i < kValues; i += 4) {
        const float four[4] = {sum[i], sum[i + 1], sum[i + 2], sum[i + 3]};
        const float v = sum_four(four);
        const int at = i + (lane == 16 ? 2 : lane == 32 ? 1 : lane == 48 ? 3 : 0);
        if (lane % 16 == 0 && at < RF * TK) h[at % TK][wave + kFewWaves * (at / TK)] = v;
    }
}

// RF: 16 ranks each.
template <int TYPE, int RF>
__global__ __launch_bounds__(kFewWaves * kLanes) void k_few(AdapterArgs p)
{
    constexpr int R = 16 * RF, kRowB = 2 * RF + 1;                       // chunks of a row of B in LDS, one of them padding
    constexpr int kEachB = kFewColumns * 2 * RF / (kFewWaves * kLanes);   // of a thread
    constexpr int kTokens = few_tokens(RF), kShare = kFewWaves / kTokens;  // waves that fetch a token's x
    __shared__ uint4 rows_b[kFewColumns * kRowB], rows_x[kTokens * kFewK / 8];
    __shared__ int lists[kFewWaves][kTile];
    __shared__ float h[kTokens][R];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes), lane = threadIdx.x & (kLanes - 1);
    // workgroups go to the eight dies in turn: those of one adapter to the same die, whose L2 then reads A once
    const uint32_t turn = blockIdx.x / kDies;
    const int n0 = (int)(turn % (uint32_t)p.blocks) * kFewColumns;
    const int slot = (int)(turn / (uint32_t)p.blocks * kDies + blockIdx.x % kDies);
    if (slot >= p.slots) return;
    const int chunks = p.K >> 3;
    int* list = lists[wave];
    Groups groups(p, 0);
    const uint64_t none = __ballot(lane < p.T && groups.mine < 0);
    int g = 0;
    for (; groups.next(); ++g) {
        if (g % p.slots != slot) continue;
        const int count = list_tokens(groups.mask, list);
        const __amdgpu_buffer_rsrc_t ar = row_buffer(p.a + (int64_t)groups.adapter * R * p.K * 2, (int64_t)R * p.K * 2);
        const __amdgpu_buffer_rsrc_t br = row_buffer(p.b + (int64_t)groups.adapter * p.N * R * 2, (int64_t)p.N * R * 2);
        const float scale = p.scale[groups.adapter];
        uint4 held[kEachB];
#pragma unroll
        for (int i = 0; i < kEachB; ++i) held[i] = load16(br, (uint32_t)n0 * R * 2u + 16u * (threadIdx.x + kFewWaves * kLanes * i));
        for (int first = 0; first < count; first += kTokens) {
            // the products below are for 1, 2, 4 or 8 tokens: x of those that are not there is zeros
            const int left = count - first, with = left == 1 ? 1 : left == 2 ? 2 : left <= 4 ? 4 : 8;
            const int at = first + wave / kShare;
            const int token = at < count ? __builtin_amdgcn_readfirstlane(list[at]) : 0;
            const __amdgpu_buffer_rsrc_t xr = row_buffer(p.x + token * p.ldx * 2, at < count ? (int64_t)p.K * 2 : 0);
            if (wave / kShare < with)
                for (int c = (wave % kShare) * kLanes + lane; c < chunks; c += kShare * kLanes) rows_x[(wave / kShare) * chunks + c] = load16(xr, 16u * c);
            if (first == 0)
#pragma unroll
                for (int i = 0; i < kEachB; ++i) {
                    const int to = threadIdx.x + kFewWaves * kLanes * i;
                    rows_b[to / (2 * RF) * kRowB + to % (2 * RF)] = held[i];
                }
            __syncthreads();
            if (with == 1) few_h<TYPE, RF, 1>(ar, rows_x, chunks, wave, h);
            else if (with == 2) few_h<TYPE, RF, 2>(ar, rows_x, chunks, wave, h);
            else if (with == 4 || kTokens == 4) few_h<TYPE, RF, 4>(ar, rows_x, chunks, wave, h);
            else few_h<TYPE, RF, kTokens>(ar, rows_x, chunks, wave, h);
            __syncthreads();
            // a column each, every other token
            const int n = n0 + (int)threadIdx.x % kFewColumns;
            const uint4* b = rows_b + threadIdx.x % kFewColumns * kRowB;
            const int t0 = __builtin_amdgcn_readfirstlane(threadIdx.x / kFewColumns);
            for (int t = t0; t < min(left, kTokens); t += 2) {
                float value = 0.0f;
#pragma unroll 2
                for (int c = 0; c < 2 * RF; ++c) {
                    Eight<TYPE> e8;
                    e8.w[0] = b[c];
                    float v[8];
                    decode8<TYPE>(e8, v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) value = __builtin_fmaf(h[t][8 * c + e], v[e], value);
                }
                if (n >= p.N) continue;
                const int64_t to = __builtin_amdgcn_readfirstlane(list[first + t]);
                const float base = to_float<TYPE>(reinterpret_cast<const uint16_t*>(p.base)[to * p.ldbase + n]);
                reinterpret_cast<uint16_t*>(p.out)[to * p.ldo + n] = from_float<TYPE>(__builtin_fmaf(value, scale, base));
            }
            __syncthreads();   // (h, x and B before the next tokens')
        }
    }
    if (p.copy && none && g % p.slots == slot) {
        const int count = list_tokens(none, list);
        copy_tokens(p, 0, list, count, wave, kFewWaves, n0, min(p.N, n0 + kFewColumns));
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

struct Plan {
    bool few;               // both products in one launch
    bool step;              // few tokens: waves share tokens and split k and n; else they split the tokens
    int rank_frags;         // k_shrink: 16 ranks each of a workgroup
    int parts, span_k;      // parts of h (none where it does not leave the workgroup)
    int span_n, expand_blocks;
    int64_t tiles;
    int slots;
};

// At most these many tokens take the step's form, which costs less for each adapter of a few tokens. Both forms, us a call, step's and tiles':
//                                        65 tokens      256            512            1024           1600
//   16 adapters, one at random for each token, 5120 -> 5120
//     rank 16                            11.8   40      16.5   41      25     42      39     52      53     80
//     rank 64                            17     56      30     59      47     61      83     78      126    124
//     rank 128                           27     92      60     98      106    103     202    134     286    201
//   one adapter, 5120 -> 5120
//     rank 16                            18     12      21     14      22     15      24     18      40     21
//     rank 64                            27     18      38     19      39     19      60     22      91     27
//     rank 128                           37     25      40     26      54     27      99     30      169    33
// So the limit is where the forms cross for such tokens of rank 64; a batch of up to 1024 tokens in which a request has many would be two to
// three times as fast in tiles, but the host does not read the index.
constexpr int kStepTokens = 1024;
constexpr int kFill = 512;          // workgroups that fill the card at two a compute unit

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

Plan plan_of(int64_t T, int64_t K, int64_t N, int64_t L, int64_t R)
{
    Plan p{};
    // One launch where few tokens of an adapter are to be expected, all in one tile, and h costs little to compute again for each 512
    // columns. One launch against two, rank 32, 5120 -> 7168, us on the card: one token 6.3 and 9.1, 12 tokens of as many adapters 10.5 and 12.0,
    // 32 of 12 12.2 and 12.1, 48 of 12 12.8 and 12.4, 64 of 16 13.5 and 13.2 (and a call's host time is 10 us against 14). L is all that the
    // host knows of how many adapters are used: where those of a large bank are few, one launch is slower from eight tokens of an adapter on
    // (eight 12.9 and 9.6, 16 18 and 10, 64 55 and 21; rank 64: 22 and 11, 33 and 11, 98 and 29), and so are 64 tokens of 64 adapters (65 and 34).
    p.few = T <= kTile && T <= 4 * L && R <= kFewRank && K <= kFewK;
    p.step = T <= kStepTokens;
    p.tiles = ceil_div(T, kTile);
    const int64_t most = T < kTile ? T : kTile, apart = L < most ? L : most;   // adapters of a tile
    if (p.few) {
        p.span_n = kFewColumns;
        p.slots = (int)apart;
    } else if (p.step) {
        const int64_t steps = ceil_div(K, 64);
        p.rank_frags = R > 16 ? 2 : 1;
        p.parts = (int)ceil_div(steps, 5 * kWaves);   // five steps a wave
        if (p.parts > 32) p.parts = 32;
        p.span_k = (int)(64 * kWaves * ceil_div(steps, p.parts * kWaves));
        p.span_n = 256;
        p.slots = (int)(apart < ceil_div(256, p.tiles) ? apart : ceil_div(256, p.tiles));
    } else {
        const int64_t steps = ceil_div(K, kBk), columns = ceil_div(N, kBn);
        p.rank_frags = (int)(R / 16);
        // Workgroups to fill the card (k), two rounds of them where the tiles alone are more than the compute units, as those that hold the border
        // between two requests take twice as long and would be the last of one round (5376 -> 1024, us a call with one round and with two: 23000
        // tokens of three requests, rank 64 102 and 97, rank 128 128 and 122; 20000 of four, rank 16 78 and 70, rank 128 110 and 106; of one
        // request 58 and 59, 75 and 80, 96 and 97 of ranks 16, 64, 128); but seven steps of k in each, as its first ones wait for memory and the
        // second product fetches every part (rank 128, 1600 tokens: 31 us with 21 parts, 24 with six; 4800: 42 with seven, 38 with six).
        int64_t parts = ceil_div(p.tiles > 256 ? 2 * kFill : kFill, p.tiles), blocks = kFill / p.tiles;
        const int64_t eighths = ceil_div(columns, 8);
        if (parts < 2) parts = 2;
        if (parts > ceil_div(steps, 7)) parts = ceil_div(steps, 7);
        p.span_k = (int)(kBk * ceil_div(steps, parts));
        p.parts = (int)ceil_div(K, p.span_k);
        // Above 64 ranks two workgroups of k_expand_tile are all that a compute unit has registers for, and where four or more of a tile are
        // one round of them, an eighth left to tiles of two adapters, more would be two (5376 -> 7168, rank 128, us a call: 6470 tokens of six
        // requests 82 with four and 90 with seven, 3200 of one 51 and 58. At rank 64 three go on a compute unit: 6470 tokens 63 with four, 60 with
        // seven).
        const int64_t round = kFill * 7 / 8 / p.tiles;
        if (R > 64 && round >= 4) blocks = round;
        else if (blocks < eighths) blocks = eighths;
        if (blocks > columns) blocks = columns;
        p.span_n = (int)(kBn * ceil_div(columns, blocks));
        // (a tile that holds the border between two requests takes twice as long: where few tiles are, its adapters go apart)
        p.slots = (int)(apart < ceil_div(256, p.tiles) ? apart : ceil_div(256, p.tiles));
    }
    p.expand_blocks = (int)ceil_div(N, p.span_n);
    return p;
}

template <int TYPE>
int launch_shrink(const AdapterArgs& p, const Plan& plan, hipStream_t stream)
{
    // a step: the adapters' slots beside each other, ranks in y; else the slots in y, those that have no adapter last
    const dim3 block(kWaves * kLanes), grid((unsigned)(plan.tiles * plan.parts * (plan.step ? plan.slots : 1)),
                                            (unsigned)(plan.step ? ceil_div(p.R, 16 * plan.rank_frags) : plan.slots));
    if (plan.step) {
        if (plan.rank_frags == 1) hipLaunchKernelGGL((k_shrink_step<TYPE, 1, kWaves>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((k_shrink_step<TYPE, 2, kWaves>), grid, block, 0, stream, p);
    } else {
        switch (plan.rank_frags) {
#define VDN_CASE(n) \
    case n: hipLaunchKernelGGL((k_shrink_tile<TYPE, n>), grid, block, 0, stream, p); break;
            VDN_CASE(1) VDN_CASE(2) VDN_CASE(3) VDN_CASE(4) VDN_CASE(5) VDN_CASE(6) VDN_CASE(7) VDN_CASE(8)
#undef VDN_CASE
        }
    }
    return check_launch("adapter_add");
}

template <int TYPE, int RF>
int launch_expand(const AdapterArgs& p, const Plan& plan, hipStream_t stream)
{
    const dim3 block(kWaves * kLanes), grid((unsigned)(plan.step ? plan.tiles * plan.expand_blocks * plan.slots : ceil_div(plan.tiles, kDies) * kDies * plan.expand_blocks),
                                            (unsigned)(plan.step ? 1 : plan.slots));
    if (plan.step) hipLaunchKernelGGL((k_expand_step<TYPE, (RF + 1) / 2>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((k_expand_tile<TYPE, RF>), grid, block, 0, stream, p);
    return check_launch("adapter_add");
}

template <int TYPE, int RF>
int launch_few(const AdapterArgs& p, const Plan& plan, hipStream_t stream)
{
    hipLaunchKernelGGL((k_few<TYPE, RF>), dim3((unsigned)(ceil_div(plan.slots, kDies) * kDies * plan.expand_blocks)), dim3(kFewWaves * kLanes), 0, stream, p);
    return check_launch("adapter_add");
}

template <int TYPE>
int launch(AdapterArgs p, const Plan& plan, hipStream_t stream)
{
    p.S = plan.parts;
    p.slots = plan.slots;
    if (plan.few) {
        p.blocks = plan.expand_blocks;
        switch (p.R / 16) {
            case 1: return launch_few<TYPE, 1>(p, plan, stream);
            case 2: return launch_few<TYPE, 2>(p, plan, stream);
            case 3: return launch_few<TYPE, 3>(p, plan, stream);
            default: return launch_few<TYPE, 4>(p, plan, stream);
        }
    }
    if (p.L > 0) {
        p.blocks = plan.parts;
        p.span = plan.span_k;
        const int st = launch_shrink<TYPE>(p, plan, stream);
        if (st != VDN_FP8_OK) return st;
    }
    p.blocks = plan.expand_blocks;
    p.span = plan.span_n;
    switch (p.R / 16) {
        case 1: return launch_expand<TYPE, 1>(p, plan, stream);
        case 2: return launch_expand<TYPE, 2>(p, plan, stream);
        case 3: return launch_expand<TYPE, 3>(p, plan, stream);
        case 4: return launch_expand<TYPE, 4>(p, plan, stream);
        case 5: return launch_expand<TYPE, 5>(p, plan, stream);
        case 6: return launch_expand<TYPE, 6>(p, plan, stream);
        case 7: return launch_expand<TYPE, 7>(p, plan, stream);
        default: return launch_expand<TYPE, 8>(p, plan, stream);
    }
}

// h's parts, tile by tile: those that a workgroup adds lie next to each other.
int64_t workspace_bytes_of(const Plan& plan, int64_t R) { return plan.tiles * plan.parts * kTile * R * 4; }

int check_sizes(int64_t T, int64_t K, int64_t N, int64_t L, int64_t R)
{
    const char* what = "adapter_add";
    if (T < 0 || K < 0 || N < 0 || L < 0 || R < 0) return set_error(VDN_FP8_EINVAL, "%s: negative shape", what);
    if (T > 1 << 23 || L > 1 << 23) return set_error(VDN_FP8_EINVAL, "%s: at most 2^23 tokens and adapters", what);   // (and a launch below 2^32 work-items)
    if (K % 8 || N % 8 || K < 8 || N < 8 || K > 1 << 17 || N > 1 << 17) return set_error(VDN_FP8_EINVAL, "%s: K=%lld and N=%lld must be multiples of 8, at most 2^17", what, (long long)K, (long long)N);
    if (R < 16 || R % 16 || R > kMostRank) return set_error(VDN_FP8_EINVAL, "%s: the rank %lld must be a multiple of 16, at most %d (pad A's rows and B's columns with zeros)", what, (long long)R, kMostRank);
    return VDN_FP8_OK;
}

}  // namespace
}  // namespace vdn

using namespace vdn;

extern "C" int vdn_fp8_adapter_add_workspace_size(int64_t T, int64_t K, int64_t N, int64_t L, int64_t R, int64_t* bytes)
{
    if (!bytes) return set_error(VDN_FP8_EINVAL, "adapter_add: null pointer");
    const int st = check_sizes(T, K, N, L, R);
    if (st != VDN_FP8_OK) return st;
    *bytes = T && L ? workspace_bytes_of(plan_of(T, K, N, L, R), R) : 0;
    return VDN_FP8_OK;
}

extern "C" int vdn_fp8_adapter_add(const void* x, int dtype, int64_t ldx, const void* base, int64_t ldbase, int64_t T, int64_t K, int64_t N,
                                   const void* a, const void* b, const float* scale, int64_t L, int64_t R, const int32_t* index,
                                   void* out, int64_t ldo, void* workspace, int64_t workspace_bytes, hipStream_t stream)
{
    const char* what = "adapter_add";
    const int st = check_sizes(T, K, N, L, R);
    if (st != VDN_FP8_OK) return st;
    if (dtype != kBf16 && dtype != kF16) return set_error(VDN_FP8_EINVAL, "%s: unknown dtype %d (bf16 or binary16)", what, dtype);
    if (T == 0) return VDN_FP8_OK;
    if (!x || !base || !out || !index || (L && (!a || !b || !scale))) return set_error(VDN_FP8_EINVAL, "%s: null pointer", what);
    if (ldx % 8 || ldbase % 8 || ldo % 8 || ldx < K || ldbase < N || ldo < N || ldx > 1 << 23 || ldbase > 1 << 23 || ldo > 1 << 23)
        return set_error(VDN_FP8_EINVAL, "%s: need the row strides multiples of 8, >= K (x) and N (base, out), at most 2^23", what);
    if (!aligned(x, 16) || !aligned(base, 16) || !aligned(out, 16) || !aligned(a, 16) || !aligned(b, 16) || !aligned(scale, 4) || !aligned(index, 4))
        return set_error(VDN_FP8_EINVAL, "%s: misaligned pointer (x, base, out, A, B 16 B)", what);
    // (workgroups read all of x, and write their columns of out when they are done with them)
    if (rows_overlap(x, ldx * 2, K * 2, out, ldo * 2, N * 2, T)) return set_error(VDN_FP8_EINVAL, "%s: out must not overlap x", what);
    if (out == base ? ldo != ldbase : rows_overlap(base, ldbase * 2, N * 2, out, ldo * 2, N * 2, T))
        return set_error(VDN_FP8_EINVAL, "%s: out must be base itself, with its stride, or not overlap it", what);
    const Plan plan = plan_of(T, K, N, L ? L : 1, R);
    const int64_t need = L ? workspace_bytes_of(plan, R) : 0;
    if (need && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
        return set_error(VDN_FP8_EINVAL, "%s: the workspace must be 16-byte aligned and hold %lld bytes", what, (long long)need);
    AdapterArgs p{};
    p.x = (const uint8_t*)x; p.ldx = ldx;
    p.base = (const uint8_t*)base; p.ldbase = ldbase;
    p.out = (uint8_t*)out; p.ldo = ldo;
    p.a = (const uint8_t*)a; p.b = (const uint8_t*)b; p.scale = scale;
    p.index = index;
    p.T = T; p.K = (int)K; p.N = (int)N; p.L = (int)L; p.R = (int)R;
    p.part = (float*)workspace;
    p.copy = out != base;
    p.once = T * N * 2 >= kOnceBytes;
    return dtype == kBf16 ? launch<kBf16>(p, plan, stream) : launch<kF16>(p, plan, stream);
}
