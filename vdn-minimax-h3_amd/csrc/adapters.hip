// Low-rank adapters of many requests beside a shared projection:
//
//   out[t][n] = round(base[t][n] + scale[i] * sum_r h[t][r] B[i][n][r]),   h[t][r] = sum_k x[t][k] A[i][r][k],   i = index[t]
//   out[t]    = base[t] where index[t] is outside [0, L)
//
// in two launches: k_shrink writes h, binary32, in S parts summed over disjoint ranges of k; k_expand
// adds the parts and the second product to the base. Both are bound by memory (2 R operations for each element of x and of base,
// R <= 128), so the matrix cores have time to spare: h is not rounded to 16 bits between the products but goes in as two
// of them, a high and a low part, which keeps 2^-17 of it and costs the second product twice over.
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
    float* part;               // [S, T, R]
    int S;                     // parts of h
    int slots;                 // workgroups that the adapters of a tile are dealt out to
    int blocks;                // ranges of k (k_shrink) or of n (k_expand) of a tile
    int span;                  // k of a part (k_shrink), or columns of a workgroup (k_expand)
    int copy;                  // out is not base: tokens without an adapter are copied
};

__device__ __forceinline__ uint4 load16(__amdgpu_buffer_rsrc_t buffer, uint32_t off)
{
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(buffer, off, 0, 0));
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

// One step of 64 k: a lane's 32 bytes of each of its rows (16 consecutive k: 8 for each of two products).
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
        const int at = k + 8 * h;
        const bool in = at < end;
#pragma unroll
        for (int f = 0; f < TF; ++f) s.x[f][h] = load16(xr, in && xrow[f] != kOutside ? xrow[f] + 2u * at : kOutside);
#pragma unroll
        for (int r = 0; r < RF; ++r) s.a[r][h] = load16(ar, in && arow[r] != kOutside ? arow[r] + 2u * at : kOutside);
    }
}

// The tokens [16 f0, 16 (f0 + TF)) of the list, 16 RF ranks from `rank` on, k from `k0` to `end`.
template <int TYPE, int RF, int TF>
__device__ __forceinline__ void shrink_tokens(const AdapterArgs& p, int64_t tile, int adapter, const int* list, int count, int f0, int rank, int k0,
                                              int end, int part)
{
    const int lane = threadIdx.x & (kLanes - 1), col = lane & 15, quad = lane >> 4;
    const int64_t rows = min(p.T - tile * kTile, (int64_t)kTile);
    const __amdgpu_buffer_rsrc_t xr = row_buffer(p.x + tile * kTile * p.ldx * 2, ((rows - 1) * p.ldx + p.K) * 2);
    const __amdgpu_buffer_rsrc_t ar = row_buffer(p.a + (int64_t)adapter * p.R * p.K * 2, (int64_t)p.R * p.K * 2);
    uint32_t arow[RF], xrow[TF];
    int token[TF];
#pragma unroll
    for (int r = 0; r < RF; ++r) {
        const int at = rank + 16 * r + col;
        arow[r] = at < p.R ? (uint32_t)at * (uint32_t)p.K * 2u : kOutside;
    }
#pragma unroll
    for (int f = 0; f < TF; ++f) {
        const int at = 16 * (f0 + f) + col;
        token[f] = at < count ? list[at] : -1;
        xrow[f] = token[f] >= 0 ? (uint32_t)token[f] * (uint32_t)p.ldx * 2u : kOutside;
    }
    f32x4_t acc[RF][TF];
#pragma unroll
    for (int r = 0; r < RF; ++r)
#pragma unroll
        for (int f = 0; f < TF; ++f) acc[r][f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    auto use = [&](const ShrinkStep<RF, TF>& s) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < RF; ++r)
#pragma unroll
                for (int f = 0; f < TF; ++f) acc[r][f] = Mma<TYPE>::mma(s.a[r][h], s.x[f][h], acc[r][f]);
    };
    ShrinkStep<RF, TF> even, odd;
    int k = k0 + 16 * quad;
    const int steps = (end - k0 + 63) / 64;
    load_step<RF, TF>(even, ar, xr, arow, xrow, k, end);
    for (int i = 0; i < steps; i += 2) {
        load_step<RF, TF>(odd, ar, xr, arow, xrow, k + 64, end);
        use(even);
        load_step<RF, TF>(even, ar, xr, arow, xrow, k + 128, end);
        use(odd);
        k += 128;
    }
    // D: column = token, rows 4 quad .. 4 quad + 3 = ranks
#pragma unroll
    for (int f = 0; f < TF; ++f) {
        if (token[f] < 0) continue;
        float* h = p.part + ((int64_t)part * p.T + tile * kTile + token[f]) * p.R + rank + 4 * quad;
#pragma unroll
        for (int r = 0; r < RF; ++r)
            if (rank + 16 * r < p.R) *reinterpret_cast<f32x4_t*>(h + 16 * r) = acc[r][f];
    }
}

// WAVES waves: WT of them share a range of k and take other tokens, WAVES / WT ranges of k.
template <int TYPE, int RF, int WAVES, int WT>
__global__ __launch_bounds__(WAVES * kLanes) void k_shrink(AdapterArgs p)
{
    __shared__ int lists[WAVES][kTile];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const uint32_t block = blockIdx.x / (uint32_t)p.blocks, range = blockIdx.x % (uint32_t)p.blocks;
    const int64_t tile = block / (uint32_t)p.slots;
    const int slot = (int)(block % (uint32_t)p.slots);
    const int part = (int)range * (WAVES / WT) + wave / WT;
    const int k0 = part * p.span, end = min(p.K, k0 + p.span);
    const int rank = blockIdx.y * 16 * RF;
    Groups groups(p, tile);
    for (int g = 0; groups.next(); ++g) {
        if (g % p.slots != slot) continue;
        const int count = list_tokens(groups.mask, lists[wave]);
        for (int f = 2 * (wave % WT); f * 16 < count; f += 2 * WT) {
            if (f * 16 + 16 < count) shrink_tokens<TYPE, RF, 2>(p, tile, groups.adapter, lists[wave], count, f, rank, k0, end, part);
            else shrink_tokens<TYPE, RF, 1>(p, tile, groups.adapter, lists[wave], count, f, rank, k0, end, part);
        }
    }
}

// ---------------------------------------------------------------------------
// out = base + scale h B^T
// ---------------------------------------------------------------------------

// Eight ranks of h as two operands of eight 16-bit values, high and low part. bf16: the upper half of the word and what it leaves
// (16 bits in all, whatever the size). float16: relative to the power of two 2^e above the token's largest, e back in the result,
// so that no h is too large for it.
template <int TYPE>
__device__ __forceinline__ void split8(const float (&h)[8], float down, uint4& high, uint4& low)
{
    uint32_t a[4], b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (TYPE == kBf16) {
            const uint32_t u0 = __float_as_uint(h[2 * e]), u1 = __float_as_uint(h[2 * e + 1]);
            a[e] = (u0 >> 16) | (u1 & 0xffff0000u);
            // (an infinity leaves nothing: the difference would be NaN)
            const float l0 = __builtin_isfinite(h[2 * e]) ? h[2 * e] - __uint_as_float(u0 & 0xffff0000u) : 0.0f;
            const float l1 = __builtin_isfinite(h[2 * e + 1]) ? h[2 * e + 1] - __uint_as_float(u1 & 0xffff0000u) : 0.0f;
            b[e] = pack_bf16x2(l0, l1);
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

template <int RK, int TF>
struct ExpandStep {
    uint4 b[2][RK], base[TF];
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
    uint4 high[TF][RK], low[TF][RK];
    float up[TF];
#pragma unroll
    for (int f = 0; f < TF; ++f) {
        const int at = 16 * (f0 + f) + col;
        const int token = at < count ? list[at] : -1;
        baserow[f] = token >= 0 ? (uint32_t)token * (uint32_t)p.ldbase * 2u : kOutside;
        outrow[f] = token >= 0 ? (uint32_t)token * (uint32_t)p.ldo * 2u : kOutside;
        float h[RK][8];
#pragma unroll
        for (int r = 0; r < RK; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) h[r][e] = 0.0f;
        if (token >= 0) {
            const float* from = p.part + (tile * kTile + token) * p.R + 8 * quad;
#pragma unroll 4
            for (int s = 0; s < p.S; ++s) {
#pragma unroll
                for (int r = 0; r < RK; ++r) {
                    if (32 * r + 8 * quad >= p.R) continue;
                    const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(from + (int64_t)s * p.T * p.R + 32 * r);
                    const f32x4_t hi = *reinterpret_cast<const f32x4_t*>(from + (int64_t)s * p.T * p.R + 32 * r + 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        h[r][e] += lo[e];
                        h[r][4 + e] += hi[e];
                    }
                }
            }
        }
        float most = 0.0f;
#pragma unroll
        for (int r = 0; r < RK; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) most = __builtin_fmaxf(most, __builtin_fabsf(h[r][e]));
        float down = 1.0f;
        up[f] = 1.0f;
        if (TYPE == kF16) {
            most = __builtin_fmaxf(most, __shfl_xor(most, 16, kLanes));
            most = __builtin_fmaxf(most, __shfl_xor(most, 32, kLanes));
            // 2^e above the largest, e in the range in which 2^-e and 2^e are normal
            const int e = most > 0.0f && __builtin_isfinite(most) ? min(max((int)(__float_as_uint(most) >> 23) - 126, -120), 120) : 0;
            down = __uint_as_float((uint32_t)(127 - e) << 23);
            up[f] = __uint_as_float((uint32_t)(127 + e) << 23);
        }
#pragma unroll
        for (int r = 0; r < RK; ++r) split8<TYPE>(h[r], down, high[f][r], low[f][r]);
    }
    // B's rows as the first operand, so that a column of the result is a token; row i of product f is column
    // n + 8 (i / 4) + 4 f + i % 4: a lane holds eight consecutive columns of its token.
    const uint32_t brow = (uint32_t)(8 * (col / 4) + col % 4) * (uint32_t)p.R * 2u + 16u * quad;
    auto load = [&](ExpandStep<RK, TF>& s, int n) {
        const bool in = n + 8 * quad < end;
#pragma unroll
        for (int f = 0; f < TF; ++f) s.base[f] = load16(baser, in && baserow[f] != kOutside ? baserow[f] + 2u * (n + 8 * quad) : kOutside);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < RK; ++r)
                s.b[h][r] = load16(br, 32 * r + 8 * quad < p.R && n < end ? brow + (uint32_t)(n + 4 * h) * (uint32_t)p.R * 2u + 64u * r : kOutside);
    };
    auto use = [&](const ExpandStep<RK, TF>& s, int n) {
        const bool in = n + 8 * quad < end;
#pragma unroll
        for (int f = 0; f < TF; ++f) {
            f32x4_t acc[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                acc[h] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int r = 0; r < RK; ++r) {
                    acc[h] = Mma<TYPE>::mma(s.b[h][r], high[f][r], acc[h]);
                    acc[h] = Mma<TYPE>::mma(s.b[h][r], low[f][r], acc[h]);
                }
            }
            float v[8];
            Eight<TYPE> o;
            o.w[0] = s.base[f];
            decode8<TYPE>(o, v);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * h + e] = __builtin_fmaf(TYPE == kF16 ? acc[h][e] * up[f] : acc[h][e], scale, v[4 * h + e]);
            o = encode8<TYPE>(v);
            store_b128_settled<0>(__builtin_bit_cast(i32x4_t, o.w[0]), outr, in && outrow[f] != kOutside ? outrow[f] + 2u * (n + 8 * quad) : kOutside, 0);
        }
    };
    ExpandStep<RK, TF> even, odd;
    load(even, n0);
    for (int n = n0; n < end; n += 64) {
        load(odd, n + 32);
        use(even, n);
        load(even, n + 64);
        use(odd, n + 32);
    }
}

// The rows of a mask's tokens, columns n0 to end, by one wave of `waves`.
__device__ __forceinline__ void copy_tokens(const AdapterArgs& p, int64_t tile, const int* list, int count, int wave, int waves, int n0, int end)
{
    const int lane = threadIdx.x & (kLanes - 1);
    for (int i = wave; i < count; i += waves) {
        const int64_t t = tile * kTile + list[i];
        const __amdgpu_buffer_rsrc_t from = row_buffer(p.base + t * p.ldbase * 2, (int64_t)end * 2), to = row_buffer(p.out + t * p.ldo * 2, (int64_t)end * 2);
        for (int n = n0 + 8 * lane; n < end; n += 8 * kLanes) store_b128_settled<0>(__builtin_bit_cast(i32x4_t, load16(from, 2u * n)), to, 2u * n, 0);
    }
}

template <int TYPE, int RK, int WAVES, int WT>
__global__ __launch_bounds__(WAVES * kLanes) void k_expand(AdapterArgs p)
{
    __shared__ int lists[WAVES][kTile];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const uint32_t block = blockIdx.x / (uint32_t)p.blocks, range = blockIdx.x % (uint32_t)p.blocks;
    const int64_t tile = block / (uint32_t)p.slots;
    const int slot = (int)(block % (uint32_t)p.slots);
    // each of WAVES / WT waves its own columns
    const int own = p.span / (WAVES / WT);
    const int n0 = (int)range * p.span + wave / WT * own, end = min(p.N, n0 + own);
    Groups groups(p, tile);
    const int lane = threadIdx.x & (kLanes - 1);
    const uint64_t none = __ballot(tile * kTile + lane < p.T && groups.mine < 0);
    int g = 0;
    for (; groups.next(); ++g) {
        if (g % p.slots != slot) continue;
        const int count = list_tokens(groups.mask, lists[wave]);
        for (int f = 2 * (wave % WT); f * 16 < count; f += 2 * WT) {
            if (f * 16 + 16 < count) expand_tokens<TYPE, RK, 2>(p, tile, groups.adapter, lists[wave], count, f, n0, end);
            else expand_tokens<TYPE, RK, 1>(p, tile, groups.adapter, lists[wave], count, f, n0, end);
        }
    }
    if (p.copy && none && g % p.slots == slot) {
        const int count = list_tokens(none, lists[wave]);
        copy_tokens(p, tile, lists[wave], count, wave % WT, WT, n0, end);
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

struct Plan {
    bool step;              // few tokens: waves share tokens and split k and n; else they split the tokens
    int rank_frags;         // k_shrink: 16 ranks each of a workgroup
    int parts, span_k, shrink_blocks;
    int span_n, expand_blocks;
    int64_t tiles;
    int slots;
};

constexpr int kStepTokens = 1024;   // at most these many take the step's form

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

Plan plan_of(int64_t T, int64_t K, int64_t N, int64_t L, int64_t R)
{
    Plan p{};
    p.step = T <= kStepTokens;
    p.tiles = ceil_div(T, kTile);
    const int64_t most = T < kTile ? T : kTile, apart = L < most ? L : most;   // adapters of a tile
    if (p.step) {
        p.rank_frags = R > 16 ? 2 : 1;
        const int64_t steps = ceil_div(K, 64);
        int64_t parts = 4 * ceil_div(steps, 20);   // five steps a wave
        if (parts > 32) parts = 32;
        p.span_k = (int)(64 * ceil_div(steps, parts));
        p.parts = (int)parts;
        p.shrink_blocks = (int)(parts / 4);
        p.span_n = 256;
        p.slots = (int)(apart < ceil_div(256, p.tiles) ? apart : ceil_div(256, p.tiles));
    } else {
        p.rank_frags = R > 64 ? 8 : R > 32 ? 4 : R > 16 ? 2 : 1;
        const int64_t steps = ceil_div(K, 64);
        p.parts = steps >= 16 ? 2 : 1;
        p.span_k = (int)(64 * ceil_div(steps, p.parts));
        p.shrink_blocks = p.parts;
        p.span_n = 1024;
        p.slots = 1;
    }
    p.expand_blocks = (int)ceil_div(N, p.span_n);
    return p;
}

template <int TYPE, int RF, bool STEP>
int launch_shrink(const AdapterArgs& p, const Plan& plan, hipStream_t stream)
{
    constexpr int waves = STEP ? 4 : 2, wt = STEP ? 1 : 2;
    const dim3 grid((unsigned)(plan.tiles * plan.slots * plan.shrink_blocks), (unsigned)ceil_div(p.R, 16 * RF));
    hipLaunchKernelGGL((k_shrink<TYPE, RF, waves, wt>), grid, dim3(waves * kLanes), 0, stream, p);
    return check_launch("adapter_add");
}

template <int TYPE, int RK, bool STEP>
int launch_expand(const AdapterArgs& p, const Plan& plan, hipStream_t stream)
{
    constexpr int waves = STEP ? 4 : 2, wt = STEP ? 1 : 2;
    const dim3 grid((unsigned)(plan.tiles * plan.slots * plan.expand_blocks));
    hipLaunchKernelGGL((k_expand<TYPE, RK, waves, wt>), grid, dim3(waves * kLanes), 0, stream, p);
    return check_launch("adapter_add");
}

template <int TYPE>
int launch(AdapterArgs p, const Plan& plan, hipStream_t stream)
{
    p.S = plan.parts;
    p.slots = plan.slots;
    p.blocks = plan.shrink_blocks;
    p.span = plan.span_k;
    int st = VDN_FP8_OK;
    if (p.L == 0) {
        // no adapter: nothing to multiply by
    } else if (plan.step) {
        st = plan.rank_frags == 1 ? launch_shrink<TYPE, 1, true>(p, plan, stream) : launch_shrink<TYPE, 2, true>(p, plan, stream);
    } else {
        st = plan.rank_frags == 1   ? launch_shrink<TYPE, 1, false>(p, plan, stream)
             : plan.rank_frags == 2 ? launch_shrink<TYPE, 2, false>(p, plan, stream)
             : plan.rank_frags == 4 ? launch_shrink<TYPE, 4, false>(p, plan, stream)
                                    : launch_shrink<TYPE, 8, false>(p, plan, stream);
    }
    if (st != VDN_FP8_OK) return st;
    p.blocks = plan.expand_blocks;
    p.span = plan.span_n;
    const int64_t steps = ceil_div(p.R, 32);
#define VDN_CASE(n) \
    if (steps == n) return plan.step ? launch_expand<TYPE, n, true>(p, plan, stream) : launch_expand<TYPE, n, false>(p, plan, stream);
    VDN_CASE(1) VDN_CASE(2) VDN_CASE(3) VDN_CASE(4)
#undef VDN_CASE
    return set_error(VDN_FP8_EINVAL, "adapter_add: unsupported rank");
}

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
    *bytes = T && L ? plan_of(T, K, N, L, R).parts * T * R * 4 : 0;
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
    const Plan plan = plan_of(T, K, N, L ? L : 1, R);
    if (L && (!workspace || !aligned(workspace, 16) || workspace_bytes < plan.parts * T * R * 4))
        return set_error(VDN_FP8_EINVAL, "%s: the workspace must be 16-byte aligned and hold %lld bytes", what, (long long)(plan.parts * T * R * 4));
    AdapterArgs p{};
    p.x = (const uint8_t*)x; p.ldx = ldx;
    p.base = (const uint8_t*)base; p.ldbase = ldbase;
    p.out = (uint8_t*)out; p.ldo = ldo;
    p.a = (const uint8_t*)a; p.b = (const uint8_t*)b; p.scale = scale;
    p.index = index;
    p.T = T; p.K = (int)K; p.N = (int)N; p.L = (int)L; p.R = (int)R;
    p.part = (float*)workspace;
    p.copy = out != base;
    return dtype == kBf16 ? launch<kBf16>(p, plan, stream) : launch<kF16>(p, plan, stream);
}
