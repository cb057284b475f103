// Softmax attention over the 8-bit key/value cache.
//
// For a query row q (one token, one head) over the visible tokens j of its sequence:
//   x_j = log2(e) scale (q . k_j),  k_j = code 2^ek,   o = sum_j 2^(x_j) v_j / sum_j 2^(x_j)
// in one pass over the pages, in units that follow them. Three choices carry the arithmetic:
//
//   Scores in the queries' own type: e4m3 codes are bf16 and binary16 numbers, so keys are decoded exactly,
//   products are exact and sums are binary32. (On the fp8 matrix cores, with a bf16 query as the sum of two
//   e4m3 terms, a product costs the same and keys need no decoding; but those cores align the 64 or 128
//   products of an instruction to the largest and drop what is below: scores were off by up to 2^-12 of the
//   largest product, where these sums stay within 2^-18 of it, for 1.99 against 2.15 ms on 3120 tokens over 32760.)
//
//   Values in binary16: e4m3 codes are binary16 numbers, and weights keep eleven bits (bf16 weights would
//   leave eight, an error as large as the output's own rounding). The value's scale 2^ev never meets the
//   codes: it joins the exponent of the weight, P' = 2^(x + ev - m + 5), where 2^m is the unit of the row's
//   accumulators, so that the product's sum is that of the real values. Sums, units and accumulators are
//   binary32, and so is the sum of the weights 2^(x - t), which has a unit 2^t of its own.
//
//   The transposed scores S^T = K Q^T leave each lane 16 consecutive keys of one query (the key that
//   a matrix row stands for is a matter of which row is loaded where), and those are the operand of
//   O^T = V^T P^T as they are: P goes from one product to the next in registers.
//
// binary16 has few exponents, and one maximum for all pages would leave them to the weights next to the row's
// largest: behind a token 17 nats above the others, or one of little weight in a page of large values, the others would
// be lost from the output, though not from the sum. So a row's unit follows its pages both ways: a page whose
// largest x + ev lies more than 10 from m moves m to it, and the accumulators by that power. A page's
// largest weight is then held as 2^-5 to 2^15 (as 2^5, without a rounding, where the unit moves: whole numbers for m would make
// the moves exact but round that weight: binary16 outputs 2.9e-4 off instead of 2.7e-4), and each weight is off by 2^-11
// of itself or 2^-20 of its page's largest. A unit comes down by 2^60 at most, which binary32 accumulators leave room for: pages
// further below a row's largest are zeros (2^-80 of it and less). On 3120 tokens over 32760, whose pages' largest scores spread by 2 in standard
// deviation, 2.19 ms; with 9, 8 and 6 in place of 10 2.24, 2.29 and 2.33; with a unit that only rises, by more than 8, 2.17.
//
// Rows are (token, head of a group) pairs of one key/value head, so grouped heads share the pages
// that they read. Two kernels:
//   k_kv_attn_rows    128 rows, 32 for each of four waves, which share the pages through LDS: keys as codes
//                     (asynchronous copies, two pages ahead; each wave decodes what it reads), values decoded
//                     once for all four. For chunks and prompts. 3120 tokens over 32760, 40 heads of 128:
//                     2.15 to 2.23 ms, 0.94 to 0.97 PF/s; the card's power limit holds its clock at 1.9 of 2.4 GHz, where bare
//                     chains of the same instructions reach 1.6 to 1.8 PF/s. Keys decoded once as well are
//                     slower (2.28 ms: LDS reads, 32 KB a wave and page, take as long as the products).
//   k_kv_attn_step    up to 16 rows; each of the four waves takes every fourth page, straight from
//                     memory into the operands' registers, and they join at the end. For single tokens.
//                     8 sequences of 71000 to 131072 tokens, 40 on 8 heads of 128: 0.29 ms, 5.6 TB/s.
// Both cut long key axes into splits where there are few rows, joined by k_kv_attn_join.
#include <stdint.h>

#include <algorithm>

#include "gemm_common.h"
#include "kv_common.h"
#include "vdn_common.h"

namespace vdn {
namespace {

constexpr int kRows = 128, kWaveRows = 32;   // of k_kv_attn_rows
constexpr int kStepRows = 16;                  // of k_kv_attn_step, at most
constexpr int kInfo = 256;                     // pages that a workgroup looks up at a time
constexpr int kMostSplits = 64;
constexpr float kNone = -3.0e38f;       // the exponent of a unit before any key: finite, so that differences stay numbers
constexpr float kWindow = 10.0f;        // a unit moves when a page's largest weight is further from it than this,
constexpr float kLargest = 5.0f;        // and weights are held times 2^5, so 2^15 at most
constexpr float kRange = 60.0f;         // how far a unit comes down, and how far scores rise above the sum's unit
constexpr int kAbsent = 1 << 30;        // first key of a page that is not there: behind every sequence

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct KvAttnArgs {
    KvCacheArgs c;
    KvBatchArgs b;
    KvUnits units;          // the units of rows
    const uint16_t* q;
    int64_t ldq;
    int group, q_heads;     // query heads for each key/value head, and in all
    float scale;            // of the scores, times log2(e)
    int causal;
    const int32_t* blocks;  // [listed units, heads, top] pages that a query block attends to, or NULL
    int top, query_block;
    int block_rows;         // rows of a query block of k_kv_attn_rows (2^30, more than a call has, where they are more)
    KvUnits listed;
    uint16_t* out;
    float* lse;
    float* part;            // splits > 1: accumulators [tokens * q_heads][splits][d], then what part_sums holds
    int splits, column_tiles;
    bool turns;             // of k_kv_attn_step: sequences may have more rows than column_tiles hold
    uint32_t items;         // workgroups of k_kv_attn_rows
};

// Of a part of a row's keys: the accumulators' unit, the sum's unit and the sum (Running), and nothing.
__device__ __forceinline__ float4* part_sums(const KvAttnArgs& p)
{
    return reinterpret_cast<float4*>(p.part + p.b.tokens * p.q_heads * p.splits * p.c.d);
}

// The key of each 32 that row r of the matrix stands for: lane group g = (r >> 2) & 1 of the output
// then holds keys 16 g .. 16 g + 15 in its registers' order.
__device__ __forceinline__ int row_key(int r) { return 16 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3); }

// The value of the lane 32 (16) away joined with one's own: lanes that hold the same row.
template <typename F>
__device__ __forceinline__ float across32(float v, F f)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <typename F>
__device__ __forceinline__ float across16(float v, F f)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// (NaN wins: the row becomes NaN anyway, and one instruction takes two values without quieting them first)
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float larger3(float a, float b, float c) { return larger(larger(a, b), c); }   // (one instruction)
__device__ __forceinline__ float added(float a, float b) { return a + b; }

__device__ __forceinline__ float exponent_f32(int e) { return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23); }

// v 2^e, where 2^e alone may be out of binary32's range.
__device__ __forceinline__ float times_power(float v, float e)
{
    const float half = __builtin_amdgcn_exp2f(0.5f * e);
    return v * half * half;
}

// One row's softmax over the pages so far: accumulators hold sum P' v in units of 2^m, P' times 2^kLargest, and the
// sum of weights (of the lane's keys) is l 2^t.
struct Running {
    float m, t;
    float low;    // m does not go below
    float l;
    __device__ __forceinline__ void start() { m = t = low = kNone, l = 0.0f; }

    // A page whose largest score is x (-inf: none seen), values' scale 2^ev: true where the unit of some row of the wave
    // moves, and then the accumulators are to be multiplied by 2^move.
    __device__ __forceinline__ bool moves(float x, float ev, float& move)
    {
        const float to = fmaxf(x + ev, low);
        if (!__any(fabsf(to - m) > kWindow || x > t + kRange)) return false;
        const float most = fmaxf(t, x);
        move = m - to;
        l *= __builtin_amdgcn_exp2f(t - most);
        m = to, t = most, low = fmaxf(low, to - kRange);
        return true;
    }
    // A page below the unit's reach adds nothing to the accumulators, but its weights count in l (values of zeros have the
    // least scale): they are lifted to 2^-55, still zeros in binary16, so that their sum is one.
    __device__ __forceinline__ float lift(float x, float ev) const { return __builtin_amdgcn_fmed3f(m - (x + ev) - kRange, 0.0f, 400.0f); }
    // What joins a score in the exponent of P'.
    __device__ __forceinline__ float base(float ev, float lift) const { return ev - m + (kLargest + lift); }
    // The page's sum of P'.
    __device__ __forceinline__ void add(float sum, float ev, float lift) { l += sum * __builtin_amdgcn_exp2f((m - t) - (ev + (kLargest + lift))); }
};

// 16 codes of one operand row -> two operands of eight values (exact).
__device__ __forceinline__ void decode16(uint4 w, f16x8_t o[2])
{
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u[i], 1.0f, false);
        const f16x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u[i], 1.0f, true);
        o[i / 2][4 * (i % 2)] = lo.x, o[i / 2][4 * (i % 2) + 1] = lo.y;
        o[i / 2][4 * (i % 2) + 2] = hi.x, o[i / 2][4 * (i % 2) + 3] = hi.y;
    }
}
__device__ __forceinline__ void decode16(uint4 w, bf16x8_t o[2])
{
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bf16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u[i], 1.0f, false);
        const bf16x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u[i], 1.0f, true);
        o[i / 2][4 * (i % 2)] = lo.x, o[i / 2][4 * (i % 2) + 1] = lo.y;
        o[i / 2][4 * (i % 2) + 2] = hi.x, o[i / 2][4 * (i % 2) + 3] = hi.y;
    }
}

// The queries' type: its operand of eight values, and the products of 32 x 32 x 16 and 16 x 16 x 32.
template <bool F16>
struct Query;
template <>
struct Query<true> {
    typedef f16x8_t Eight;
    __device__ __forceinline__ static f32x16_t mma32(Eight a, Eight b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    __device__ __forceinline__ static f32x4_t mma16(Eight a, Eight b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Query<false> {
    typedef bf16x8_t Eight;
    __device__ __forceinline__ static f32x16_t mma32(Eight a, Eight b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    __device__ __forceinline__ static f32x4_t mma16(Eight a, Eight b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// Eight query values at `row` (NULL: zeros).
template <bool F16>
__device__ __forceinline__ typename Query<F16>::Eight query8(const uint16_t* row)
{
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row) v = *reinterpret_cast<const uint4*>(row);
    return __builtin_bit_cast(typename Query<F16>::Eight, v);
}

constexpr int waitcnt_lgkm0() { return 15 | (7 << 4) | (0 << 8) | (3 << 14); }   // any vmcnt

// What the workgroup knows of a page: its number in the pool (-1: not there), its number in the
// sequence, and its scales' exponents. Looked up by all threads at once, kInfo pages at a time, so
// that the loops over pages meet no chain of dependent loads.
struct PageInfo {
    int page, w, ek, ev;
};

__device__ __forceinline__ void look_up(const KvAttnArgs& p, int b, int h, int length, const int32_t* list, int i0, int hi, PageInfo* info)
{
    const int i = i0 + (int)threadIdx.x;
    if (threadIdx.x < kInfo && i < hi) {
        // (no load under a condition on another; an entry outside the sequence is read at 0 and passed over)
        PageInfo a;
        const int have = (length + kPage - 1) / kPage;
        a.w = list ? list[i] : i;
        const bool inside = a.w >= 0 && a.w < have;
        a.page = kv_page(p.b, p.c, b, inside ? a.w : 0);
        const int64_t ph = (int64_t)max(a.page, 0) * p.c.heads + h;
        a.ek = p.c.k_scale[ph] - 127, a.ev = p.c.v_scale[ph] - 127;
        if (!inside) a.page = -1;
        info[threadIdx.x] = a;
    }
}

// One entry, in scalar registers.
__device__ __forceinline__ PageInfo info_at(const PageInfo* info, int i)
{
    const int4 v = *reinterpret_cast<const int4*>(info + i);
    return PageInfo{__builtin_amdgcn_readfirstlane(v.x), __builtin_amdgcn_readfirstlane(v.y), __builtin_amdgcn_readfirstlane(v.z),
                    __builtin_amdgcn_readfirstlane(v.w)};
}
__device__ __forceinline__ int first_key(const PageInfo& a) { return a.page >= 0 ? a.w * kPage : kAbsent; }

// Codes of 16 tokens of which the first `have` are in the sequence: the others become zeros (they hold what
// an earlier owner of the page left). The NaN codes left are marked in `nan` by their top bits.
__device__ __forceinline__ uint4 keep_tokens(uint4 v, int have, uint4& nan)
{
    uint32_t u[4] = {v.x, v.y, v.z, v.w}, n[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = have - 4 * i;
        u[i] = k >= 4 ? u[i] : k <= 0 ? 0u : u[i] & (0xffffffffu >> (32 - 8 * k));
        n[i] = ((u[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    }
    nan = make_uint4(n[0], n[1], n[2], n[3]);
    return make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ bool any_of(uint4 v) { return (v.x | v.y | v.z | v.w) != 0; }
// The marked codes without their bytes; the marks as e4m3 ones.
__device__ __forceinline__ uint4 without(uint4 v, uint4 nan)
{
    return make_uint4(v.x & ~((nan.x >> 7) * 0xffu), v.y & ~((nan.y >> 7) * 0xffu), v.z & ~((nan.z >> 7) * 0xffu), v.w & ~((nan.w >> 7) * 0xffu));
}
__device__ __forceinline__ uint4 as_ones(uint4 nan)
{
    return make_uint4((nan.x >> 7) * 0x38u, (nan.y >> 7) * 0x38u, (nan.z >> 7) * 0x38u, (nan.w >> 7) * 0x38u);
}
// Which of eight tokens from `first` on a row sees, as ones. (Opaque, so that it is computed where it is
// rarely needed and not kept in registers where it is not.)
__device__ __forceinline__ f16x8_t seen_ones(int first, int limit)
{
    asm volatile("" : "+v"(limit));
    f16x8_t o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = first + j < limit ? (_Float16)1.0f : (_Float16)0.0f;
    return o;
}

// One wave's 32 rows of k_kv_attn_rows: the queries, the running softmax, the output's accumulators.
// Lane l: column l % 32 is the row of the problem, g = l / 32 its half of the keys.
template <int D, bool F16>
struct WaveRows {
    static constexpr int kSteps = D / 16, kTiles = D / 32;
    typedef typename Query<F16>::Eight Eight;
    Eight q[kSteps];
    f32x16_t acc[kTiles];
    Running run;       // (l of this half's keys)

    // row: the row's values (NULL: none, zeros).
    __device__ __forceinline__ void start(const uint16_t* row, int g)
    {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) q[s] = query8<F16>(row ? row + 64 * (s >> 2) + 32 * g + 8 * (s & 3) : nullptr);
        run.start();
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
    }

    // Scores of 64 keys: key(kt, s) gives 16 codes, 64 (s / 2) + 32 g + 16 (s % 2) on, of this lane's matrix row.
    template <typename Key>
    __device__ __forceinline__ void scores(Key key, f32x16_t s[2]) const
    {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kt][i] = 0.0f;
#pragma unroll
            for (int st = 0; st < kSteps / 2; ++st) {
                Eight k[2];
                decode16(key(kt, st), k);
                s[kt] = Query<F16>::mma32(k[0], q[2 * st], s[kt]);
                s[kt] = Query<F16>::mma32(k[1], q[2 * st + 1], s[kt]);
            }
        }
    }

    // Keys from key0 on that the row does not see: from `limit` on.
    __device__ __forceinline__ void mask(f32x16_t s[2], int limit, int key0, int g) const
    {
        const int seen = limit - key0 - 16 * g;   // visible ones of this half's keys, counted from its first
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kt][i] = 32 * kt + i < seen ? s[kt][i] : -__builtin_inff();
    }

    // Scores -> weights in binary16, for a page whose scales are 2^ek and 2^ev; scale: of the scores.
    __device__ __forceinline__ void weights(f32x16_t s[2], float scale, int ek, int ev, f16x8_t w[2][2])
    {
        const float f = fmaxf(scale * exponent_f32(ek), 1e-37f);   // (never 0: a masked score stays -inf)
        const float shift = (float)ev;
        float four[4];   // (two new scores an instruction)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x16_t& a = s[i / 2];
            const int j = 8 * (i % 2);
            four[i] = larger3(larger3(larger3(larger(a[j], a[j + 1]), a[j + 2], a[j + 3]), a[j + 4], a[j + 5]), a[j + 6], a[j + 7]);
        }
        const float x = across32(larger(larger3(four[0], four[1], four[2]), four[3]), larger) * f;
        float move;
        if (run.moves(x, shift, move)) {
            const float a = __builtin_amdgcn_exp2f(move);
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[t][i] *= a;
        }
        const float lift = run.lift(x, shift), base = run.base(shift, lift);
        float sum = 0.0f;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][8 * h + j], f, base));
                    sum += p;
                    w[kt][h][j] = (_Float16)p;
                }
        run.add(sum, shift, lift);
    }

    // Adds the weighted values of a page: value(kt, h, t) gives one element's values of the eight tokens from
    // 32 kt + 16 g + 8 h on.
    template <typename Value>
    __device__ __forceinline__ void add_values(const f16x8_t (&v0)[2][kTiles], Value value, const f16x8_t w[2][2])
    {
        f16x8_t v1[2][kTiles];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0[h][t], w[0][h], acc[t], 0, 0, 0);
                v1[h][t] = value(1, h, t);
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
                acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v1[h][t], w[1][h], acc[t], 0, 0, 0);
    }

    // A page in which some rows see NaN values that others do not (its NaN were stored as zeros): the rows
    // that see one become NaN, by a product of indicators. codes(kt, t): 16 tokens from 32 kt + 16 g on.
    template <typename Codes>
    __device__ __forceinline__ void add_nan(Codes codes, int limit, int key0, int end, int g)
    {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            __builtin_amdgcn_sched_barrier(0);
            f32x16_t hit;
#pragma unroll
            for (int i = 0; i < 16; ++i) hit[i] = 0.0f;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const int first = key0 + 32 * kt + 16 * g;
                uint4 nan;
                keep_tokens(codes(kt, t), end - first, nan);
                f16x8_t is_nan[2];
                decode16(as_ones(nan), is_nan);
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    hit = __builtin_amdgcn_mfma_f32_32x32x16_f16(is_nan[h], seen_ones(first + 8 * h, limit), hit, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[t][i] = hit[i] > 0.0f ? __builtin_nanf("") : acc[t][i];
        }
    }
};

// One wave's 16 rows of k_kv_attn_step: lane l holds row l % 16, and the keys 16 g .. 16 g + 15 of a page
// (g = l / 16), tile t of the scores standing for keys 16 g + 4 t + i. (Half the accumulators and scores
// that 32 columns would take. Two such sets to a wave spilled from d = 128 on: with groups of 8 and 4
// queries 61 us against 58 for two workgroups that read the pages twice, 229 against 143 at d = 256.)
template <int D, bool F16>
struct StepRows {
    static constexpr int kSteps = D / 32, kTiles = D / 16;
    typedef typename Query<F16>::Eight Eight;
    Eight q[kSteps];
    f32x4_t acc[kTiles];
    Running run;
    int limit;

    // (the inner dimension of the scores: lane group g takes elements g D / 4 on, eight a step)
    __device__ __forceinline__ void start(const uint16_t* row, int g)
    {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) q[s] = query8<F16>(row ? row + D / 4 * g + 8 * s : nullptr);
        run.start();
#pragma unroll
        for (int t = 0; t < kTiles; ++t) acc[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // k[t][j]: 16 codes of a key of tile t, of this lane's D / 4.
    __device__ __forceinline__ void scores(const uint4 (&k)[4][D / 64], f32x4_t s[4]) const
    {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
                Eight a[2];
                decode16(k[t][j], a);
                s[t] = Query<F16>::mma16(a[0], q[2 * j], s[t]);
                s[t] = Query<F16>::mma16(a[1], q[2 * j + 1], s[t]);
            }
        }
    }

    __device__ __forceinline__ void mask(f32x4_t s[4], int key0, int g) const
    {
        const int seen = limit - key0 - 16 * g;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][i] = 4 * t + i < seen ? s[t][i] : -__builtin_inff();
    }

    __device__ __forceinline__ void weights(const f32x4_t s[4], float scale, int ek, int ev, f16x8_t w[2])
    {
        const float shift = (float)ev, f = fmaxf(scale * exponent_f32(ek), 1e-37f);
        float four[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) four[i] = larger(larger3(s[i][0], s[i][1], s[i][2]), s[i][3]);
        const float x = across16(across32(larger(larger3(four[0], four[1], four[2]), four[3]), larger), larger) * f;
        float move;
        if (run.moves(x, shift, move)) {
            const float a = __builtin_amdgcn_exp2f(move);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) acc[t] *= a;
        }
        const float lift = run.lift(x, shift), base = run.base(shift, lift);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 4][i % 4], f, base));
            sum += p;
            w[i / 8][i % 8] = (_Float16)p;
        }
        run.add(sum, shift, lift);
    }

    // v[t]: the codes of 16 tokens, one element.
    __device__ __forceinline__ void add_values(const uint4 v[kTiles], const f16x8_t w[2])
    {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            f16x8_t a[2];
            decode16(v[t], a);
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], w[0], acc[t], 0, 0, 0);
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[1], w[1], acc[t], 0, 0, 0);
        }
    }

    // A page with tokens that some row does not see: tokens behind the end become zeros, and so do NaN
    // values, after the rows that see one have become NaN.
    __device__ __forceinline__ void settle_values(uint4 v[kTiles], int key0, int end, int g)
    {
        bool some = false;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            uint4 nan;
            v[t] = keep_tokens(v[t], end - (key0 + 16 * g), nan);
            some |= any_of(nan);
        }
        if (!__any(some)) return;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            __builtin_amdgcn_sched_barrier(0);
            uint4 nan;
            keep_tokens(v[t], 16, nan);
            f16x8_t is_nan[2];
            decode16(as_ones(nan), is_nan);
            f32x4_t hit = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int h = 0; h < 2; ++h) hit = __builtin_amdgcn_mfma_f32_16x16x32_f16(is_nan[h], seen_ones(key0 + 16 * g + 8 * h, limit), hit, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = hit[i] > 0.0f ? __builtin_nanf("") : acc[t][i];
            v[t] = without(v[t], nan);
        }
    }
};

// log(l 2^t)
__device__ __forceinline__ float log_sum(float l, float t) { return l == 0.0f ? -__builtin_inff() : (t + __builtin_log2f(l)) * 0.6931471805599453f; }

template <bool F16>
__device__ __forceinline__ uint32_t pack_out(float lo, float hi)
{
    if (!F16) return pack_bf16x2(lo, hi);
    const f16x2_t p = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, p);
}

// The rows of key/value head h for the tokens behind the last sequence: zeros, and no weight.
__device__ __forceinline__ void clear_rows(const KvAttnArgs& p, int64_t first, int64_t end, int h)
{
    const int64_t rows = (end - first) * p.group;
    const int chunks = p.c.d / 8;
    for (int64_t i = threadIdx.x; i < rows * chunks; i += blockDim.x) {
        const int64_t row = i / chunks, at = (first + row / p.group) * p.q_heads + h * p.group + row % p.group;
        *reinterpret_cast<uint4*>(p.out + at * p.c.d + 8 * (i % chunks)) = make_uint4(0, 0, 0, 0);
        if (p.lse && i % chunks == 0) p.lse[at] = -__builtin_inff();
    }
}

// The rows [r0, r0 + 128) of one sequence and key/value head, or the part of their keys that is split
// `split`'s.
template <int D, bool F16>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_kv_attn_rows(KvAttnArgs p)
{
    constexpr int kPageBytes = kPage * D;            // of k, and of v
    constexpr int kCopies = D / 64;                  // of 4 KB, of k and of v
    // three pages of k codes, two of v in binary16
    __shared__ __attribute__((aligned(128))) uint8_t lds_k[3 * kPageBytes];
    __shared__ __attribute__((aligned(128))) uint8_t lds_v[2 * 2 * kPageBytes];
    __shared__ __attribute__((aligned(16))) PageInfo info[kInfo];
    __shared__ int nan_page[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, g = lane >> 5;

    // XCD (blockIdx % 8) takes a run of items, neighbours in which read the same pages
    uint32_t item;
    {
        const uint32_t per = p.items / 8, rest = p.items % 8, x = blockIdx.x % 8, i = blockIdx.x / 8;
        item = (x < rest ? x * (per + 1) : rest * (per + 1) + (x - rest) * per) + i;
    }
    const int split = (int)(item % p.splits);
    item /= p.splits;
    const uint32_t units = p.items / p.splits / p.c.heads;
    const int h = __builtin_amdgcn_readfirstlane((int)(item / units));
    uint32_t at64;
    // (the last units of a sequence first: with a causal mask they are the longest)
    KvSequence s{};
    const int b = __builtin_amdgcn_readfirstlane(kv_locate(p.b, p.units, units - 1 - item % units, at64, s));
    if (b == p.b.batch) {   // behind the last sequence
        if (split == 0) {
            const int64_t end = min(max((int64_t)p.b.q_start[b], (int64_t)0), p.b.tokens);
            const int64_t each = max(kRows / p.group, 1);   // tokens; as many units as kv_unit_count leaves take turns
            for (int64_t t = end + (int64_t)at64 * each; t < p.b.tokens; t += each * (int64_t)(units - kv_first_unit(p.b, p.units, b)))
                clear_rows(p, t, min(t + each, p.b.tokens), h);
        }
        return;
    }
    const int rows = s.n * p.group, tiles = (rows + kRows - 1) / kRows;   // (tokens * q_heads < 2^30)
    if (at64 >= (uint32_t)tiles) return;
    const int at = __builtin_amdgcn_readfirstlane((int)at64), r0 = at * kRows;
    const int last = min(r0 + kRows, rows) - 1;
    auto limit_of = [&](int row) -> int {
        if (!p.causal) return s.length;
        return (int)min(max(s.first + (uint32_t)row / (uint32_t)p.group + 1, (int64_t)0), (int64_t)s.length);
    };
    const int32_t* list = nullptr;
    int lo, hi;
    if (p.blocks) {
        // the query block's number, as p.listed counts them
        const int64_t block = r0 / p.block_rows;
        const int64_t unit = (p.b.q_start ? (int64_t)kv_first_unit(p.b, p.listed, b) : (int64_t)b * p.listed.each) + block;
        list = p.blocks + (unit * p.c.heads + h) * p.top;
        lo = 0, hi = p.b.width > 0 ? p.top : 0;   // (no pages, no list to look at)
    } else {
        lo = 0, hi = (limit_of(last) + kPage - 1) / kPage;
    }
    if (p.splits > 1) {
        const int per = max((hi + p.splits - 1) / p.splits, 1);
        lo = min(split * per, hi);
        hi = min(lo + per, hi);
    }

    WaveRows<D, F16> rowset;
    const int w0 = r0 + wave * kWaveRows;
    const bool idle = w0 >= rows;   // this wave copies only
    // The lane's row, from a value that the compiler does not know, so that what follows from it (a place, a limit) is
    // computed where it is rarely needed: kept through the loop it takes registers that d = 256 lacks (the values under
    // way are then waited for, to be moved: 0.79 against 0.73 ms on 3120 rows of 8 heads over 16000 tokens).
    auto own_row = [&]() -> int {
        int t = tid;
        asm volatile("" : "+v"(t));
        return w0 + (t & 31);
    };
    auto token_of = [&](int row) -> int64_t { return s.start + (uint32_t)row / (uint32_t)p.group; };
    auto head_of = [&](int row) -> int { return h * p.group + (uint32_t)row % (uint32_t)p.group; };
    auto own_limit = [&]() -> int {
        const int row = own_row();
        return row < rows ? limit_of(row) : 0;
    };
    {
        const int row = own_row();
        rowset.start(row < rows ? p.q + token_of(row) * p.ldq + (int64_t)head_of(row) * D : nullptr, g);
    }
    const int least = limit_of(min(w0, last)), most = limit_of(min(w0 + kWaveRows - 1, last));

    // k goes to LDS as it is, by asynchronous copies of this thread's 16 bytes of each 4 KB; v passes through
    // registers, where each thread decodes its share for all four waves. Lines of 128 bytes: of k a row (64
    // codes: two rows) of 128 codes, the next 128 behind all rows; of v a row's 64 tokens. Chunk c of row r
    // lies at c ^ ((r >> 1) & 7) (two rows a line: chunk c of line L at c ^ (L & 7)), so that the
    // reads of 32 rows by 64 lanes fall on all banks. Rows are in the matrix's order (row_key).
    const int line = tid / 8, slot = tid % 8;
    uint32_t from_k;
    {
        const int x = slot ^ (line & 7), row2 = 2 * line + (x >> 2);
        if (D == 64) from_k = (uint32_t)(((row2 & 32) + row_key(row2 & 31)) * D + (x & 3) * 16);
        else from_k = (uint32_t)(row_key(line) * D + (slot ^ ((line >> 1) & 7)) * 16);
    }
    const uint32_t base_k = (uint32_t)(uintptr_t)(lds_void_t*)lds_k + wave * 1024;
    auto copy_k = [&](const PageInfo& a, int buffer) {
        const i32x4_t rk = rsrc_words(p.c.k + ((int64_t)max(a.page, 0) * p.c.heads + h) * kPageBytes, kPageBytes);
        const uint32_t to = __builtin_amdgcn_readfirstlane(base_k + buffer * kPageBytes);
#pragma unroll
        for (int j = 0; j < kCopies; ++j) copy16_to_lds(rk, to + j * 4096, from_k, D == 64 ? 0 : (j & 1) * 32 * D + (j >> 1) * 128);
    };
    const int v_row = tid / 4, v_part = tid % 4;   // this thread's rows (v_row + 64 j), 16 tokens of each
    const int from_v = ((v_row & 32) + row_key(v_row & 31)) * kPage + v_part * 16;
    uint4 vr[kCopies];
    auto load_v = [&](const PageInfo& a) {
        const uint8_t* const src = p.c.v + ((int64_t)max(a.page, 0) * p.c.heads + h) * kPageBytes;
#pragma unroll
        for (int j = 0; j < kCopies; ++j) vr[j] = *reinterpret_cast<const uint4*>(src + from_v + j * 4096);
    };
    // Of a page with tokens that some row does not see, those behind the end and NaN become zeros, and
    // nan_page remembers a page with NaN.
    const int least_all = limit_of(r0);
    auto store_v = [&](const PageInfo& a, int i, int buffer) {
        const int sv = (v_row >> 1) & 7, key0 = first_key(a);
        if (key0 + kPage > least_all) {
            bool some = false;
#pragma unroll
            for (int j = 0; j < kCopies; ++j) {
                uint4 nan;
                vr[j] = keep_tokens(vr[j], s.length - (key0 + 16 * v_part), nan);
                if (any_of(nan)) some = true, vr[j] = without(vr[j], nan);
            }
            if (some) nan_page[buffer] = i;
        }
        uint8_t* const to = lds_v + buffer * (2 * kPageBytes) + v_row * 128;
#pragma unroll
        for (int j = 0; j < kCopies; ++j) {
            f16x8_t o[2];
            decode16(vr[j], o);
            *reinterpret_cast<f16x8_t*>(to + j * 8192 + ((2 * v_part) ^ sv) * 16) = o[0];
            *reinterpret_cast<f16x8_t*>(to + j * 8192 + ((2 * v_part + 1) ^ sv) * 16) = o[1];
        }
    };
    // Reads: lane (r, g) takes 32 codes of a key in two pieces, eight tokens of a value's element in one.
    const int sw = (r >> 1) & 7;
    const int k_line = D == 64 ? (r >> 1) * 128 : r * 128, k_chunk = D == 64 ? (r & 1) * 4 + 2 * g : 2 * g;

    look_up(p, b, h, s.length, list, lo, hi, info);
    if (tid < 2) nan_page[tid] = -1;
    __syncthreads();
    for (int first = lo; first < hi; first += kInfo) {
        const int count = min(hi - first, kInfo);
        if (first > lo) {
            __syncthreads();   // (all reads of the pages before are done)
            look_up(p, b, h, s.length, list, first, hi, info);
            if (tid < 2) nan_page[tid] = -1;
            __syncthreads();
        }
        PageInfo now = info_at(info, 0), next = now;
        copy_k(now, 0);
        load_v(now);
        __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));   // (the copies too, which the compiler does not count)
        store_v(now, first, 0);
        if (count > 1) {
            next = info_at(info, 1);
            copy_k(next, 1);
            load_v(next);
        }
        int buffer = 0;   // of k; page i of v is in buffer i & 1
        for (int i = 0; i < count; ++i) {
            // All waves' stores of page i, and their copies of it, which each waited for before it stored the
            // page's values, are done; so are the reads of page i - 1.
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(waitcnt_lgkm0());
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            PageInfo after = next;
            if (i + 1 < count) {
                __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));   // issued one page ago
                asm volatile("" ::: "memory");
                store_v(next, first + i + 1, (i + 1) & 1);
                if (i + 2 < count) {
                    after = info_at(info, i + 2);
                    copy_k(after, buffer == 0 ? 2 : buffer - 1);
                    load_v(after);
                }
            }
            const int key0 = first_key(now);
            if (!idle && key0 < most) {
                const uint8_t* const kb = lds_k + buffer * kPageBytes;
                const uint8_t* const vb = lds_v + (i & 1) * (2 * kPageBytes) + r * 128;
                auto key = [&](int kt, int st) {   // 16 codes: 64 (st / 2) + 32 g + 16 (st % 2) on
                    const uint8_t* const at_k = kb + k_line + (D == 64 ? kt * 2048 : kt * 4096 + (st >> 2) * 8192);
                    const int c = (D == 64 ? k_chunk : k_chunk + 4 * ((st >> 1) & 1)) + (st & 1);
                    return *reinterpret_cast<const uint4*>(at_k + ((c ^ sw) * 16));
                };
                auto value = [&](int kt, int half, int t) {
                    return *reinterpret_cast<const f16x8_t*>(vb + t * 4096 + (((4 * kt + 2 * g + half) ^ sw) * 16));
                };
                if (key0 + kPage > least_all && nan_page[i & 1] == first + i) {   // (also where this wave sees the whole page)
                    const uint8_t* const src = p.c.v + ((int64_t)now.page * p.c.heads + h) * kPageBytes + row_key(r) * kPage + 16 * g;
                    rowset.add_nan([&](int kt, int t) { return *reinterpret_cast<const uint4*>(src + t * 32 * kPage + 32 * kt); }, own_limit(), key0, s.length, g);
                }
                f32x16_t sc[2];
                f16x8_t w[2][2];
                rowset.scores(key, sc);
                const bool masked = key0 + kPage > least;
                f16x8_t v0[2][D / 32];
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int tt = 0; tt < D / 32; ++tt) v0[hf][tt] = value(0, hf, tt);
                __builtin_amdgcn_sched_barrier(0);
                if (masked) rowset.mask(sc, own_limit(), key0, g);
                rowset.weights(sc, p.scale, now.ek, now.ev, w);
                rowset.add_values(v0, value, w);
            }
            now = next, next = after;
            buffer = buffer == 2 ? 0 : buffer + 1;
        }
    }

    const int row = own_row();
    if (row >= rows) return;
    const float l = across32(rowset.run.l, added);
    const int64_t out_row = token_of(row) * p.q_heads + head_of(row);
    if (p.splits > 1) {
        float* const dst = p.part + (out_row * p.splits + split) * D + 16 * g;
        if (lo < hi)
#pragma unroll
            for (int t = 0; t < D / 32; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<float4*>(dst + 32 * t + 4 * i) = make_float4(rowset.acc[t][4 * i], rowset.acc[t][4 * i + 1],
                                                                                 rowset.acc[t][4 * i + 2], rowset.acc[t][4 * i + 3]);
        if (g == 0) part_sums(p)[out_row * p.splits + split] = make_float4(rowset.run.m, rowset.run.t, l, 0.0f);
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l, power = rowset.run.m - rowset.run.t - kLargest;
    auto out_at = [&](int t, int i) { return times_power(rowset.acc[t][i] * inv, power); };
    uint16_t* const dst = p.out + out_row * D + 16 * g;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 8)
            *reinterpret_cast<uint4*>(dst + 32 * t + i) =
                make_uint4(pack_out<F16>(out_at(t, i), out_at(t, i + 1)), pack_out<F16>(out_at(t, i + 2), out_at(t, i + 3)),
                           pack_out<F16>(out_at(t, i + 4), out_at(t, i + 5)), pack_out<F16>(out_at(t, i + 6), out_at(t, i + 7)));
    if (p.lse && g == 0) p.lse[out_row] = log_sum(l, rowset.run.t);
}

// Up to 16 rows of one sequence (or of one token, where each has its own pages) and key/value head.
// TURNS: max_query may be less than a sequence's rows.
template <int D, bool F16, bool TURNS>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_kv_attn_step(KvAttnArgs p)
{
    constexpr int kTiles = D / 16;
    constexpr int kPart = D < 128 ? D : 128;
    __shared__ __attribute__((aligned(16))) float acc[4][kStepRows][kPart];
    __shared__ float4 sums[4][kStepRows];   // as part_sums
    __shared__ __attribute__((aligned(16))) PageInfo info[kInfo];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;

    uint32_t item = blockIdx.x;
    const int split = (int)(item % p.splits);
    item /= p.splits;
    const int first_tile = (int)(item % p.column_tiles);
    item /= p.column_tiles;
    const int h = __builtin_amdgcn_readfirstlane((int)(item % p.c.heads));
    const uint32_t unit = item / p.c.heads;
    int b = (int)unit;
    KvSequence s{};
    if (p.blocks) {   // a unit is a token
        uint32_t at_token;
        b = __builtin_amdgcn_readfirstlane(kv_locate(p.b, KvUnits{1, (uint32_t)p.b.each, 1, 0}, unit, at_token, s));
    } else if (b < p.b.batch) {
        s = kv_sequence(p.b, b);
    }
    if (b == p.b.batch) {   // behind the last sequence
        if (split == 0 && first_tile == 0) {
            const int64_t end = min(max((int64_t)p.b.q_start[b], (int64_t)0), p.b.tokens);
            clear_rows(p, p.blocks ? unit : end, p.blocks ? unit + 1 : p.b.tokens, h);
        }
        return;
    }
    const int at = p.blocks ? (int)((int64_t)unit - s.start) : 0;   // the unit's first token in its sequence
    if (at < 0 || at >= s.n) return;
    const int rows = p.blocks ? p.group : s.n * p.group;
    // One tile, but for more rows than max_query said: the unit's workgroups then take turns (an instance of its own: the
    // loop costs the others 0.4 us in 10).
#pragma unroll 1
    for (int tile = first_tile; tile * kStepRows < rows; tile += p.column_tiles) {
        if (TURNS && tile != first_tile) __syncthreads();   // (the join before has been read)
        const int first_token = at + tile * kStepRows / p.group, last_token = at + (min((tile + 1) * kStepRows, rows) - 1) / p.group;
        auto limit_of = [&](int t) -> int {
            return p.causal ? (int)min(max(s.first + t + 1, (int64_t)0), (int64_t)s.length) : s.length;
        };
        const int32_t* list = p.blocks ? p.blocks + ((int64_t)unit * p.c.heads + h) * p.top : nullptr;
        int lo = 0, hi = list ? (p.b.width > 0 ? p.top : 0) : (limit_of(last_token) + kPage - 1) / kPage;
        if (p.splits > 1) {
            const int per = max((hi + p.splits - 1) / p.splits, 4);
            lo = min(split * per, hi);
            hi = min(lo + per, hi);
        }

        StepRows<D, F16> rowset;
        {
            const int row = tile * kStepRows + r, own = at + row / p.group;
            const bool valid = row < rows;
            rowset.start(valid ? p.q + (s.start + own) * p.ldq + (int64_t)(h * p.group + row % p.group) * D : nullptr, g);
            rowset.limit = valid ? limit_of(own) : 0;
        }
        const int least = limit_of(first_token), most = limit_of(last_token);

        const int from_k = (16 * (r >> 2) + (r & 3)) * D + D / 4 * g, from_v = r * kPage + 16 * g;
        uint4 kr[4][D / 64], vr[kTiles];
        auto load_k = [&](const PageInfo& a) {
            const uint8_t* const src = p.c.k + ((int64_t)max(a.page, 0) * p.c.heads + h) * (kPage * D);
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int j = 0; j < D / 64; ++j) kr[t][j] = *reinterpret_cast<const uint4*>(src + from_k + t * 4 * D + j * 16);
        };
        auto load_v = [&](const PageInfo& a) {
            const uint8_t* const src = p.c.v + ((int64_t)max(a.page, 0) * p.c.heads + h) * (kPage * D);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) vr[t] = *reinterpret_cast<const uint4*>(src + from_v + t * 16 * kPage);
        };
        look_up(p, b, h, s.length, list, lo, hi, info);
        __syncthreads();
        for (int first = lo; first < hi; first += kInfo) {
            const int count = min(hi - first, kInfo);
            if (first > lo) {
                __syncthreads();
                look_up(p, b, h, s.length, list, first, hi, info);
                __syncthreads();
            }
            PageInfo now{}, next{};
            int i = wave;
            if (i < count) {
                now = info_at(info, i);
                load_k(now);
                load_v(now);
            }
            for (; i < count; i += 4) {
                const bool more = i + 4 < count;
                if (more) next = info_at(info, i + 4);
                f32x4_t sc[4];
                f16x8_t w[2];
                rowset.scores(kr, sc);
                if (more) load_k(next);
                const int key0 = first_key(now);
                if (key0 < most) {
                    const bool masked = key0 + kPage > least;
                    if (masked) rowset.mask(sc, key0, g);
                    rowset.weights(sc, p.scale, now.ek, now.ev, w);
                    if (masked) rowset.settle_values(vr, key0, s.length, g);
                    rowset.add_values(vr, w);
                }
                if (more) load_v(next);
                now = next;
            }
        }

        // The four waves' parts of each row, joined in LDS, 128 elements at a time.
        const int kept = min(rows - tile * kStepRows, kStepRows);
        const float l = across16(across32(rowset.run.l, added), added);
        if (g == 0) sums[wave][r] = make_float4(rowset.run.m, rowset.run.t, l, 0.0f);
#pragma unroll
        for (int d0 = 0; d0 < D; d0 += kPart) {
            if (d0 > 0) __syncthreads();
#pragma unroll
            for (int t = 0; t < kPart / 16; ++t) {
                const f32x4_t v = rowset.acc[d0 / 16 + t];
                *reinterpret_cast<float4*>(&acc[wave][r][16 * t + 4 * g]) = make_float4(v[0], v[1], v[2], v[3]);
            }
            __syncthreads();
            for (int e = tid; e < kept * (kPart / 4); e += 256) {
                const int row_e = e / (kPart / 4), d = 4 * (e % (kPart / 4));
                float4 of[4];
                float m = kNone, t = kNone;
#pragma unroll
                for (int wv = 0; wv < 4; ++wv) of[wv] = sums[wv][row_e], m = fmaxf(m, of[wv].x), t = fmaxf(t, of[wv].y);
                float total = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int wv = 0; wv < 4; ++wv) {
                    const float f = __builtin_amdgcn_exp2f(of[wv].x - m);
                    const float4 a = *reinterpret_cast<const float4*>(&acc[wv][row_e][d]);
                    total += of[wv].z * __builtin_amdgcn_exp2f(of[wv].y - t);
                    o[0] += f * a.x, o[1] += f * a.y, o[2] += f * a.z, o[3] += f * a.w;
                }
                const int row_at = tile * kStepRows + row_e;
                const int64_t out_row = (s.start + at + row_at / p.group) * p.q_heads + h * p.group + row_at % p.group;
                if (p.splits > 1) {
                    *reinterpret_cast<float4*>(p.part + (out_row * p.splits + split) * D + d0 + d) = make_float4(o[0], o[1], o[2], o[3]);
                    if (d0 + d == 0) part_sums(p)[out_row * p.splits + split] = make_float4(m, t, total, 0.0f);
                } else {
                    const float inv = total == 0.0f ? 0.0f : 1.0f / total, power = m - t - kLargest;
                    *reinterpret_cast<uint2*>(p.out + out_row * D + d0 + d) =
                        make_uint2(pack_out<F16>(times_power(o[0] * inv, power), times_power(o[1] * inv, power)),
                                   pack_out<F16>(times_power(o[2] * inv, power), times_power(o[3] * inv, power)));
                    if (p.lse && d0 + d == 0) p.lse[out_row] = log_sum(total, t);
                }
            }
        }
        if (!TURNS) break;
    }
}

// One wave joins the splits of one row.
template <int D, bool F16>
__global__ __launch_bounds__(256) void k_kv_attn_join(KvAttnArgs p)
{
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= p.b.tokens * p.q_heads) return;
    if (p.b.q_start && row / p.q_heads >= p.b.q_start[p.b.batch]) return;   // behind the last sequence
    float4 own = make_float4(kNone, kNone, 0.0f, 0.0f);
    if (lane < p.splits) own = part_sums(p)[row * p.splits + lane];
    float m = own.x, t = own.y;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64)), t = fmaxf(t, __shfl_xor(t, off, 64));
    const float f = __builtin_amdgcn_exp2f(own.x - m);
    float total = own.z * __builtin_amdgcn_exp2f(own.y - t);
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) total += __shfl_xor(total, off, 64);
    float o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
    const float* const src = p.part + row * p.splits * D + lane * E;
    for (int i0 = 0; i0 < p.splits; i0 += 8) {   // (eight splits' loads before their use)
        float v[8][E];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) v[i][e] = src[(int64_t)min(i0 + i, p.splits - 1) * D + e];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // (a split without keys has not written its accumulators; lanes beyond the splits hold none)
            const bool some = __shfl(own.z, (i0 + i) & 63, 64) != 0.0f && i0 + i < p.splits;
            const float w = __shfl(f, (i0 + i) & 63, 64);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += some ? w * v[i][e] : 0.0f;
        }
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total, power = m - t - kLargest;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = times_power(o[e] * inv, power);
    uint16_t* const dst = p.out + row * D + lane * E;
    if (E == 1) dst[0] = (uint16_t)pack_out<F16>(o[0], 0.0f);
    else
#pragma unroll
        for (int e = 0; e + 1 < E; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack_out<F16>(o[e], o[e + 1]);
    if (p.lse && lane == 0) p.lse[row] = log_sum(total, t);
}

// Which kernel a call takes, its units and its splits.
struct Plan {
    bool step;
    int64_t items;          // workgroups
    int splits, column_tiles;
    int64_t bytes;          // of workspace
};

Plan make_plan(KvAttnArgs& p, int64_t max_query, int cus)
{
    Plan plan{};
    const int64_t n = p.b.q_start ? (max_query > 0 && max_query < p.b.tokens ? max_query : p.b.tokens) : p.b.tokens / p.b.batch;
    const int64_t most = p.blocks ? p.query_block : n;   // tokens of a unit of the step kernel
    // Steps up to 16 rows, at d = 256 up to 32 (4 queries in groups of 8 over 30000 tokens, eight sequences:
    // d = 64 37 us in either kernel, 128 58 us in two tiles of k_kv_attn_step against 52, 256 143 against 172).
    plan.step = p.blocks ? p.query_block == 1 : n * p.group <= (p.c.d == 256 ? 2 : 1) * kStepRows;
    const int64_t pages = p.blocks ? p.top : p.b.width;
    int64_t groups;
    if (plan.step) {
        plan.column_tiles = (int)((most * p.group + kStepRows - 1) / kStepRows);
        // (and one unit that clears what is behind the last sequence)
        groups = (p.blocks ? p.b.tokens : (int64_t)p.b.batch + (p.b.q_start ? 1 : 0)) * p.c.heads * plan.column_tiles;
    } else {
        plan.column_tiles = 1;
        p.units = KvUnits{kRows, (uint32_t)((n * p.group + kRows - 1) / kRows), p.group, 1};
        groups = (kv_unit_count(p.b, p.units) + (p.b.q_start ? 1 : 0)) * p.c.heads;
    }
    // Splits where the workgroups alone leave compute units idle: enough for four workgroups (steps) or two
    // (rows) on each, of at least eight (four) pages, and only where the pages that a workgroup is spared take longer than
    // the join and its launch (3.4 us) and the parts (a row's 0.13 + 0.0022 d ns, written and read). A page takes max(1, d / 100) us of
    // k_kv_attn_rows, d / 400 of k_kv_attn_step, whose waves take four at once. Measured (us, whole and split): one token,
    // d = 128, 20 pages 11.2 and 11.4, 24 12.6 and 10.9, 31 14.9 and 11.9; d = 256, 14 16.3 and 16.3, 16 17.6 and 15.5;
    // d = 64, 22 7.7 and 8.6; 3 x 77 rows of 12 heads of 64, 8 11.6 and 11.7, 12 15.9 and 12.4, 31 35.3 and 15.1;
    // 200 rows of 16 heads on 8 of 128, 8 15.4 and 16.9, 12 20.5 and 18.3; 4 x 300 rows of 8 heads of 128, 14 23.2 and 30.4,
    // 24 36.0 and 32.2; 1000 rows of 16 heads of 64, 24 28.0 and 32.2, 32 35.9 and 34.8.
    const int64_t want = (int64_t)cus * (plan.step ? 4 : 2), least = plan.step ? 8 : 4, rows = p.b.tokens * p.q_heads;
    int64_t splits = groups > 0 ? want / groups : 1;
    splits = std::min(std::min(splits, pages / least), (int64_t)kMostSplits);
    if (splits > 1) {
        const double page = plan.step ? p.c.d / 400.0 : std::max(1.0, p.c.d / 100.0), part = rows * (0.13 + 0.0022 * p.c.d) * 1e-3;
        if ((pages - (pages + splits - 1) / splits) * page < 3.4 + splits * part) splits = 1;
    }
    plan.splits = (int)std::max(splits, (int64_t)1);
    plan.items = groups * plan.splits;
    plan.bytes = plan.splits > 1 ? rows * plan.splits * (p.c.d + 4) * 4 : 0;
    return plan;
}

int check_plan(const Plan& plan)
{
    if (plan.items < ((int64_t)1 << 24)) return VDN_FP8_OK;
    return set_error(VDN_FP8_EINVAL, "kv_attention: %lld workgroups, 2^24 at most", (long long)plan.items);
}

template <int D, bool F16>
int launch(const KvAttnArgs& p, bool step, hipStream_t stream)
{
    int st;
    if (step) {
        if (p.turns) hipLaunchKernelGGL((k_kv_attn_step<D, F16, true>), dim3(p.items), dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((k_kv_attn_step<D, F16, false>), dim3(p.items), dim3(256), 0, stream, p);
        st = check_launch("kv_attention");
    } else {
        hipLaunchKernelGGL((k_kv_attn_rows<D, F16>), dim3(p.items), dim3(256), 0, stream, p);
        st = check_launch("kv_attention");
    }
    if (st != VDN_FP8_OK || p.splits == 1) return st;
    hipLaunchKernelGGL((k_kv_attn_join<D, F16>), dim3((unsigned)((p.b.tokens * p.q_heads + 3) / 4)), dim3(256), 0, stream, p);
    return check_launch("kv_attention join");
}

// The arguments that the size query and the call share.
int attn_arguments(const vdn_fp8_kv_cache* cache, const vdn_fp8_kv_batch* batch, int64_t q_heads, int64_t max_query, int64_t top,
                   int64_t query_block, bool listed, KvAttnArgs& p)
{
    const int st = kv_arguments("kv_attention", cache, batch, p.c, p.b);
    if (st != VDN_FP8_OK) return st;
    if (q_heads < 1 || q_heads > (1 << 16) || q_heads % p.c.heads)
        return set_error(VDN_FP8_EINVAL, "kv_attention: %lld query heads for %d key/value heads", (long long)q_heads, p.c.heads);
    if (max_query < 0) return set_error(VDN_FP8_EINVAL, "kv_attention: negative max_query");
    p.group = (int)(q_heads / p.c.heads), p.q_heads = (int)q_heads;
    if (listed) {
        if (top < 1 || top > (1 << 24)) return set_error(VDN_FP8_EINVAL, "kv_attention: top must be in [1, 2^24]");
        if (query_block < 1 || query_block > (1 << 20) || (query_block > 1 && query_block * p.group % kRows))
            return set_error(VDN_FP8_EINVAL, "kv_attention: query_block must be 1, or such that query_block * group is a multiple of %d "
                             "(got %lld with groups of %d)", kRows, (long long)query_block, p.group);
        p.top = (int)top, p.query_block = (int)query_block;
        p.block_rows = (int)std::min(query_block * p.group, (int64_t)1 << 30);
        const int64_t n = p.b.batch > 0 ? p.b.tokens / p.b.batch : 0;
        p.listed = KvUnits{(uint32_t)query_block, (uint32_t)((n + query_block - 1) / query_block), 1, query_block == 1 ? 0 : 1};
        p.blocks = (const int32_t*)(uintptr_t)4;   // replaced by the call
    }
    if (p.b.tokens * q_heads >= ((int64_t)1 << 30))
        return set_error(VDN_FP8_EINVAL, "kv_attention: %lld tokens of %lld heads, 2^30 rows at most", (long long)p.b.tokens, (long long)q_heads);
    return VDN_FP8_OK;
}

}  // namespace
}  // namespace vdn

using namespace vdn;

extern "C" int vdn_fp8_kv_attention_workspace_size(const vdn_fp8_kv_cache* cache, const vdn_fp8_kv_batch* batch, int64_t q_heads,
                                                   int64_t max_query, int64_t top, int64_t query_block, int64_t* bytes)
{
    KvAttnArgs p{};
    if (!bytes) return set_error(VDN_FP8_EINVAL, "kv_attention_workspace_size: null pointer");
    *bytes = 0;
    const int st = attn_arguments(cache, batch, q_heads, max_query, top, query_block, top > 0, p);
    if (st != VDN_FP8_OK || p.b.tokens == 0) return st;
    const int cus = device_cus();
    if (cus == 0) return set_error(VDN_FP8_ELAUNCH, "kv_attention_workspace_size: the device cannot be queried");
    const Plan plan = make_plan(p, max_query, cus);
    *bytes = plan.bytes;
    return check_plan(plan);
}

extern "C" int vdn_fp8_kv_attention(const vdn_fp8_kv_cache* cache, const vdn_fp8_kv_batch* batch, const void* query, int dtype,
                                    int64_t q_heads, int64_t ldq, int64_t max_query, float scale, int causal, const int32_t* blocks,
                                    int64_t top, int64_t query_block, void* out, float* lse, void* workspace, int64_t workspace_bytes,
                                    hipStream_t stream)
{
    KvAttnArgs p{};
    if (dtype != VDN_FP8_DTYPE_BF16 && dtype != VDN_FP8_DTYPE_F16) return set_error(VDN_FP8_EINVAL, "kv_attention: dtype must be bf16 or binary16");
    const int st = attn_arguments(cache, batch, q_heads, max_query, top, query_block, blocks != nullptr, p);
    if (st != VDN_FP8_OK || p.b.tokens == 0) return st;
    if (!query || !out) return set_error(VDN_FP8_EINVAL, "kv_attention: null pointer");
    if (ldq % 8 || ldq < q_heads * p.c.d) return set_error(VDN_FP8_EINVAL, "kv_attention: need ldq a multiple of 8 and >= q_heads * head_dim");
    if (!aligned(query, 16) || !aligned(out, 16) || !aligned(lse, 4) || !aligned(blocks, 4) || !aligned(workspace, 16))
        return set_error(VDN_FP8_EINVAL, "kv_attention: misaligned pointer (query, out, workspace 16 B; lse, blocks 4 B)");
    if (!(scale > 0.0f) || scale > 2e38f) return set_error(VDN_FP8_EINVAL, "kv_attention: scale must be positive and finite");
    const int cus = device_cus();
    if (cus == 0) return set_error(VDN_FP8_ELAUNCH, "kv_attention: the device cannot be queried");
    const Plan plan = make_plan(p, max_query, cus);
    const int fits = check_plan(plan);
    if (fits != VDN_FP8_OK) return fits;
    if (plan.bytes > 0 && (!workspace || workspace_bytes < plan.bytes))
        return set_error(VDN_FP8_EINVAL, "kv_attention: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)plan.bytes);
    p.q = (const uint16_t*)query, p.ldq = ldq, p.scale = scale * 1.4426950408889634f, p.causal = causal != 0;
    p.blocks = blocks, p.out = (uint16_t*)out, p.lse = lse, p.part = (float*)workspace;
    p.splits = plan.splits, p.column_tiles = plan.column_tiles, p.items = (uint32_t)plan.items;
    p.turns = p.b.q_start && !blocks && max_query > 0 && max_query < p.b.tokens;
    const bool f16 = dtype == VDN_FP8_DTYPE_F16;
    switch (p.c.d) {
        case 64: return f16 ? launch<64, true>(p, plan.step, stream) : launch<64, false>(p, plan.step, stream);
        case 128: return f16 ? launch<128, true>(p, plan.step, stream) : launch<128, false>(p, plan.step, stream);
        default: return f16 ? launch<256, true>(p, plan.step, stream) : launch<256, false>(p, plan.step, stream);
    }
}
