// QK preparation with positions of several axes: per-head RMSNorm (or none) of q and of k, then the rotary
// embedding whose angles come from each token's positions, in one launch.
//
//   rstd     = 1 / sqrt(sum_i x[i]^2 / d + eps),   n[i] = (x[i] rstd) w[i]        (binary32)
//   angle_j  = positions[t][axis[j]] * inv_freq[j]                                (j < R / 2)
//   halves:    pair j is elements (j, j + R/2);  pairs: elements (2j, 2j + 1)
//   out[lo]  = n[lo] cos(angle_j) - n[hi] sin(angle_j),   out[hi] = n[hi] cos(angle_j) + n[lo] sin(angle_j)
//   out[i]   = n[i] for i >= R
// rounded once, at the store. Cosines and sines are binary32 (a table of bf16 values, as k_qk_prep takes,
// is off by 2^-9 of a turn's radius).
//
// Angles. What matters of an angle is its fraction of a turn, and at far positions binary32 has none of it
// left (position 10^6 at frequency 1: half a unit in the last place is 2^-5 rad). So the turns p f / 2 pi are
// formed in binary64, the nearest whole number is taken off by an exact fma, and a quarter turn's remainder,
// |g| <= pi / 4, goes to binary32, where Taylor's series to g^9 and g^10 have errors below 2^-28.
//
// Layout. Chunks are eight elements, a lane's; a head is d / 8 consecutive lanes, as in k_qk_prep; a slot is 64 chunks of q or of k
// of a token, and a wave takes up to CPL slots of one token, the last of q and the first of k among them. Its lanes first compute one angle
// each (R / 2 <= 128 of them), leave cosine and sine in the wave's own LDS, and read those of their chunks from there: an angle costs
// its wave about 60 operations once, and not once for each of the lanes that need it. The little that the angles need is fetched ahead of
// the slots (loads come back in order), so that they are ready when those are.
//
// On the card: 32760 tokens of 40 + 40 heads of 128 224 us, 6.0 TB/s read and written, with the VALU busy 0.86 of the time (235 with what
// the angles need fetched behind the rows); 5329 tokens of 16 + 16 heads of 64 11.3; 6405 float32 tokens of 32 + 8 heads of 128 52,
// 5.1 TB/s; 16 tokens of 40 + 8 heads 3.8, a chain of the positions' load, the angles and the store.
#include <stdint.h>

#include "eight.h"
#include "qk_prep.h"
#include "vdn_common.h"

namespace vdn {
namespace {

constexpr int kLanes = 64;
constexpr int kWaves = 4;            // of a workgroup
constexpr int kMostAxes = 8;
constexpr int kMostPairs = 128;      // R / 2 at d = 256

struct RopeSide {
    const void* x;        // [T, heads, d], row stride ld
    int64_t ld;
    int heads, slots;
    int norm;
    const void* weight;   // [d] or NULL
    float eps;
    void* out;
    int64_t ldo;
};

struct RopeArgs {
    RopeSide side[2];
    int64_t T;
    int d, R;
    const double* inv_freq;   // [R / 2]
    const int32_t* axis;      // [R / 2]
    const void* positions;    // [T, axes]
    int64_t ldpos;
    int axes, position_type;
    int spans, per;           // waves of a token, and slots of a wave
    int once;                 // the outputs only pass through the last-level cache
};

__device__ __forceinline__ double position_at(const RopeArgs& p, int64_t at)
{
    if (p.position_type == VDN_FP8_POSITION_I32) return (double)static_cast<const int32_t*>(p.positions)[at];
    if (p.position_type == VDN_FP8_POSITION_I64) return (double)static_cast<const int64_t*>(p.positions)[at];
    return (double)static_cast<const float*>(p.positions)[at];
}

// Cosine and sine of 2 pi p f, f in turns.
__device__ __forceinline__ void turn(double p, double f, float& cosine, float& sine)
{
    // p f less its nearest whole number; once more where p f is so large that the first leaves a few turns
    double r = __builtin_fma(p, f, -__builtin_rint(p * f));
    r -= __builtin_rint(r);
    const double quarter = __builtin_rint(4.0 * r);
    const float g = (float)((r - 0.25 * quarter) * 6.283185307179586477);
    const float z = g * g;
    // sin g = g - g^3/3! + ... + g^9/9!, cos g = 1 - g^2/2! + ... - g^10/10!
    const float s = __builtin_fmaf(g * z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), g);
    const float c = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const int q = (int)quarter & 3;
    const float a = q & 1 ? s : c, b = q & 1 ? c : s;
    cosine = q == 1 || q == 2 ? -a : a;
    sine = q & 2 ? -b : b;
}

// G = d / 8 lanes of a head; CPL slots a wave at most; PAIRS: which elements a pair is.
template <int TYPE, int G, int CPL, bool PAIRS>
__global__ __launch_bounds__(kWaves * kLanes) void k_rope_axes(RopeArgs p, int64_t first_token)
{
    __shared__ float turned[kWaves][2][kMostPairs];
    const int lane = threadIdx.x & (kLanes - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const uint32_t unit = blockIdx.x * kWaves + wave;
    const int64_t t = first_token + unit / (uint32_t)p.spans;
    if (t >= p.T) return;
    const int first_slot = (int)(unit % (uint32_t)p.spans) * p.per, slots = min(p.side[0].slots + p.side[1].slots - first_slot, p.per);
    const int j = lane % G, i0 = 8 * j, half = p.R / 2;
    const int esize = element_bytes(TYPE);

    // what the angles need, then the weights, then the slots
    const int a0 = min(lane, half - 1), a1 = min(lane + kLanes, half - 1);   // (-1 without any)
    const double mine = lane < p.axes ? position_at(p, t * p.ldpos + lane) : 0.0;
    int axis[2] = {0, 0};
    double f[2] = {0.0, 0.0};
    if (half > 0) {
        axis[0] = p.axis[a0];
        f[0] = p.inv_freq[a0];
        if (half > kLanes) {
            axis[1] = p.axis[a1];
            f[1] = p.inv_freq[a1];
        }
    }
    Eight<TYPE> raw_weight[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const void* w = p.side[s].weight;
        raw_weight[s] = load8<TYPE, 0>(row_buffer(w ? w : (const void*)p.positions, w ? p.d * esize : 0), (uint32_t)j);
    }
    // slot c of the wave: its side, its row and this lane's chunk of it
    auto is_key = [&](int c) { return first_slot + c >= p.side[0].slots; };
    auto chunk = [&](int c) { return (uint32_t)((first_slot + c - (is_key(c) ? p.side[0].slots : 0)) * kLanes + lane); };
    auto row = [&](int c, const void* x0, int64_t ld0, const void* x1, int64_t ld1) {
        const bool key = is_key(c);
        const int64_t bytes = (int64_t)(key ? p.side[1].heads : p.side[0].heads) * p.d * esize;
        return row_buffer((const uint8_t*)(key ? x1 : x0) + t * (key ? ld1 : ld0) * esize, c < slots ? bytes : 0);
    };
    Eight<TYPE> v[CPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c) v[c] = load8<TYPE, kBufferLoadOnce>(row(c, p.side[0].x, p.side[0].ld, p.side[1].x, p.side[1].ld), chunk(c));
    __builtin_amdgcn_sched_barrier(0);

    if (half > 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int a = lane + kLanes * i;
            if (kLanes * i < half) {
                float c, s;
                turn(__shfl(mine, min(max(axis[i], 0), p.axes - 1), kLanes), f[i] * 0.15915494309189533577, c, s);
                if (a < half) {
                    turned[wave][0][a] = c;
                    turned[wave][1][a] = s;
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }

    const bool rot = i0 < p.R;
    const bool first = i0 < half;                                     // (halves)
    const int partner = lane + (first ? half / 8 : -(half / 8));      // (halves: the chunk R / 2 elements away)
    float cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int pair = PAIRS ? i0 / 2 + e / 2 : (first ? i0 : i0 - half) + e;
        cs[e] = rot ? turned[wave][0][pair] : 1.0f;
        sn[e] = rot ? turned[wave][1][pair] : 0.0f;
    }
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
        if (c >= slots) break;
        const bool key = is_key(c);
        float n[8], o[8];
        decode8<TYPE>(v[c], n);
        if (key ? p.side[1].norm : p.side[0].norm) {
            float w[8];
            decode8<TYPE>(key ? raw_weight[1] : raw_weight[0], w);
            const bool weight = key ? p.side[1].weight != nullptr : p.side[0].weight != nullptr;
            const float ss = head_sum_squares<G>(n);
            const float rstd = 1.0f / __builtin_sqrtf(ss / (float)p.d + (key ? p.side[1].eps : p.side[0].eps));
#pragma unroll
            for (int e = 0; e < 8; ++e) n[e] = (n[e] * rstd) * (weight ? w[e] : 1.0f);
        }
        if (PAIRS) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                o[e] = rot ? n[e] * cs[e] - n[e + 1] * sn[e] : n[e];
                o[e + 1] = rot ? n[e + 1] * cs[e] + n[e] * sn[e] : n[e + 1];
            }
        } else {
            rotate8<G>(n, cs, sn, p.R == p.d, rot, first, partner, lane, o);
        }
        const __amdgpu_buffer_rsrc_t outr = row(c, p.side[0].out, p.side[0].ldo, p.side[1].out, p.side[1].ldo);
        if (p.once) store8<TYPE, kBufferLoadOnce>(encode8<TYPE>(o), outr, chunk(c));
        else store8<TYPE, 0>(encode8<TYPE>(o), outr, chunk(c));
    }
}

// Outputs of at least this many bytes are stored non-temporally: beyond what the last-level cache holds,
// cached stores only evict each other.
constexpr int64_t kOnceBytes = 256ll << 20;
// A slot a wave below this, up to six from there on: us with one and with six, 40 + 40 heads of 128: 256 tokens 5.4 and 6.4, 512 8.6 and 8.3, 1024
// 14.4 and 12.2; 40 + 8: 512 5.9 and 7.1, 800 8.4 and 8.8, 1024 9.9 and 9.6, 3000 22 and 17; 16 + 16 of 64: 1024 4.9 and 6.1, 3000 10.0 and 9.4.
constexpr int64_t kFewTokens = 1024;

template <int TYPE, int G, bool PAIRS>
int launch(RopeArgs p, hipStream_t stream)
{
    int slots = 0;
    for (RopeSide& s : p.side) slots += s.slots = (s.heads * G + kLanes - 1) / kLanes;
    // up to six slots a wave, alike
    const int most = p.T < kFewTokens ? 1 : 6;
    p.spans = (slots + most - 1) / most;
    p.per = (slots + p.spans - 1) / p.spans;
    p.spans = (slots + p.per - 1) / p.per;
    p.once = p.T * (p.side[0].heads + p.side[1].heads) * p.d * element_bytes(TYPE) >= kOnceBytes;
    const int64_t slab = kLaunchRows * kWaves / p.spans, T = p.T;   // tokens of a launch
    return in_slabs(T, slab, [&](int64_t t, int64_t tokens) {
        const dim3 grid((unsigned)((tokens * p.spans + kWaves - 1) / kWaves)), block(kWaves * kLanes);
        p.T = t + tokens;
        if (p.per <= 1) hipLaunchKernelGGL((k_rope_axes<TYPE, G, 1, PAIRS>), grid, block, 0, stream, p, t);
        else if (p.per <= 2) hipLaunchKernelGGL((k_rope_axes<TYPE, G, 2, PAIRS>), grid, block, 0, stream, p, t);
        else if (p.per <= 4) hipLaunchKernelGGL((k_rope_axes<TYPE, G, 4, PAIRS>), grid, block, 0, stream, p, t);
        else hipLaunchKernelGGL((k_rope_axes<TYPE, G, 6, PAIRS>), grid, block, 0, stream, p, t);
        return check_launch("qk_prep_axes");
    });
}

template <int TYPE, int G>
int launch(const RopeArgs& p, bool pairs, hipStream_t stream)
{
    return pairs ? launch<TYPE, G, true>(p, stream) : launch<TYPE, G, false>(p, stream);
}

template <int TYPE>
int launch_type(const RopeArgs& p, bool pairs, hipStream_t stream)
{
    return p.d == 64 ? launch<TYPE, 8>(p, pairs, stream) : p.d == 128 ? launch<TYPE, 16>(p, pairs, stream) : launch<TYPE, 32>(p, pairs, stream);
}

}  // namespace
}  // namespace vdn

using namespace vdn;

extern "C" int vdn_fp8_qk_prep_axes(const void* query, int64_t q_heads, int64_t ldq, const void* key, int64_t k_heads, int64_t ldk,
                                    int64_t T, int64_t d, int dtype, int norm_q, const void* weight_q, float eps_q, int norm_k,
                                    const void* weight_k, float eps_k, const double* inv_freq, const int32_t* axis, int64_t rotary_dim,
                                    int pairs, const void* positions, int position_type, int64_t axes, int64_t ldpos, void* out_q,
                                    int64_t ldoq, void* out_k, int64_t ldok, hipStream_t stream)
{
    const char* what = "qk_prep_axes";
    if (T < 0 || q_heads < 0 || k_heads < 0) return set_error(VDN_FP8_EINVAL, "%s: negative shape", what);
    if (dtype < kBf16 || dtype > kF32) return set_error(VDN_FP8_EINVAL, "%s: unknown dtype %d", what, dtype);
    if (d != 64 && d != 128 && d != 256) return set_error(VDN_FP8_EINVAL, "%s: head dim %lld not in {64, 128, 256}", what, (long long)d);
    if (q_heads * d > 65536 || k_heads * d > 65536) return set_error(VDN_FP8_EINVAL, "%s: more than 65536 elements a token", what);
    if (T == 0 || q_heads + k_heads == 0) return VDN_FP8_OK;
    const int64_t unit = pairs ? 8 : 16;
    if (rotary_dim < 0 || rotary_dim > d || rotary_dim % unit)
        return set_error(VDN_FP8_EINVAL, "%s: the rotary dim %lld must be a multiple of %lld in [0, d]", what, (long long)rotary_dim, (long long)unit);
    if (rotary_dim > 0) {
        if (!inv_freq || !axis || !positions) return set_error(VDN_FP8_EINVAL, "%s: null pointer (frequencies, axes or positions)", what);
        if (axes < 1 || axes > kMostAxes || ldpos < axes) return set_error(VDN_FP8_EINVAL, "%s: 1 to %d axes, and positions' row stride >= that (got %lld, %lld)", what, kMostAxes, (long long)axes, (long long)ldpos);
        if (position_type < VDN_FP8_POSITION_I32 || position_type > VDN_FP8_POSITION_F32) return set_error(VDN_FP8_EINVAL, "%s: unknown type of positions %d", what, position_type);
        const uintptr_t wide = position_type == VDN_FP8_POSITION_I64 ? 8 : 4;
        if (!aligned(inv_freq, 8) || !aligned(axis, 4) || !aligned(positions, wide)) return set_error(VDN_FP8_EINVAL, "%s: misaligned pointer (frequencies, axes or positions)", what);
    }
    if (!(eps_q >= 0.0f) || !(eps_k >= 0.0f)) return set_error(VDN_FP8_EINVAL, "%s: eps must be >= 0", what);
    auto bad = [&](const void* x, int64_t heads, int64_t ld, const void* out, int64_t ldo) {
        return heads && (!x || !out || ld % 8 || ldo % 8 || ld < heads * d || ldo < heads * d || !aligned(x, 16) || !aligned(out, 16));
    };
    if (bad(query, q_heads, ldq, out_q, ldoq) || bad(key, k_heads, ldk, out_k, ldok))
        return set_error(VDN_FP8_EINVAL, "%s: rows must be given, 16-byte aligned, with strides multiples of 8 and >= heads * d", what);
    if (!aligned(weight_q, 16) || !aligned(weight_k, 16)) return set_error(VDN_FP8_EINVAL, "%s: misaligned pointer (weights 16 B)", what);
    // (waves write their slots of a token when they are done with them, in any order)
    struct Rows { const void* at; int64_t ld, bytes; };
    const int64_t E = element_bytes(dtype);
    auto overlap = [&](const Rows& a, const Rows& b) { return a.bytes && b.bytes && rows_overlap(a.at, a.ld, a.bytes, b.at, b.ld, b.bytes, T); };
    const Rows q{query, ldq * E, q_heads * d * E}, k{key, ldk * E, k_heads * d * E}, oq{out_q, ldoq * E, q.bytes}, ok{out_k, ldok * E, k.bytes};
    if ((out_q == query ? q_heads && T > 1 && ldoq != ldq : overlap(q, oq)) || (out_k == key ? k_heads && T > 1 && ldok != ldk : overlap(k, ok)) ||
        overlap(q, ok) || overlap(k, oq) || overlap(oq, ok))
        return set_error(VDN_FP8_EINVAL, "%s: an output must be its own input, with its stride, or not overlap other rows", what);
    const RopeArgs p{{{query, ldq, (int)q_heads, 0, norm_q != 0, weight_q, eps_q, out_q, ldoq},
                      {key, ldk, (int)k_heads, 0, norm_k != 0, weight_k, eps_k, out_k, ldok}},
                     T, (int)d, (int)rotary_dim, inv_freq, axis, positions, ldpos, rotary_dim > 0 ? (int)axes : 0, position_type, 0, 0, 0};
    return dtype == kBf16 ? launch_type<kBf16>(p, pairs != 0, stream)
         : dtype == kF16  ? launch_type<kF16>(p, pairs != 0, stream)
                          : launch_type<kF32>(p, pairs != 0, stream);
}
