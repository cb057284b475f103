// The arithmetic of QK preparation (per-head RMSNorm, then rotary embedding) on one
// 16-byte chunk of a head, shared by every kernel that runs it so that all give the
// same bits.
#pragma once

#include "vdn_common.h"

namespace vdn {

// Eight table values for elements i0 .. i0 + 7 of one row, rounded to bf16 and
// returned as binary32, from the 32 bytes at the row's element i0 (binary32
// tables use both halves, bf16 tables the first).
__device__ __forceinline__ void decode_table8(uint4 lo, uint4 hi, bool bf16, float v[8])
{
    if (bf16) {
        const uint32_t w[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[2 * e] = bf16_lo(w[e]); v[2 * e + 1] = bf16_hi(w[e]); }
    } else {
        const uint32_t raw[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const uint32_t r = pack_bf16x2(__uint_as_float(raw[e]), __uint_as_float(raw[e + 1]));
            v[e] = bf16_lo(r);
            v[e + 1] = bf16_hi(r);
        }
    }
}

// Lane exchanges inside a 16-lane DPP row (d = 128: one head per row), as
// register moves rather than LDS round trips.
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
constexpr int kDppRor8 = 0x128;        // lane i <- lane (i + 8) mod 16 within each row

// Sum over the 16 lanes of a row, every lane receiving it.
__device__ __forceinline__ float row16_sum(float v)
{
    v += dpp_f32<kDppXor1>(v);
    v += dpp_f32<kDppXor2>(v);
    v += dpp_f32<kDppHalfMirror>(v);
    v += dpp_f32<kDppMirror>(v);
    return v;
}

// The sum of squares of a head: each lane's own eight elements in order, then over the G = d / 8
// lanes that hold it.
template <int G>
__device__ __forceinline__ float head_sum_squares(const float x[8])
{
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
    if (G == 16) {
        ss = row16_sum(ss);
    } else {
#pragma unroll
        for (int off = 1; off < G; off <<= 1) ss += __shfl_xor(ss, off, 64);
    }
    return ss;
}

// The rotation of one chunk: o = n c + r s with r the partner chunk R / 16 lanes away (negated for
// the first half). full: R = d (uniform); rot: this chunk rotates; every lane of the wave takes part.
template <int G>
__device__ __forceinline__ void rotate8(const float n[8], const float cs[8], const float sn[8], bool full, bool rot,
                                        bool first, int partner, int lane, float o[8])
{
    if (G == 16 && full) {
        // R = d = 128: the partner chunk is 8 lanes away inside the row
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float pe = dpp_f32<kDppRor8>(n[e]);
            o[e] = n[e] * cs[e] + (first ? -pe : pe) * sn[e];
        }
    } else {
        // (the lanes of pass-through chunks read a value they do not use)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float pe = __shfl(n[e], rot ? partner : lane, 64);
            const float r = first ? -pe : pe;
            o[e] = rot ? n[e] * cs[e] + r * sn[e] : n[e];
        }
    }
}

}  // namespace vdn
