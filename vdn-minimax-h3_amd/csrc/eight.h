// Rows of bf16, float16 or float32 in chunks of eight elements: a lane's 16 bytes (32 of float32),
// loaded and stored through a row's buffer descriptor, so that chunks past the row read as zeros
// and are not stored, without a branch.
#pragma once

#include "vdn_common.h"

namespace vdn {

constexpr int kBf16 = VDN_FP8_DTYPE_BF16, kF16 = VDN_FP8_DTYPE_F16, kF32 = VDN_FP8_DTYPE_F32;

constexpr int element_bytes(int type) { return type == kF32 ? 4 : 2; }

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

template <int TYPE>
struct Eight {
    uint4 w[TYPE == kF32 ? 2 : 1];
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const void* p, int64_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}

// Chunk q of the row.
template <int TYPE, int POL>
__device__ __forceinline__ Eight<TYPE> load8(__amdgpu_buffer_rsrc_t row, uint32_t q)
{
    Eight<TYPE> v;
    const uint32_t off = q * (TYPE == kF32 ? 32u : 16u);
    v.w[0] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(row, off, 0, POL));
    if (TYPE == kF32) v.w[TYPE == kF32] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(row, off + 16u, 0, POL));
    return v;
}

template <int TYPE, int POL>
__device__ __forceinline__ void store8(const Eight<TYPE>& v, __amdgpu_buffer_rsrc_t row, uint32_t q)
{
    const uint32_t off = q * (TYPE == kF32 ? 32u : 16u);
    store_b128_settled<POL>(__builtin_bit_cast(i32x4_t, v.w[0]), row, off, 0);
    if (TYPE == kF32) store_b128_settled<POL>(__builtin_bit_cast(i32x4_t, v.w[TYPE == kF32]), row, off + 16u, 0);
}

template <int TYPE>
__device__ __forceinline__ void decode8(const Eight<TYPE>& v, float (&x)[8])
{
    const uint32_t w[4] = {v.w[0].x, v.w[0].y, v.w[0].z, v.w[0].w};
    if (TYPE == kF32) {
        const uint4 u = v.w[TYPE == kF32];
        const uint32_t h[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = __uint_as_float(w[e]);
            x[4 + e] = __uint_as_float(h[e]);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (TYPE == kBf16) {
            x[2 * e] = bf16_lo(w[e]);
            x[2 * e + 1] = bf16_hi(w[e]);
        } else {
            const f16x2_t p = __builtin_bit_cast(f16x2_t, w[e]);
            x[2 * e] = (float)p[0];
            x[2 * e + 1] = (float)p[1];
        }
    }
}

// Rounded to the type once (to nearest, ties to even).
template <int TYPE>
__device__ __forceinline__ Eight<TYPE> encode8(const float (&x)[8])
{
    Eight<TYPE> v;
    uint32_t w[4];
    if (TYPE == kF32) {
        v.w[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
        v.w[TYPE == kF32] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
        return v;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (TYPE == kBf16) {
            w[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
        } else {
            const f16x2_t p = {(_Float16)x[2 * e], (_Float16)x[2 * e + 1]};
            w[e] = __builtin_bit_cast(uint32_t, p);
        }
    }
    v.w[0] = make_uint4(w[0], w[1], w[2], w[3]);
    return v;
}

// host: whether two sets of `rows` rows share memory, of of_a and of_b bytes, lda and ldb bytes apart. Two column
// ranges of one matrix do not.
inline bool rows_overlap(const void* a, int64_t lda, int64_t of_a, const void* b, int64_t ldb, int64_t of_b, int64_t rows)
{
    const int64_t from_a = (int64_t)(uintptr_t)a, from_b = (int64_t)(uintptr_t)b;
    if (from_a + (rows - 1) * lda + of_a <= from_b || from_b + (rows - 1) * ldb + of_b <= from_a) return false;
    if (lda != ldb) return true;
    const int64_t apart = ((from_b - from_a) % lda + lda) % lda;   // b's columns behind a's
    return apart < of_a || apart + of_b > lda;
}

}  // namespace vdn
