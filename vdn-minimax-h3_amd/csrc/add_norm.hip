// The residual's addition, the root-mean-square norm with its affine, and the codes of the next
// projection's input, in one pass over the rows:
//   h[k]    = S(fma(g[i][k], b[k], r[k]))                (r[k] + b[k] without a gate; S the stream's type)
//   rstd    = 1 / sqrt(sum_k h[k]^2 / K + eps)           (binary32)
//   n[k]    = fma(h[k] * rstd, w[k] (1 + sc[i][k]), sh[i][k])      ((h rstd) w without a table)
//   scale   = max(max_k |n[k]| / 448, 1e-12),  code[k] = e4m3(n[k] / scale),  normed[k] = B(n[k])
// with i = index[row], clamped into the tables. The stream is rounded where it is stored, and the
// stored row is the one that is normed, as if a later call read it. n is not rounded before the
// codes: e4m3's half step is 2^-4 of a value, and a rounding to bf16 in between would only move values
// across its borders.
#include <stdint.h>

#include "eight.h"
#include "vdn_common.h"

namespace vdn {
namespace {

constexpr int kLanes = 64;

struct AddNormArgs {
    const void* residual;
    int64_t ldr;
    const void* branch;
    int64_t ldb;
    const void* gate;      // [rows, K] or NULL
    int64_t ldgate;
    const void* weight;    // [K] or NULL
    const void* scale;     // [rows, K] or NULL, as shift
    const void* shift;
    int64_t ldmod;
    const int32_t* index;  // [M] or NULL (row 0)
    int64_t rows;
    float eps;
    int64_t M, K;
    void* hidden;
    int64_t ldh;
    uint8_t* y;
    int64_t ldy;
    float* y_scale;
    void* normed;          // [M, K] or NULL
    int64_t ldn;
};

// A value's code from its scale s and r = RN(1 / s); EXACT: the IEEE quotient, for scales that are not finite.
template <bool EXACT>
__device__ __forceinline__ uint2 codes8(const float (&n)[8], float s, float r)
{
    float q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = EXACT ? n[e] / s : div_by_scale(n[e], s, r);
    return make_uint2(pack_e4m3x4(q[0], q[1], q[2], q[3]), pack_e4m3x4(q[4], q[5], q[6], q[7]));
}

// A workgroup of WPR waves per row: wave w holds chunks 64 w + lane + 64 WPR c of it, as binary32 in
// registers from the addition to the codes; the partial sums of squares and the maxima meet in LDS.
// S, B: the types of the stream, and of the branch and its parameters.
template <int S, int B, int WPR, int CPL>
__global__ __launch_bounds__(WPR * kLanes) void k_add_norm(AddNormArgs p, int64_t first)
{
    __shared__ float ssum[WPR];
    __shared__ uint32_t smax[WPR];
    const int64_t row = first + blockIdx.x;
    const int lane = threadIdx.x & (kLanes - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const int nch = (int)(p.K >> 3);
    const int64_t sbytes = p.K * element_bytes(S), bbytes = p.K * element_bytes(B);
    auto chunk = [&](int c) { return (uint32_t)(wave * kLanes + lane + kLanes * WPR * c); };

    const __amdgpu_buffer_rsrc_t rr = row_buffer((const uint8_t*)p.residual + row * p.ldr * element_bytes(S), sbytes);
    const __amdgpu_buffer_rsrc_t br = row_buffer((const uint8_t*)p.branch + row * p.ldb * element_bytes(B), bbytes);
    Eight<S> r[CPL];
    Eight<B> b[CPL], g[CPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
        r[c] = load8<S, kBufferLoadOnce>(rr, chunk(c));
        b[c] = load8<B, kBufferLoadOnce>(br, chunk(c));
    }
    int64_t ti = 0;
    if (p.index) ti = min(max((int64_t)p.index[row], (int64_t)0), p.rows - 1);
    if (p.gate) {
        const __amdgpu_buffer_rsrc_t gr = row_buffer((const uint8_t*)p.gate + ti * p.ldgate * element_bytes(B), bbytes);
#pragma unroll
        for (int c = 0; c < CPL; ++c) g[c] = load8<B, 0>(gr, chunk(c));
    }

    const __amdgpu_buffer_rsrc_t hr = row_buffer((uint8_t*)p.hidden + row * p.ldh * element_bytes(S), sbytes);
    float n[CPL][8], ss = 0.0f;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
        float x[8], y[8];
        decode8<S>(r[c], x);
        decode8<B>(b[c], y);
        if (p.gate) {
            float f[8];
            decode8<B>(g[c], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __builtin_fmaf(f[e], y[e], x[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] += y[e];
        }
        const Eight<S> h = encode8<S>(x);
        store8<S, 0>(h, hr, chunk(c));
        decode8<S>(h, n[c]);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(n[c][e], n[c][e], ss);
    }
    ss = wave_sum_f32(ss);
    if (WPR > 1) {
        if (lane == 0) ssum[wave] = ss;
        __syncthreads();
        ss = ssum[0];
#pragma unroll
        for (int w = 1; w < WPR; ++w) ss += ssum[w];
    }
    const float rstd = 1.0f / __builtin_sqrtf(ss / (float)p.K + p.eps);

    const __amdgpu_buffer_rsrc_t wr = row_buffer(p.weight ? p.weight : p.branch, p.weight ? bbytes : 0);
    const __amdgpu_buffer_rsrc_t scr = row_buffer(p.scale ? (const uint8_t*)p.scale + ti * p.ldmod * element_bytes(B) : p.branch, p.scale ? bbytes : 0);
    const __amdgpu_buffer_rsrc_t shr = row_buffer(p.shift ? (const uint8_t*)p.shift + ti * p.ldmod * element_bytes(B) : p.branch, p.shift ? bbytes : 0);
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
        float w[8];
        decode8<B>(load8<B, 0>(wr, chunk(c)), w);
        if (!p.weight)
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = 1.0f;
        if (p.scale) {
            float sc[8], sh[8];
            decode8<B>(load8<B, 0>(scr, chunk(c)), sc);
            decode8<B>(load8<B, 0>(shr, chunk(c)), sh);
#pragma unroll
            for (int e = 0; e < 8; ++e) n[c][e] = __builtin_fmaf(n[c][e] * rstd, w[e] * (1.0f + sc[e]), sh[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) n[c][e] = (n[c][e] * rstd) * w[e];
        }
        float most = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) most = __builtin_elementwise_maximum(most, __builtin_fabsf(n[c][e]));
        if (chunk(c) < (uint32_t)nch) top = __builtin_elementwise_maximum(top, most);   // (0 times an infinite rstd, past the row)
    }
    uint32_t bits = wave_max_u32(__float_as_uint(top) & 0x7fffffffu);
    if (WPR > 1) {
        if (lane == 0) smax[wave] = bits;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WPR; ++w) bits = max(bits, smax[w]);
    }
    const float scale = row_scale(__uint_as_float(bits));
    if (threadIdx.x == 0) p.y_scale[row] = scale;
    const float inverse = 1.0f / scale;
    const bool finite = __builtin_isfinite(scale);
    const __amdgpu_buffer_rsrc_t yr = row_buffer(p.y + row * p.ldy, p.K);
    const __amdgpu_buffer_rsrc_t nr = row_buffer(p.normed ? (uint8_t*)p.normed + row * p.ldn * element_bytes(B) : p.y, p.normed ? bbytes : 0);
    typedef int i32x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
        if (p.normed) store8<B, 0>(encode8<B>(n[c]), nr, chunk(c));
        const uint2 q = finite ? codes8<false>(n[c], scale, inverse) : codes8<true>(n[c], scale, inverse);
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(i32x2_t, q), yr, chunk(c) * 8u, 0, 0);
    }
}

template <int S, int B>
int launch(const AddNormArgs& p, hipStream_t stream)
{
    const int64_t nch = p.K / 8;
    return in_slabs(p.M, kLaunchRows / 4, [&](int64_t m, int64_t rows) {
        // (a workgroup has 1024 threads at most, and a launch fewer than 2^32 work-items)
#define VDN_CASE(w, n)                                                                                             \
        if (nch <= (int64_t)w * n * kLanes) {                                                                      \
            hipLaunchKernelGGL((k_add_norm<S, B, w, n>), dim3((unsigned)rows), dim3(w * kLanes), 0, stream, p, m); \
            return check_launch("add_norm_quantize");                                                              \
        }
        VDN_CASE(1, 1) VDN_CASE(1, 2)
        if (p.M <= 512) { VDN_CASE(4, 1) VDN_CASE(8, 1) VDN_CASE(16, 1) VDN_CASE(16, 2) }
        VDN_CASE(4, 1) VDN_CASE(4, 2) VDN_CASE(4, 3) VDN_CASE(4, 4) VDN_CASE(4, 6) VDN_CASE(4, 8)
#undef VDN_CASE
        return set_error(VDN_FP8_EINVAL, "add_norm_quantize: unsupported K");
    });
}

}  // namespace
}  // namespace vdn

using namespace vdn;

extern "C" int vdn_fp8_add_norm_quantize(const void* residual, int stream_type, int64_t ldr, const void* branch, int dtype, int64_t ldb,
                                         int64_t M, int64_t K, const void* gate, int64_t ldgate, const void* weight, float eps,
                                         const void* mod_scale, const void* mod_shift, int64_t ldmod, const int32_t* index, int64_t rows,
                                         void* hidden, int64_t ldh, void* y, int64_t ldy, float* y_scale, void* normed, int64_t ldn,
                                         hipStream_t stream)
{
    const char* what = "add_norm_quantize";
    if (M < 0 || K < 0) return set_error(VDN_FP8_EINVAL, "%s: negative shape", what);
    if (dtype < kBf16 || dtype > kF32 || !(stream_type == dtype || (stream_type == kF32 && dtype < kF32)))
        return set_error(VDN_FP8_EINVAL, "%s: the stream's dtype %d must be the branch's (%d), or binary32", what, stream_type, dtype);
    if (M == 0) return VDN_FP8_OK;
    if (K < 8 || K % 8 || K > 16384) return set_error(VDN_FP8_EINVAL, "%s: K=%lld must be a multiple of 8, at most 16384", what, (long long)K);
    if (!residual || !branch || !hidden || !y || !y_scale) return set_error(VDN_FP8_EINVAL, "%s: null pointer", what);
    if (!mod_scale != !mod_shift) return set_error(VDN_FP8_EINVAL, "%s: scale and shift go together", what);
    if (!(eps >= 0.0f)) return set_error(VDN_FP8_EINVAL, "%s: eps must be >= 0", what);
    const bool tables = gate || mod_scale;
    if (tables && rows < 1) return set_error(VDN_FP8_EINVAL, "%s: a table needs at least 1 row", what);
    if (index && !tables) return set_error(VDN_FP8_EINVAL, "%s: an index needs a table", what);
    auto bad = [&](int64_t ld) { return ld % 8 != 0 || ld < K; };
    if (bad(ldr) || bad(ldb) || bad(ldh) || bad(ldy) || (normed && bad(ldn)) || (gate && rows > 1 && bad(ldgate)) ||
        (mod_scale && rows > 1 && bad(ldmod)))
        return set_error(VDN_FP8_EINVAL, "%s: need the row strides multiples of 8 and >= K", what);
    if (!aligned(residual, 16) || !aligned(branch, 16) || !aligned(hidden, 16) || !aligned(y, 8) || !aligned(y_scale, 4) ||
        !aligned(normed, 16) || !aligned(gate, 16) || !aligned(weight, 16) || !aligned(mod_scale, 16) || !aligned(mod_shift, 16) ||
        !aligned(index, 4))
        return set_error(VDN_FP8_EINVAL, "%s: misaligned pointer (rows, weight and tables 16 B; y 8 B)", what);
    const AddNormArgs p{residual, ldr, branch, ldb, gate, ldgate, weight, mod_scale, mod_shift, ldmod, index, rows, eps, M, K,
                        hidden, ldh, (uint8_t*)y, ldy, y_scale, normed, ldn};
    if (stream_type == kF32)
        return dtype == kBf16 ? launch<kF32, kBf16>(p, stream) : dtype == kF16 ? launch<kF32, kF16>(p, stream) : launch<kF32, kF32>(p, stream);
    return dtype == kBf16 ? launch<kBf16, kBf16>(p, stream) : launch<kF16, kF16>(p, stream);
}
