// The residual's addition, the root-mean-square norm with its affine, and the codes of the next
// projection's input, in one pass over the rows:
//   h[k]    = S(fma(g[i][k], b[k], r[k]))                (r[k] + b[k] without a gate; S the stream's type)
//   rstd    = 1 / sqrt(sum_k h[k]^2 / K + eps)           (binary32)
//   n[k]    = fma(h[k] * rstd, w[k] (1 + sc[i][k]), sh[i][k])
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
constexpr int kMostWaves = 16;   // of a workgroup
// One chunk a thread up to here, two beyond: us with one and with two, rows of 5120: 64 rows 4.2 and 4.4, 300 6.4 and 6.3, 512 7.7 and 7.9, 821
// 11.6 and 10.4, 3485 31 and 29; rows of 4104: 512 7.1 and 7.2, 821 10.3 and 10.1, 1500 14.5 and 15.4, 3485 26.5 and 26.0.
constexpr int64_t kFewRows = 512;

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

// Codes of eight values n + low: (n + low) (R + R_low), R + R_low = 1 / scale before the scale's roundings; the
// product and its corrections are rounded once. EXACT: the IEEE quotient, for scales that are not finite.
template <bool EXACT>
__device__ __forceinline__ uint2 codes8(const float (&n)[8], const float (&low)[8], float scale, float R, float R_low)
{
    float q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = EXACT ? n[e] / scale : __builtin_fmaf(n[e], R, __builtin_fmaf(low[e], R, n[e] * R_low));
    return make_uint2(pack_e4m3x4(q[0], q[1], q[2], q[3]), pack_e4m3x4(q[4], q[5], q[6], q[7]));
}

// v, or eight ones where it is absent.
template <int TYPE>
__device__ __forceinline__ Eight<TYPE> or_ones(const Eight<TYPE>& v, bool present)
{
    constexpr uint32_t one = TYPE == kBf16 ? 0x3f803f80u : TYPE == kF16 ? 0x3c003c00u : 0x3f800000u;
    if (present) return v;
    Eight<TYPE> u = v;
    u.w[0] = make_uint4(one, one, one, one);
    if (TYPE == kF32) u.w[TYPE == kF32] = u.w[0];
    return u;
}

// Streams of at least this many bytes are stored non-temporally: they only pass through the last-level cache.
constexpr int64_t kOnceBytes = 256ll << 20;

// A workgroup per row, of as many waves as its chunks fill: thread t holds chunk t, or t and t + threads, as
// binary32 in registers from the addition to the codes, and the partial sums of squares and the maxima meet in
// LDS. One chunk a thread makes a row short for the few of a step (16 of 5120: 4.3 us on the card); two halve what
// every wave does once, which costs time where there are many (32760 of 5376, gated and modulated: 243 us and
// 5.1 TB/s, as fast as a copy of those bytes; with one chunk a thread 3% slower). All loads go out before the first of
// them is used, the tables' as soon as the row's index is there; a table that is absent is a descriptor of no
// bytes, which reads zeros. S, B: the types of the stream, and of the branch and its parameters; AFFINE: scale and
// shift are there; ONCE: hidden is stored non-temporally.
template <int S, int B, int CPL, bool AFFINE, bool ONCE>
__global__ __launch_bounds__(kMostWaves * kLanes) void k_add_norm(AddNormArgs p, int waves, int64_t first)
{
    __shared__ float ssum[kMostWaves];
    __shared__ uint32_t smax[kMostWaves];
    __shared__ int32_t slow;
    const int64_t row = first + blockIdx.x;
    const int lane = threadIdx.x & (kLanes - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const int nch = (int)(p.K >> 3);
    const int64_t sbytes = p.K * element_bytes(S), bbytes = p.K * element_bytes(B);
    auto chunk = [&](int c) { return (uint32_t)threadIdx.x + (uint32_t)(kLanes * waves * c); };
    auto table = [&](const void* t, int64_t at) { return row_buffer(t ? (const uint8_t*)t + at * element_bytes(B) : (const uint8_t*)p.branch, t ? bbytes : 0); };

    const __amdgpu_buffer_rsrc_t rr = row_buffer((const uint8_t*)p.residual + row * p.ldr * element_bytes(S), sbytes);
    const __amdgpu_buffer_rsrc_t br = row_buffer((const uint8_t*)p.branch + row * p.ldb * element_bytes(B), bbytes);
    Eight<S> r[CPL];
    Eight<B> b[CPL], g[CPL], w[CPL], sc[CPL], sh[CPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
        r[c] = load8<S, kBufferLoadOnce>(rr, chunk(c));
        b[c] = load8<B, kBufferLoadOnce>(br, chunk(c));
    }
    int64_t ti = 0;
    if (p.index) ti = min(max((int64_t)p.index[row], (int64_t)0), p.rows - 1);
    const __amdgpu_buffer_rsrc_t gr = table(p.gate, ti * p.ldgate), wr = table(p.weight, 0), scr = table(p.scale, ti * p.ldmod),
                                 shr = table(p.shift, ti * p.ldmod);
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
        g[c] = load8<B, 0>(gr, chunk(c));
        w[c] = load8<B, 0>(wr, chunk(c));
    }
    if (AFFINE)
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
            sc[c] = load8<B, 0>(scr, chunk(c));
            sh[c] = load8<B, 0>(shr, chunk(c));
        }
    __builtin_amdgcn_sched_barrier(0);

    const __amdgpu_buffer_rsrc_t hr = row_buffer((uint8_t*)p.hidden + row * p.ldh * element_bytes(S), sbytes);
    float n[CPL][8], low[CPL][8], ss = 0.0f;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
        float x[8], y[8], f[8];
        decode8<S>(r[c], x);
        decode8<B>(b[c], y);
        decode8<B>(or_ones<B>(g[c], p.gate), f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = __builtin_fmaf(f[e], y[e], x[e]);
            if (S == kF16) asm volatile("" : "+v"(x[e]));   // a binary32 value first, not one fma that rounds to binary16
        }
        const Eight<S> h = encode8<S>(x);
        store8<S, ONCE ? kBufferLoadOnce : 0>(h, hr, chunk(c));
        decode8<S>(h, n[c]);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(n[c][e], n[c][e], ss);
    }
    ss = wave_sum_f32(ss);
    // (a lane of each 16 takes a wave's, and the 16 add them up by exchanges)
    if (lane == 0) ssum[wave] = ss;
    __syncthreads();
    ss = lane % kMostWaves < waves ? ssum[lane % kMostWaves] : 0.0f;
    ss += __uint_as_float(dpp_u32<kDppXor1>(__float_as_uint(ss)));
    ss += __uint_as_float(dpp_u32<kDppXor2>(__float_as_uint(ss)));
    ss += __uint_as_float(dpp_u32<kDppHalfMirror>(__float_as_uint(ss)));
    ss += __uint_as_float(dpp_u32<kDppMirror>(__float_as_uint(ss)));
    // rstd + rstd_low = 1 / sqrt(square), the second a step of Newton's method (none where square is 0 or not finite)
    const float square = ss / (float)p.K + p.eps, rstd = 1.0f / __builtin_sqrtf(square), root = square * rstd;
    const float off = __builtin_fmaf(-root, rstd, 1.0f) - __builtin_fmaf(square, rstd, -root) * rstd;
    const float rstd_low = __builtin_fabsf(off) < 0x1p-20f ? 0.5f * rstd * off : 0.0f;

    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
        float f[8], u[8], v[8];
        decode8<B>(or_ones<B>(w[c], p.weight), f);
        if (AFFINE) {
            decode8<B>(sc[c], u);
            decode8<B>(sh[c], v);
        }
        float most = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // n + low: low is what the rounding of h rstd leaves out of n, and with a shift that of rstd (without one it cancels
            // against the scale's), without a shift that of the product with w. A code moves where such errors carry a value across a
            // border between two, the largest's (below) for a whole row: 110 to 140 of the 176 million codes of 32760 x 5376 (means of
            // inputs of six seeds: 129) and none of 16 x 5120 without a shift (of twelve); 301 and 6.3 where n, the scale and the quotient
            // are each rounded to binary32.
            const float t = n[c][e] * rstd, left = __builtin_fmaf(n[c][e], rstd, -t);
            const float t_low = AFFINE ? __builtin_fmaf(n[c][e], rstd_low, left) : left;
            if (AFFINE) {
                const float factor = f[e] * (1.0f + u[e]);
                low[c][e] = t_low * factor;
                n[c][e] = __builtin_fmaf(t, factor, v[e]);
            } else {
                n[c][e] = t * f[e];
                low[c][e] = __builtin_fmaf(t_low, f[e], __builtin_fmaf(t, f[e], -n[c][e]));
            }
            most = __builtin_elementwise_maximum(most, __builtin_fabsf(n[c][e]));
        }
        if (chunk(c) < (uint32_t)nch) top = __builtin_elementwise_maximum(top, most);   // (0 times an infinite rstd, past the row)
    }
    uint32_t bits = wave_max_u32(__float_as_uint(top) & 0x7fffffffu);
    if (lane == 0) smax[wave] = bits;
    if (threadIdx.x == 0) slow = 0x80000000;
    __syncthreads();
    bits = wave_max_u32(lane % kMostWaves < waves ? smax[lane % kMostWaves] : 0u);
    // the largest's own low part; of several that are as large a lane's last, and of lanes the largest (as integers in the same
    // order), so that it is the same in every call
    if (__float_as_uint(top) == bits) {
        float rest = 0.0f;
#pragma unroll
        for (int c = 0; c < CPL; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (__builtin_fabsf(n[c][e]) == top) rest = __builtin_copysignf(1.0f, n[c][e]) * low[c][e];
        const int32_t word = (int32_t)__float_as_uint(rest);
        __hip_atomic_fetch_max(&slow, word < 0 ? word ^ 0x7fffffff : word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
    __syncthreads();
    const float most = __uint_as_float(bits), scale = row_scale(most);
    if (threadIdx.x == 0) p.y_scale[row] = scale;
    // 1 / scale in two parts: 448 / (most and its low part), or 1 / scale at the floor
    const bool floor = most / 448.0f < 1e-12f;
    const float over = floor ? 1.0f : 448.0f, under = floor ? scale : most;
    const float rest = floor ? 0.0f : __uint_as_float((uint32_t)(slow < 0 ? slow ^ 0x7fffffff : slow));
    const float R = over / under, R_low = (__builtin_fmaf(-R, under, over) - R * rest) / under;
    const bool finite = __builtin_isfinite(scale);
    const __amdgpu_buffer_rsrc_t yr = row_buffer(p.y + row * p.ldy, p.K);
    const __amdgpu_buffer_rsrc_t nr = row_buffer(p.normed ? (uint8_t*)p.normed + row * p.ldn * element_bytes(B) : p.y, p.normed ? bbytes : 0);
    typedef int i32x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
        if (p.normed) store8<B, 0>(encode8<B>(n[c]), nr, chunk(c));
        const uint2 q = finite ? codes8<false>(n[c], low[c], scale, R, R_low) : codes8<true>(n[c], low[c], scale, R, R_low);
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(i32x2_t, q), yr, chunk(c) * 8u, 0, 0);
    }
}

template <int S, int B>
int launch(const AddNormArgs& p, hipStream_t stream)
{
    const int64_t nch = p.K / 8;
    const bool once = p.M * p.K * element_bytes(S) >= kOnceBytes;
    return in_slabs(p.M, kLaunchRows / 4, [&](int64_t m, int64_t rows) {
        // (a workgroup has 1024 threads at most, and a launch fewer than 2^32 work-items)
        const bool two = nch > kMostWaves * kLanes || (nch > 256 && p.M > kFewRows);
        const int waves = (int)((nch + kLanes * (two ? 2 : 1) - 1) / (kLanes * (two ? 2 : 1)));
#define VDN_LAUNCH(n, a, o) hipLaunchKernelGGL((k_add_norm<S, B, n, a, o>), dim3((unsigned)rows), dim3(waves * kLanes), 0, stream, p, waves, m)
#define VDN_FORM(n)                                            \
        if (p.scale && once) VDN_LAUNCH(n, true, true);        \
        else if (p.scale) VDN_LAUNCH(n, true, false);          \
        else if (once) VDN_LAUNCH(n, false, true);             \
        else VDN_LAUNCH(n, false, false);
        if (two) { VDN_FORM(2) } else { VDN_FORM(1) }
#undef VDN_FORM
#undef VDN_LAUNCH
        return check_launch("add_norm_quantize");
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
    // (workgroups write their rows when they are done with them, in any order)
    struct Rows { const void* at; int64_t ld, bytes; };
    const int64_t S = element_bytes(stream_type), B = element_bytes(dtype);
    auto overlap = [&](const Rows& a, const Rows& b) { return a.at && b.at && rows_overlap(a.at, a.ld, a.bytes, b.at, b.ld, b.bytes, M); };
    const Rows r{residual, ldr * S, K * S}, b{branch, ldb * B, K * B}, h{hidden, ldh * S, K * S}, codes{y, ldy, K}, n{normed, ldn * B, K * B};
    if ((hidden == residual ? M > 1 && ldh != ldr : overlap(r, h)) ||
        (hidden == branch ? stream_type != dtype || (M > 1 && ldh != ldb) : overlap(b, h)))
        return set_error(VDN_FP8_EINVAL, "%s: hidden must be residual or branch itself, with its stride and type, or not overlap them", what);
    for (const Rows& in : {r, b, h})
        if (overlap(in, codes) || overlap(in, n)) return set_error(VDN_FP8_EINVAL, "%s: y and normed must not overlap the other rows", what);
    if (overlap(codes, n)) return set_error(VDN_FP8_EINVAL, "%s: y and normed must not overlap the other rows", what);
    const AddNormArgs p{residual, ldr, branch, ldb, gate, ldgate, weight, mod_scale, mod_shift, ldmod, index, rows, eps, M, K,
                        hidden, ldh, (uint8_t*)y, ldy, y_scale, normed, ldn};
    if (stream_type == kF32)
        return dtype == kBf16 ? launch<kF32, kBf16>(p, stream) : dtype == kF16 ? launch<kF32, kF16>(p, stream) : launch<kF32, kF32>(p, stream);
    return dtype == kBf16 ? launch<kBf16, kBf16>(p, stream) : launch<kF16, kF16>(p, stream);
}
