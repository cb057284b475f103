// Storing keys and values in the 8-bit cache, alone or behind QK preparation.
//
// A page holds 64 tokens of each key/value head: k [64][d] and v [d][64] in e4m3 (v transposed, so
// that the attention's second product reads tokens contiguously), a power-of-two scale each, and
// the mean key. For the tokens that a call puts into a page, with amax over their finite elements:
//   e     = least integer with amax <= 448 2^e, within [-100, 120]   (-100 for zeros)
//   e     = max(e, the page's own)        where the page keeps earlier tokens
//   code  = e4m3(x 2^-e)                  (one rounding: the product is exact; non-finite: NaN)
//   kept codes become e4m3(code 2^(own - e)), exact but for what falls below e4m3's least step
//   k_mean = bf16((sum of the page's codes / their number) 2^e)
// The sum is exact in binary32 in any order: codes are multiples of 2^-9 up to 448, and 64 of them
// stay below 2^24 steps. Powers of two cost e4m3 no precision (its own exponent absorbs them) and
// make every product here exact, so a result does not depend on how the tokens were cut into calls
// but for the least steps of kept codes.
//
// What bounds it: bytes, each key and value read once (16-byte loads) and each code written once.
// One workgroup takes a page of one head, so that the page's maximum needs no second pass over
// memory: the rows stay in registers between the maximum and the cast. A thread holds P = d / 32
// consecutive tokens of one 8-element chunk; k is packed along the chunk, v along the tokens, so the
// transposition is a matter of which values one conversion takes, and one pass through LDS makes
// whole 16-byte stores of it.
#include <stdint.h>

#include "kv_common.h"
#include "qk_prep.h"
#include "vdn_common.h"

namespace vdn {
namespace {

constexpr int kThreads = 256;
// Workgroups of a launch at most; each takes further units in steps of the grid.
constexpr int64_t kMostGroups = 1 << 20;

struct KvAppendArgs {
    KvCacheArgs c;
    KvBatchArgs b;
    KvUnits units;
    uint32_t page_units;  // pages of all sequences that the call may touch, times the heads
    int page_groups;      // workgroups that store pages; the others prepare queries
    const void* key;
    const void* value;
    int64_t ldk, ldv;
    // QK preparation (PREP)
    const uint16_t* query;
    uint16_t* out;
    int64_t ldq, ldo;
    int q_heads;
    const uint16_t* weight_q;
    const uint16_t* weight_k;
    float eps_q, eps_k;
    const void* cos;
    const void* sin;
    int64_t ldcs;
    int R, cs_bf16;
};

// Eight elements of a row as binary32.
template <int DTYPE>
__device__ __forceinline__ void load8(const void* base, int64_t i, float x[8])
{
    if (DTYPE == VDN_FP8_DTYPE_F32) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(base) + i);
        const uint4 lo = load_once(p), hi = load_once(p + 1);
        const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e]);
    } else {
        const uint4 v = load_once(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (DTYPE == VDN_FP8_DTYPE_BF16) {
                x[2 * e] = bf16_lo(w[e]);
                x[2 * e + 1] = bf16_hi(w[e]);
            } else {
                x[2 * e] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[e]);
                x[2 * e + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e] >> 16));
            }
        }
    }
}

__device__ __forceinline__ float power_of_two(int e)   // e in [-126, 127]
{
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// The magnitude of a finite value as bits, 0 for others: ordered as the magnitudes are.
__device__ __forceinline__ uint32_t finite_magnitude(float x)
{
    const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}

// Least e with amax <= 448 * 2^e (448 = 1.75 * 2^8), from amax's bits.
__device__ __forceinline__ int scale_exponent(uint32_t amax)
{
    const int e = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    return amax == 0 ? kLeastScale : min(max(e, kLeastScale), kMostScale);
}

// Four codes times 2^delta (delta <= 0), rounded again.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, int delta)
{
    const float f = power_of_two(max(delta, -126));
    return pack_e4m3x4(__builtin_amdgcn_cvt_f32_fp8(w, 0) * f, __builtin_amdgcn_cvt_f32_fp8(w, 1) * f,
                       __builtin_amdgcn_cvt_f32_fp8(w, 2) * f, __builtin_amdgcn_cvt_f32_fp8(w, 3) * f);
}

// What one lane of QK preparation keeps of its token: the rotation of its chunk.
struct Rotation {
    float cs[8], sn[8];
};

template <int D>
__device__ __forceinline__ Rotation load_rotation(const KvAppendArgs& p, int64_t token, int i0, bool rot)
{
    Rotation r;
    if (rot) {
        const int64_t at = token * p.ldcs + i0;
        uint4 c0, c1, s0, s1;
        if (p.cs_bf16) {
            c0 = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.cos) + at);
            s0 = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.sin) + at);
            c1 = s1 = make_uint4(0, 0, 0, 0);
        } else {
            const uint4* c = reinterpret_cast<const uint4*>(static_cast<const float*>(p.cos) + at);
            const uint4* s = reinterpret_cast<const uint4*>(static_cast<const float*>(p.sin) + at);
            c0 = c[0], c1 = c[1], s0 = s[0], s1 = s[1];
        }
        decode_table8(c0, c1, p.cs_bf16, r.cs);
        decode_table8(s0, s1, p.cs_bf16, r.sn);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) r.cs[e] = 1.0f, r.sn[e] = 0.0f;
    }
    return r;
}

__device__ __forceinline__ void load_weight(const uint16_t* weight, int i0, float w[8])
{
    if (!weight) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = 1.0f;
        return;
    }
    const uint4 v = *reinterpret_cast<const uint4*>(weight + i0);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) w[2 * e] = bf16_lo(u[e]), w[2 * e + 1] = bf16_hi(u[e]);
}

// The norm and the rotation of one chunk, the same operations as k_qk_prep's. Every lane takes part.
template <int D>
__device__ __forceinline__ void prepare8(const KvAppendArgs& p, const float x[8], const float w[8], float eps, const Rotation& r,
                                         int lane, float o[8])
{
    constexpr int G = D / 8;
    const int i0 = 8 * (lane % G), half = p.R / 2;
    const bool rot = i0 < p.R, first = i0 < half;
    const int partner = lane + (first ? half / 8 : -(half / 8));
    const float ss = head_sum_squares<G>(x);
    const float rstd = 1.0f / __builtin_sqrtf(ss / (float)D + eps);
    float n[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) n[e] = (x[e] * rstd) * w[e];
    rotate8<G>(n, r.cs, r.sn, p.R == D, rot, first, partner, lane, o);
}

// The queries of one token: each wave takes every fourth sweep of 64 lanes over its heads, four
// sweeps' loads before their arithmetic.
template <int D>
__device__ __forceinline__ void prepare_query(const KvAppendArgs& p, int64_t token)
{
    constexpr int G = D / 8, kSweeps = 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i0 = 8 * (lane % G), chunks = p.q_heads * G;
    float w[8];
    load_weight(p.weight_q, i0, w);
    const Rotation r = load_rotation<D>(p, token, i0, i0 < p.R);
    for (int base = wave * 64; base < chunks; base += 4 * 64 * kSweeps) {
        float x[kSweeps][8];
#pragma unroll
        for (int s = 0; s < kSweeps; ++s) {
            const int q = base + s * 256 + lane;
            if (q < chunks) load8<VDN_FP8_DTYPE_BF16>(p.query, token * p.ldq + 8 * q, x[s]);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) x[s][e] = 0.0f;
        }
#pragma unroll
        for (int s = 0; s < kSweeps; ++s) {
            const int q = base + s * 256 + lane;
            if (base + s * 256 >= chunks) break;   // (wave-uniform)
            float o[8];
            prepare8<D>(p, x[s], w, p.eps_q, r, lane, o);
            if (q < chunks) {
                const uint4 v = make_uint4(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4], o[5]),
                                           pack_bf16x2(o[6], o[7]));
                *reinterpret_cast<uint4*>(p.out + token * p.ldo + 8 * q) = v;
            }
        }
    }
}

template <int D, int DTYPE, bool PREP>
__device__ __forceinline__ void store_page(const KvAppendArgs& p, uint32_t unit, uint32_t* vt, float* part, uint32_t* top)
{
    constexpr int CH = D / 8;               // chunks of a row: one lane each
    constexpr int P = kPage * CH / kThreads;   // consecutive tokens of a thread: 2, 4, 8
    constexpr int kRow = 17;                // dwords of a v row in LDS (16 and one to spread the banks)
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h = (int)(unit % (uint32_t)p.c.heads);
    uint32_t at;
    const int b = kv_locate(p.b, p.units, unit / (uint32_t)p.c.heads, at);
    if (b == p.b.batch) return;   // behind the last sequence
    const KvSequence s = kv_sequence(p.b, b);
    const int64_t w64 = max(s.first, (int64_t)0) / kPage + at;
    if (w64 * kPage >= s.length) return;
    const int w = (int)w64;
    const int lo = (int)max(s.first - w64 * kPage, (int64_t)0), hi = (int)min((int64_t)s.length - w64 * kPage, (int64_t)kPage);
    if (lo >= hi) return;
    const int page = kv_page(p.b, p.c, b, w);
    if (page < 0) return;
    const int64_t ph = (int64_t)page * p.c.heads + h;
    const int64_t row0 = s.start + w64 * kPage - s.first;   // the call's row of the page's token 0 (may lie before the call)

    const int ch = tid % CH, i0 = 8 * ch, t0 = (tid / CH) * P;
    float kx[P][8], vx[P][8];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int t = t0 + i;
        if (t >= lo && t < hi) {
            load8<DTYPE>(p.key, (row0 + t) * p.ldk + h * D + i0, kx[i]);
            load8<DTYPE>(p.value, (row0 + t) * p.ldv + h * D + i0, vx[i]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) kx[i][e] = vx[i][e] = 0.0f;
        }
    }
    if (PREP) {
        float w8[8];
        load_weight(p.weight_k, i0, w8);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int t = t0 + i;
            const bool on = t >= lo && t < hi;
            const Rotation r = load_rotation<D>(p, on ? row0 + t : 0, i0, on && i0 < p.R);
            float o[8];
            prepare8<D>(p, kx[i], w8, p.eps_k, r, lane, o);
#pragma unroll
            for (int e = 0; e < 8; ++e) kx[i][e] = on ? round_bf16(o[e]) : 0.0f;   // the bf16 key that k_qk_prep stores
        }
    }

    uint32_t ak = 0, av = 0;
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            ak = max(ak, finite_magnitude(kx[i][e]));
            av = max(av, finite_magnitude(vx[i][e]));
        }
    ak = wave_max_u32(ak), av = wave_max_u32(av);
    if (lane == 0) top[wave] = ak, top[4 + wave] = av;
    const int own_k = p.c.k_scale[ph] - 127, own_v = p.c.v_scale[ph] - 127;
    __syncthreads();
    int ek = scale_exponent(max(max(top[0], top[1]), max(top[2], top[3])));
    int ev = scale_exponent(max(max(top[4], top[5]), max(top[6], top[7])));
    const bool keeps = lo > 0;
    if (keeps) ek = max(ek, own_k), ev = max(ev, own_v);
    const int dk = own_k - ek, dv = own_v - ev;   // used where the page keeps tokens: <= 0
    const float fk = power_of_two(-min(ek, 126)), fv = power_of_two(-min(ev, 126));

    // v: one dword of four tokens' codes per element, to LDS
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        uint32_t* const at_e = vt + (i0 + e) * kRow;
        if (P == 2) {
            const uint32_t c2 = pack_e4m3x4(vx[0][e] * fv, vx[1][e] * fv, 0.0f, 0.0f);
            reinterpret_cast<uint16_t*>(at_e)[t0 / 2] = (uint16_t)c2;
        } else {
#pragma unroll
            for (int i = 0; i + 3 < P; i += 4)
                at_e[(t0 + i) / 4] = pack_e4m3x4(vx[i][e] * fv, vx[i + 1][e] * fv, vx[i + 2][e] * fv, vx[i + 3][e] * fv);
        }
    }
    // k: eight codes of a token, and their sums
    float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    const bool means = p.c.k_mean != nullptr;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int t = t0 + i;
        if (t >= hi || (t < lo && !means && dk == 0)) continue;
        uint2* const dst = reinterpret_cast<uint2*>(p.c.k + (ph * kPage + t) * D + i0);
        uint2 c8;
        if (t >= lo) {
            c8 = make_uint2(pack_e4m3x4(kx[i][0] * fk, kx[i][1] * fk, kx[i][2] * fk, kx[i][3] * fk),
                            pack_e4m3x4(kx[i][4] * fk, kx[i][5] * fk, kx[i][6] * fk, kx[i][7] * fk));
            *dst = c8;
        } else {
            c8 = *dst;
            if (dk < 0) {
                c8 = make_uint2(rescale4(c8.x, dk), rescale4(c8.y, dk));
                *dst = c8;
            }
        }
        sum[0] += __builtin_amdgcn_cvt_f32_fp8(c8.x, 0), sum[1] += __builtin_amdgcn_cvt_f32_fp8(c8.x, 1);
        sum[2] += __builtin_amdgcn_cvt_f32_fp8(c8.x, 2), sum[3] += __builtin_amdgcn_cvt_f32_fp8(c8.x, 3);
        sum[4] += __builtin_amdgcn_cvt_f32_fp8(c8.y, 0), sum[5] += __builtin_amdgcn_cvt_f32_fp8(c8.y, 1);
        sum[6] += __builtin_amdgcn_cvt_f32_fp8(c8.y, 2), sum[7] += __builtin_amdgcn_cvt_f32_fp8(c8.y, 3);
    }
    if (means) {
#pragma unroll
        for (int off = CH; off < 64; off <<= 1)
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += __shfl_xor(sum[e], off, 64);
        if (lane < CH)
#pragma unroll
            for (int e = 0; e < 8; ++e) part[wave * D + i0 + e] = sum[e];
    }
    __syncthreads();
    if (means) {
        for (int i = tid; i < D / 2; i += kThreads) {
            float m[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float total = 0.0f;
#pragma unroll
                for (int g = 0; g < 4; ++g) total += part[g * D + 2 * i + e];
                m[e] = (total / (float)hi) * power_of_two(ek);
            }
            reinterpret_cast<uint32_t*>(p.c.k_mean + ph * D)[i] = pack_bf16x2(m[0], m[1]);
        }
    }
    // v: 16 tokens of one element per store; bytes outside [lo, hi) stay, but for kept codes at a new scale
    for (int u = tid; u < D * 4; u += kThreads) {
        const int d = u / 4, c = u % 4, first = 16 * c;
        const bool some = first < hi && first + 16 > lo, shift = keeps && dv < 0 && first < lo;
        if (!some && !shift) continue;
        uint4* const dst = reinterpret_cast<uint4*>(p.c.v + (ph * D + d) * kPage) + c;
        const uint32_t* const src = vt + d * kRow + 4 * c;
        uint32_t o[4] = {src[0], src[1], src[2], src[3]};
        if (first < lo || first + 16 > hi) {
            const uint4 old = *dst;
            const uint32_t was[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t kept = shift ? rescale4(was[j], dv) : was[j];
                uint32_t r = 0;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int token = first + 4 * j + t;
                    const uint32_t from = token < lo ? kept : token < hi ? o[j] : was[j];
                    r |= from & (0xffu << (8 * t));
                }
                o[j] = r;
            }
        }
        *dst = make_uint4(o[0], o[1], o[2], o[3]);
    }
    if (tid == 0) {
        p.c.k_scale[ph] = (uint8_t)(ek + 127);
        p.c.v_scale[ph] = (uint8_t)(ev + 127);
    }
}

template <int D, int DTYPE, bool PREP>
__global__ __launch_bounds__(kThreads) void k_kv_append(KvAppendArgs p)
{
    __shared__ uint32_t vt[D * 17];
    __shared__ float part[4 * D];
    __shared__ uint32_t top[8];
    if ((int)blockIdx.x < p.page_groups) {
        for (uint32_t u = blockIdx.x; u < p.page_units; u += p.page_groups) {
            store_page<D, DTYPE, PREP>(p, u, vt, part, top);
            __syncthreads();   // before the next page's values overwrite LDS
        }
    } else if (PREP) {
        const int64_t groups = gridDim.x - p.page_groups;
        for (int64_t t = (int64_t)blockIdx.x - p.page_groups; t < p.b.tokens; t += groups) prepare_query<D>(p, t);
    }
}

template <int DTYPE, bool PREP>
int launch(const KvAppendArgs& p, hipStream_t stream)
{
    const int64_t groups = p.page_groups + (PREP ? (p.b.tokens < kMostGroups ? p.b.tokens : kMostGroups) : 0);
    const dim3 grid((unsigned)groups), block(kThreads);
    switch (p.c.d) {
        case 64: hipLaunchKernelGGL((k_kv_append<64, DTYPE, PREP>), grid, block, 0, stream, p); break;
        case 128: hipLaunchKernelGGL((k_kv_append<128, DTYPE, PREP>), grid, block, 0, stream, p); break;
        default: hipLaunchKernelGGL((k_kv_append<256, DTYPE, PREP>), grid, block, 0, stream, p); break;
    }
    return check_launch("kv_append");
}

// The part of both entry points that concerns the cache; PREP's fields come after it.
int append_arguments(const char* what, const vdn_fp8_kv_cache* cache, const vdn_fp8_kv_batch* batch, const void* key, int64_t ldk,
                     const void* value, int64_t ldv, KvAppendArgs& p)
{
    const int st = kv_arguments(what, cache, batch, p.c, p.b);
    if (st != VDN_FP8_OK) return st;
    if (p.b.tokens == 0) return VDN_FP8_OK;
    if (!key || !value) return set_error(VDN_FP8_EINVAL, "%s: null pointer", what);
    const int64_t row = (int64_t)p.c.heads * p.c.d;
    if (ldk % 8 || ldv % 8 || ldk < row || ldv < row)
        return set_error(VDN_FP8_EINVAL, "%s: need ldk, ldv multiples of 8 and >= heads * head_dim", what);
    if (!aligned(key, 16) || !aligned(value, 16)) return set_error(VDN_FP8_EINVAL, "%s: key and value must be 16-byte aligned", what);
    // n tokens touch at most floor(n / 64) + 2 pages; none where they start at one's first token and end with it
    const int64_t n = p.b.q_start ? p.b.tokens : p.b.each;
    p.units = KvUnits{kPage, (uint32_t)((n + kPage - 2) / kPage + 1), 1, 2};
    const int64_t units = kv_unit_count(p.b, p.units) * p.c.heads;
    if (units >= INT32_MAX) return set_error(VDN_FP8_EINVAL, "%s: %lld pages and heads, 2^31 at most", what, (long long)units);
    p.page_units = (uint32_t)units;
    p.page_groups = (int)(p.page_units < kMostGroups ? p.page_units : kMostGroups);
    p.key = key, p.value = value, p.ldk = ldk, p.ldv = ldv;
    return VDN_FP8_OK;
}

}  // namespace

int kv_arguments(const char* what, const vdn_fp8_kv_cache* c, const vdn_fp8_kv_batch* b, KvCacheArgs& cache, KvBatchArgs& batch)
{
    if (!c || !b) return set_error(VDN_FP8_EINVAL, "%s: null cache or batch", what);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return set_error(VDN_FP8_EINVAL, "%s: head dim %lld not in {64, 128, 256}", what, (long long)c->head_dim);
    if (c->heads < 1 || c->heads > 4096) return set_error(VDN_FP8_EINVAL, "%s: heads must be in [1, 4096]", what);
    if (c->pages < 0 || c->pages > INT32_MAX) return set_error(VDN_FP8_EINVAL, "%s: pages must be in [0, 2^31)", what);
    if (b->tokens < 0 || b->tokens > INT32_MAX || b->batch < 0 || b->batch > (1 << 24))
        return set_error(VDN_FP8_EINVAL, "%s: tokens must be in [0, 2^31) and batch in [0, 2^24]", what);
    if (b->max_pages < 0 || b->max_pages > (1 << 24)) return set_error(VDN_FP8_EINVAL, "%s: max_pages must be in [0, 2^24]", what);
    if (b->tokens > 0) {
        if (b->batch == 0) return set_error(VDN_FP8_EINVAL, "%s: tokens of an empty batch", what);
        if (!b->lengths || (b->max_pages > 0 && !b->page_table)) return set_error(VDN_FP8_EINVAL, "%s: null page table or lengths", what);
        if (b->ldtable < 0) return set_error(VDN_FP8_EINVAL, "%s: negative ldtable", what);   // (0: one row for all)
        if (!b->q_start && b->tokens % b->batch)
            return set_error(VDN_FP8_EINVAL, "%s: %lld tokens do not divide among %lld sequences (pass q_start)", what,
                             (long long)b->tokens, (long long)b->batch);
        if (!aligned(b->page_table, 4) || !aligned(b->lengths, 4) || !aligned(b->q_start, 4))
            return set_error(VDN_FP8_EINVAL, "%s: page_table, lengths and q_start must be 4-byte aligned", what);
    }
    if (c->pages > 0) {
        if (!c->k || !c->v || !c->k_scale || !c->v_scale) return set_error(VDN_FP8_EINVAL, "%s: null cache buffer", what);
        if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_mean, 16))
            return set_error(VDN_FP8_EINVAL, "%s: k, v and k_mean must be 16-byte aligned", what);
    }
    cache = KvCacheArgs{(uint8_t*)c->k, (uint8_t*)c->v, (uint8_t*)c->k_scale, (uint8_t*)c->v_scale, (uint16_t*)c->k_mean,
                        c->pages, (int)c->heads, (int)c->head_dim};
    // (without pages every table entry is outside the pool: a table of no columns says the same)
    batch = KvBatchArgs{b->page_table, b->ldtable, c->pages > 0 ? (int)b->max_pages : 0, b->lengths, b->q_start, (int)b->batch, b->tokens,
                        b->batch > 0 ? (int)(b->tokens / b->batch) : 0};
    return VDN_FP8_OK;
}

}  // namespace vdn

using namespace vdn;

extern "C" int vdn_fp8_kv_append(const vdn_fp8_kv_cache* cache, const vdn_fp8_kv_batch* batch, const void* key, int64_t ldk,
                                 const void* value, int64_t ldv, int dtype, hipStream_t stream)
{
    KvAppendArgs p{};
    if (dtype != VDN_FP8_DTYPE_BF16 && dtype != VDN_FP8_DTYPE_F16 && dtype != VDN_FP8_DTYPE_F32)
        return set_error(VDN_FP8_EINVAL, "kv_append: unknown dtype %d", dtype);
    const int st = append_arguments("kv_append", cache, batch, key, ldk, value, ldv, p);
    if (st != VDN_FP8_OK || p.b.tokens == 0) return st;
    switch (dtype) {
        case VDN_FP8_DTYPE_BF16: return launch<VDN_FP8_DTYPE_BF16, false>(p, stream);
        case VDN_FP8_DTYPE_F16: return launch<VDN_FP8_DTYPE_F16, false>(p, stream);
        default: return launch<VDN_FP8_DTYPE_F32, false>(p, stream);
    }
}

extern "C" int vdn_fp8_qk_prep_append(const vdn_fp8_kv_cache* cache, const vdn_fp8_kv_batch* batch, const void* query, int64_t q_heads,
                                      int64_t ldq, const void* key, int64_t ldk, const void* value, int64_t ldv, const void* weight_q,
                                      float eps_q, const void* weight_k, float eps_k, const void* cos, const void* sin,
                                      int64_t rotary_dim, int64_t ldcs, int cs_bf16, void* out, int64_t ldo, hipStream_t stream)
{
    KvAppendArgs p{};
    const int st = append_arguments("qk_prep_append", cache, batch, key, ldk, value, ldv, p);
    if (st != VDN_FP8_OK || p.b.tokens == 0) return st;
    if (!query || !out) return set_error(VDN_FP8_EINVAL, "qk_prep_append: null pointer");
    if (q_heads < 1 || q_heads > (1 << 16)) return set_error(VDN_FP8_EINVAL, "qk_prep_append: query heads must be in [1, 65536]");
    if (rotary_dim < 0 || rotary_dim > p.c.d || rotary_dim % 16)
        return set_error(VDN_FP8_EINVAL, "qk_prep_append: rotary_dim %lld must be a multiple of 16 in [0, head_dim]", (long long)rotary_dim);
    if (rotary_dim > 0 && (!cos || !sin || ldcs < rotary_dim))
        return set_error(VDN_FP8_EINVAL, "qk_prep_append: rotary tables missing or row stride below rotary_dim");
    if (ldq % 8 || ldo % 8 || ldq < q_heads * p.c.d || ldo < q_heads * p.c.d)
        return set_error(VDN_FP8_EINVAL, "qk_prep_append: need ldq, ldo multiples of 8 and >= q_heads * head_dim");
    if (!(eps_q >= 0.0f) || !(eps_k >= 0.0f)) return set_error(VDN_FP8_EINVAL, "qk_prep_append: eps must be >= 0");
    if (!aligned(query, 16) || !aligned(out, 16) || !aligned(weight_q, 16) || !aligned(weight_k, 16) ||
        (rotary_dim > 0 && (!aligned(cos, 16) || !aligned(sin, 16) || ldcs % (cs_bf16 ? 8 : 4))))
        return set_error(VDN_FP8_EINVAL, "qk_prep_append: misaligned pointer (query, out, weights, cos, sin 16 B; table rows 16 B)");
    p.query = (const uint16_t*)query, p.out = (uint16_t*)out, p.ldq = ldq, p.ldo = ldo, p.q_heads = (int)q_heads;
    p.weight_q = (const uint16_t*)weight_q, p.weight_k = (const uint16_t*)weight_k, p.eps_q = eps_q, p.eps_k = eps_k;
    p.cos = cos, p.sin = sin, p.R = (int)rotary_dim, p.ldcs = ldcs, p.cs_bf16 = cs_bf16;
    return launch<VDN_FP8_DTYPE_BF16, true>(p, stream);
}
