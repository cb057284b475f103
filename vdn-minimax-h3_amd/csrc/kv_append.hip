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
// memory: the rows stay in registers between the maximum and the cast. A thread holds two consecutive
// tokens of one 8-element chunk, packed as they came (4 d threads a page; with four tokens and 256 threads
// the registers left a compute unit 2.3 waves a SIMD: 67 us for 3120 tokens of 40 + 2 x 40 heads, 51 us now).
// k is packed along the chunk, v along the tokens, so the transposition is a matter of which values one
// conversion takes, and one pass through LDS makes whole 16-byte stores of it. Where pages alone fill the
// part, a workgroup takes up to four heads of a page (1: 59 us): it reads the next head's rows while it
// stores one, and keeps the tokens' rotations. (3.4 TB/s of reads and writes at those 3120 tokens; 47.5 us a
// call among others.)
#include <stdint.h>

#include "kv_common.h"
#include "qk_prep.h"
#include "vdn_common.h"

namespace vdn {
namespace {

// Threads of a workgroup: two consecutive tokens of one chunk each.
constexpr int threads_of(int d) { return 4 * d; }
// Workgroups of a launch at most; each takes further units in steps of the grid.
constexpr int64_t kMostGroups = 1 << 20;
// Waves from which on the part is full (16 a compute unit), and heads of a unit at most.
constexpr int64_t kFill = 4096;
constexpr int kMostHeads = 4;

struct KvAppendArgs {
    KvCacheArgs c;
    KvBatchArgs b;
    KvUnits units;
    uint32_t page_units;  // pages of all sequences that the call may touch, times the heads' shares
    int page_groups;      // workgroups that store pages; the others prepare queries
    int unit_heads;       // heads of a unit
    int query_parts;      // waves that share a token's queries: all of a workgroup's or 1
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

// Eight elements of a row, as they are stored and as binary32.
template <int DTYPE>
struct Chunk {
    static constexpr int kWords = DTYPE == VDN_FP8_DTYPE_F32 ? 2 : 1;
    uint4 v[kWords];
    __device__ __forceinline__ void load(const void* base, int64_t i)
    {
        const int size = DTYPE == VDN_FP8_DTYPE_F32 ? 4 : 2;
        const uint4* const p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + i * size);
#pragma unroll
        for (int j = 0; j < kWords; ++j) v[j] = load_once(p + j);
    }
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int j = 0; j < kWords; ++j) v[j] = make_uint4(0, 0, 0, 0);
    }
    // (what is unpacked from it before and after is unpacked twice, and not kept in registers in between)
    __device__ __forceinline__ void hide()
    {
#pragma unroll
        for (int j = 0; j < kWords; ++j) asm volatile("" : "+v"(v[j].x), "+v"(v[j].y), "+v"(v[j].z), "+v"(v[j].w));
    }
    __device__ __forceinline__ void get(float x[8]) const
    {
        const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[kWords - 1].x, v[kWords - 1].y, v[kWords - 1].z, v[kWords - 1].w};
        if (DTYPE == VDN_FP8_DTYPE_F32) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e]);
            return;
        }
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
};

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

// The rotation of one chunk of a token, as the bf16 that its cosines and sines are rounded to.
struct Rotation {
    uint32_t cs[4], sn[4];
    __device__ __forceinline__ void hide()
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(cs[j]), "+v"(sn[j]));
    }
    // (i0 < R: the chunk rotates; otherwise zeros that nothing uses)
    __device__ __forceinline__ void load(const KvAppendArgs& p, int64_t token, int i0)
    {
        if (i0 >= p.R) {
#pragma unroll
            for (int j = 0; j < 4; ++j) cs[j] = sn[j] = 0;
            return;
        }
        const int64_t at = token * p.ldcs + i0;
        if (p.cs_bf16) {
            const uint4 c = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.cos) + at);
            const uint4 s = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.sin) + at);
            cs[0] = c.x, cs[1] = c.y, cs[2] = c.z, cs[3] = c.w;
            sn[0] = s.x, sn[1] = s.y, sn[2] = s.z, sn[3] = s.w;
        } else {
            const float4* const c = reinterpret_cast<const float4*>(static_cast<const float*>(p.cos) + at);
            const float4* const s = reinterpret_cast<const float4*>(static_cast<const float*>(p.sin) + at);
            const float4 c0 = c[0], c1 = c[1], s0 = s[0], s1 = s[1];
            cs[0] = pack_bf16x2(c0.x, c0.y), cs[1] = pack_bf16x2(c0.z, c0.w), cs[2] = pack_bf16x2(c1.x, c1.y), cs[3] = pack_bf16x2(c1.z, c1.w);
            sn[0] = pack_bf16x2(s0.x, s0.y), sn[1] = pack_bf16x2(s0.z, s0.w), sn[2] = pack_bf16x2(s1.x, s1.y), sn[3] = pack_bf16x2(s1.z, s1.w);
        }
    }
};

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
    float n[8], cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) n[e] = (x[e] * rstd) * w[e];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        cs[2 * e] = bf16_lo(r.cs[e]), cs[2 * e + 1] = bf16_hi(r.cs[e]);
        sn[2 * e] = bf16_lo(r.sn[e]), sn[2 * e + 1] = bf16_hi(r.sn[e]);
    }
    rotate8<G>(n, cs, sn, p.R == D, rot, first, partner, lane, o);
}

// The queries of one token, or the part of them that is wave `part`'s of `parts`: every parts-th sweep of 64
// lanes over its heads, four sweeps' loads before their arithmetic.
template <int D>
__device__ __forceinline__ void prepare_query(const KvAppendArgs& p, int64_t token, int part, int parts)
{
    constexpr int G = D / 8, kSweeps = 4;
    const int lane = threadIdx.x & 63;
    const int i0 = 8 * (lane % G), chunks = p.q_heads * G, step = 64 * parts;
    float w[8];
    load_weight(p.weight_q, i0, w);
    Rotation r;
    r.load(p, token, i0);
    for (int base = part * 64; base < chunks; base += step * kSweeps) {
        Chunk<VDN_FP8_DTYPE_BF16> v[kSweeps];
#pragma unroll
        for (int s = 0; s < kSweeps; ++s) v[s].load(p.query, token * p.ldq + 8 * min(base + s * step + lane, chunks - 1));
#pragma unroll
        for (int s = 0; s < kSweeps; ++s) {
            const int q = base + s * step + lane;
            if (base + s * step >= chunks) break;   // (wave-uniform)
            float x[8], o[8];
            v[s].get(x);
            prepare8<D>(p, x, w, p.eps_q, r, lane, o);
            if (q < chunks)
                *reinterpret_cast<uint4*>(p.out + token * p.ldo + 8 * q) =
                    make_uint4(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7]));
        }
    }
}

// One page of p.unit_heads heads, one after the other: the rows of the next head are read while one is stored,
// and the tokens' rotations are kept.
template <int D, int DTYPE, bool PREP>
__device__ __forceinline__ void store_page(const KvAppendArgs& p, uint32_t unit, uint32_t* vt, float* part, uint32_t* top)
{
    constexpr int CH = D / 8;               // chunks of a row: one lane each
    constexpr int P = 2, kThreads = threads_of(D), kWaves = kThreads / 64;
    constexpr int kRow = 17;                // dwords of a v row in LDS (16 and one to spread the banks)
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t turns = (uint32_t)(p.c.heads + p.unit_heads - 1) / (uint32_t)p.unit_heads;
    const int h0 = (int)(unit % turns) * p.unit_heads, h_end = min(h0 + p.unit_heads, p.c.heads);
    uint32_t at;
    KvSequence s{};
    const int b = kv_locate(p.b, p.units, unit / turns, at, s);
    if (b == p.b.batch) return;   // behind the last sequence
    const int64_t w64 = max(s.first, (int64_t)0) / kPage + at;
    if (w64 * kPage >= s.length) return;
    const int w = (int)w64;
    const int lo = (int)max(s.first - w64 * kPage, (int64_t)0), hi = (int)min((int64_t)s.length - w64 * kPage, (int64_t)kPage);
    if (lo >= hi) return;
    const int64_t row0 = s.start + w64 * kPage - s.first;   // the call's row of the page's token 0 (may lie before the call)

    const int ch = tid % CH, i0 = 8 * ch, t0 = (tid / CH) * P;
    Chunk<DTYPE> kc[P], vc[P];
    auto read = [&](int h) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            // (rows that are not the call's are read as the nearest that is, and passed over)
            const int64_t row = row0 + min(max(t0 + i, lo), hi - 1);
            kc[i].load(p.key, row * p.ldk + h * D + i0);
            vc[i].load(p.value, row * p.ldv + h * D + i0);
        }
    };
    read(h0);
    const int page = kv_page(p.b, p.c, b, w);
    if (page < 0) return;
    Rotation rot[PREP ? P : 1];
    uint4 w4 = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);   // ones
    if (PREP) {
        if (p.weight_k) w4 = *reinterpret_cast<const uint4*>(p.weight_k + i0);
#pragma unroll
        for (int i = 0; i < P; ++i) rot[i].load(p, row0 + min(max(t0 + i, lo), hi - 1), i0);
    }
    for (int h = h0; h < h_end; ++h) {
        const int64_t ph = (int64_t)page * p.c.heads + h;
        const int own_k = p.c.k_scale[ph] - 127, own_v = p.c.v_scale[ph] - 127;
        // This head's rows as they are to be stored, still packed: prepared keys as bf16, zeros where the row
        // is not the call's.
        Chunk<DTYPE> ks[P], vs[P];
        uint32_t ak = 0, av = 0;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const bool on = t0 + i >= lo && t0 + i < hi;
            ks[i] = kc[i], vs[i] = vc[i];
            float x[8];
            if (PREP) {
                float o[8], w8[8];
                ks[i].get(x);
                asm volatile("" : "+v"(w4.x), "+v"(w4.y), "+v"(w4.z), "+v"(w4.w));
                w8[0] = bf16_lo(w4.x), w8[1] = bf16_hi(w4.x), w8[2] = bf16_lo(w4.y), w8[3] = bf16_hi(w4.y);
                w8[4] = bf16_lo(w4.z), w8[5] = bf16_hi(w4.z), w8[6] = bf16_lo(w4.w), w8[7] = bf16_hi(w4.w);
                rot[i].hide();   // (unpacked for each head, not once for all in twice the registers)
                prepare8<D>(p, x, w8, p.eps_k, rot[i], lane, o);
                ks[i].v[0] = make_uint4(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7]));
            }
            if (!on) ks[i].clear(), vs[i].clear();
            ks[i].get(x);
#pragma unroll
            for (int e = 0; e < 8; ++e) ak = max(ak, finite_magnitude(x[e]));
            vs[i].get(x);
#pragma unroll
            for (int e = 0; e < 8; ++e) av = max(av, finite_magnitude(x[e]));
        }
        if (h + 1 < h_end) read(h + 1);
#pragma unroll
        for (int i = 0; i < P; ++i) ks[i].hide(), vs[i].hide();
        ak = wave_max_u32(ak), av = wave_max_u32(av);
        if (lane == 0) top[wave] = ak, top[kWaves + wave] = av;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWaves; ++i) ak = max(ak, top[i]), av = max(av, top[kWaves + i]);
        int ek = scale_exponent(ak), ev = scale_exponent(av);
        const bool keeps = lo > 0;
        if (keeps) ek = max(ek, own_k), ev = max(ev, own_v);
        const int dk = own_k - ek, dv = own_v - ev;   // used where the page keeps tokens: <= 0
        const float fk = power_of_two(-min(ek, 126)), fv = power_of_two(-min(ev, 126));

        // v: the two tokens' codes of each element, to LDS
        {
            float x[P][8];
#pragma unroll
            for (int i = 0; i < P; ++i) vs[i].get(x[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                reinterpret_cast<uint16_t*>(vt + (i0 + e) * kRow)[t0 / 2] = (uint16_t)pack_e4m3x4(x[0][e] * fv, x[1][e] * fv, 0.0f, 0.0f);
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
                float x[8];
                ks[i].get(x);
                c8 = make_uint2(pack_e4m3x4(x[0] * fk, x[1] * fk, x[2] * fk, x[3] * fk), pack_e4m3x4(x[4] * fk, x[5] * fk, x[6] * fk, x[7] * fk));
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
                    for (int g = 0; g < kWaves; ++g) total += part[g * D + 2 * i + e];
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
            uint32_t* const dst = reinterpret_cast<uint32_t*>(p.c.v + (ph * D + d) * kPage) + 4 * c;
            const uint32_t* const src = vt + d * kRow + 4 * c;
            if (first >= lo && first + 16 <= hi) {
                *reinterpret_cast<uint4*>(dst) = make_uint4(src[0], src[1], src[2], src[3]);
                continue;
            }
#pragma unroll 1
            for (int j = 0; j < 4; ++j) {   // (at a page's first and last call)
                const uint32_t was = dst[j], kept = shift ? rescale4(was, dv) : was, now = src[j];
                uint32_t r = 0;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int token = first + 4 * j + t;
                    r |= (token < lo ? kept : token < hi ? now : was) & (0xffu << (8 * t));
                }
                dst[j] = r;
            }
        }
        if (tid == 0) {
            p.c.k_scale[ph] = (uint8_t)(ek + 127);
            p.c.v_scale[ph] = (uint8_t)(ev + 127);
        }
        __syncthreads();   // before the next values overwrite LDS
    }
}

template <int D, int DTYPE, bool PREP>
__global__ __launch_bounds__(threads_of(D), 4) void k_kv_append(KvAppendArgs p)
{
    __shared__ uint32_t vt[D * 17];
    __shared__ float part[threads_of(D) / 64 * D];
    __shared__ uint32_t top[2 * threads_of(D) / 64];
    if ((int)blockIdx.x < p.page_groups) {
        for (uint32_t u = blockIdx.x; u < p.page_units; u += p.page_groups) store_page<D, DTYPE, PREP>(p, u, vt, part, top);
    } else if (PREP) {
        const int64_t groups = gridDim.x - p.page_groups;
        const int each = (int)(blockDim.x >> 6) / p.query_parts, wave = threadIdx.x >> 6;   // tokens of a workgroup
        for (int64_t t = ((int64_t)blockIdx.x - p.page_groups) * each + wave / p.query_parts; t < p.b.tokens; t += groups * each)
            prepare_query<D>(p, t, wave % p.query_parts, p.query_parts);
    }
}

template <int DTYPE, bool PREP>
int launch(const KvAppendArgs& p, hipStream_t stream)
{
    const int threads = threads_of(p.c.d), waves = threads / 64;
    KvAppendArgs q = p;
    q.query_parts = p.b.tokens >= kFill / 2 ? 1 : waves;
    const int64_t tokens = PREP ? (p.b.tokens * q.query_parts + waves - 1) / waves : 0;
    const int64_t groups = p.page_groups + (tokens < kMostGroups ? tokens : kMostGroups);
    const dim3 grid((unsigned)groups), block(threads);
    switch (p.c.d) {
        case 64: hipLaunchKernelGGL((k_kv_append<64, DTYPE, PREP>), grid, block, 0, stream, q); break;
        case 128: hipLaunchKernelGGL((k_kv_append<128, DTYPE, PREP>), grid, block, 0, stream, q); break;
        default: hipLaunchKernelGGL((k_kv_append<256, DTYPE, PREP>), grid, block, 0, stream, q); break;
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
    // Heads of a unit: several where the pages alone fill the part, for the rotations that they share (and
    // the loads of the next that run beside the stores of one).
    const int64_t pages = kv_unit_count(p.b, p.units);
    p.unit_heads = 1;
    while (p.unit_heads < kMostHeads && pages * p.c.heads / (2 * p.unit_heads) * (threads_of(p.c.d) / 64) >= kFill) p.unit_heads *= 2;
    const int64_t units = pages * ((p.c.heads + p.unit_heads - 1) / p.unit_heads);
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
