// w4a8_attention.cuh -- what the two attention kernels share: exact conversion of
// cache codes, the powers of two that keep fp16 operands in range, the batch's
// bounds, and the record of a segment's part in the workspace.
#pragma once

#include <cuda_fp16.h>

#include "w4a8_common.cuh"
#include "w4a8_kernels.h"

namespace w4a8 {

constexpr int kMaxBatch = 2048;            // W4A8_ATTENTION_MAX_BATCH
constexpr float kNegInf = -INFINITY;
// Sequences of more packed query rows go to attend_many_kernel.  At 25 rows (5 tokens of
// 5 heads) 64 sequences of 1,000 take 86 us here and 98 there, but 8 of 4,000 take 46 and
// 41; at 40 rows 120 and 100, 61 and 42.
constexpr int kFewRows = 32;

__device__ __forceinline__ uint4 lds128(uint32_t a)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
// Two int8 codes in bytes 0 and 2 of w (bytes 1 and 3: anything) -> fp16 pair,
// exactly: the bits 0x6400 | (code + 128) are the fp16 number 1024 + code + 128.
__device__ __forceinline__ uint32_t codes_to_f16x2(uint32_t w)
{
    const uint32_t m = (w & 0x00FF00FFu) ^ 0x64806480u;
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&m), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&d);
}

// The same from codes already biased (code ^ 0x80): bytes 0 and 1, or 2 and 3, of w.
__device__ __forceinline__ uint32_t biased_f16x2(uint32_t m)
{
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&m), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ uint32_t biased_lo(uint32_t w) { return biased_f16x2(__byte_perm(w, 0x64646464u, 0x4140)); }
__device__ __forceinline__ uint32_t biased_hi(uint32_t w) { return biased_f16x2(__byte_perm(w, 0x64646464u, 0x4342)); }

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi)
{
    const __half2 b = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}

// 2^-e for a row whose largest magnitude is m, m * 2^-e in [2^13, 2^14); 1 for a
// zero or non-finite m.  e is held within what fp32 can scale by.
__device__ __forceinline__ float row_shrink(float m)
{
    if (!(m > 0.0f) || m == INFINITY) return 1.0f;
    const int e = static_cast<int>((__float_as_uint(m) >> 23) & 0xFFu) - 127 - 13;
    return __uint_as_float(static_cast<uint32_t>(127 - min(max(e, -126), 126)) << 23);
}

// The smallest power of two at or above a positive finite v (at least 2^-100);
// 1 for a non-finite v.
__device__ __forceinline__ float pow2_above(float v)
{
    if (!(v < INFINITY)) return 1.0f;
    const uint32_t b = __float_as_uint(fmaxf(v, 7.888609052210118e-31f));
    return __uint_as_float((b & 0x7F800000u) + ((b & 0x007FFFFFu) ? 0x00800000u : 0u));
}
constexpr float kVrMin = 7.888609052210118e-31f;   // 2^-100
constexpr float kWeightOne = 16384.0f;             // 2^14
constexpr float kSlack = 1.9f;                     // log2 by which scores may exceed the reference maximum: weights stay below 2^15.9

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}

// What is added to a row's scaled scores: minus its reference maximum.  Before the
// first score it is so large that any finite score exceeds the slack.
__device__ __forceinline__ float first_reference(float m) { return m == kNegInf ? 1e38f : -m; }

// 2^x (one MUFU instruction; results below 2^-126 are 0).
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ------------------------------------------------------------------ the batch

// A sequence as the kernels see it, every value but `pos` held within the tensors.
struct Seq {
    int q0, n;       // first query token and their number
    int len;         // tokens that the page table has columns for
    int pos;         // the first query token's position (the sequence may be longer than the table)
};

__device__ __forceinline__ Seq load_seq(const CacheView& c, int s)
{
    Seq r;
    const int64_t a = min(static_cast<int64_t>(max(c.cu[s], 0)), c.tokens);
    const int64_t b = min(static_cast<int64_t>(max(c.cu[s + 1], 0)), c.tokens);
    r.q0 = static_cast<int>(a);
    r.n = static_cast<int>(max(b - a, static_cast<int64_t>(0)));
    const int whole = max(c.kv_lens[s], 0);
    r.len = min(whole, c.table_cols << c.page_log2);        // (the product fits: checked on the host)
    r.pos = whole - r.n;
    return r;
}

// One per CTA and slot, in the workspace: which segment the part belongs to, and
// where its rows go.
struct Partial {
    long long seg;      // -1: none
    int q0, rows;       // the sequence's first query token, its packed rows
    int head, row0;     // kv head, the segment's first packed row
};

// Adds one segment's n parts for NV times 4 elements of one row: parts are the
// leader's slot 1 and slot 0 of the CTAs behind it.  Loads of NB parts (maximum, sum,
// values) are in flight together.
template <int NB, int NV, class M, class V>
__device__ __forceinline__ void join_parts(int n, const M& ml, const V& value, float4 (&o)[NV])
{
    float mx = kNegInf, ls = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) o[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int base = 0; base < n; base += NB) {
        float m[NB], l[NB];
        float4 x[NB][NV];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            m[i] = kNegInf;
            l[i] = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v) x[i][v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (base + i < n) {
                const float2 t = ml(base + i);
                m[i] = t.x;
                l[i] = t.y;
#pragma unroll
                for (int v = 0; v < NV; ++v) x[i][v] = value(base + i, v);
            }
        }
        float mn = mx;
#pragma unroll
        for (int i = 0; i < NB; ++i) mn = fmaxf(mn, m[i]);
        const float keep = mx == kNegInf ? (mn == kNegInf ? 1.0f : 0.0f) : exp2f(mx - mn);
        ls *= keep;
#pragma unroll
        for (int v = 0; v < NV; ++v) o[v] = make_float4(o[v].x * keep, o[v].y * keep, o[v].z * keep, o[v].w * keep);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if (base + i >= n) break;
            // (a part without a visible token has m = -inf, l = 0 and zeros)
            const float a = m[i] == kNegInf ? 1.0f : exp2f(m[i] - mn);
            ls += a * l[i];
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                o[v].x += a * x[i][v].x;
                o[v].y += a * x[i][v].y;
                o[v].z += a * x[i][v].z;
                o[v].w += a * x[i][v].w;
            }
        }
        mx = mn;
    }
    const float inv = ls > 0.0f ? __fdiv_rn(1.0f, ls) : (ls == 0.0f ? 0.0f : ls);
#pragma unroll
    for (int v = 0; v < NV; ++v) o[v] = make_float4(o[v].x * inv, o[v].y * inv, o[v].z * inv, o[v].w * inv);
}

// row / group: the query token of a packed row.  With M = floor(2^64 / g) + 1 the
// high word of row * M is the quotient for every 32-bit row (row * (M g - 2^64)
// stays below 2^64).
__device__ __forceinline__ int row_token(const AttentionParams& p, int row)
{
    return p.group_magic == 0 ? row : static_cast<int>(__umul64hi(static_cast<uint64_t>(static_cast<uint32_t>(row)), p.group_magic));
}

// Output row `row` of the packed rows, for one kv head, of the sequence whose first
// query token is q0.
__device__ __forceinline__ uint16_t* out_row(const AttentionParams& p, int q0, int head, int row)
{
    const int tok = row_token(p, row), g = row - tok * p.group;
    return p.out + static_cast<int64_t>(q0 + tok) * p.ldo + static_cast<int64_t>(head * p.group + g) * p.c.D;
}

// The segment that begins in CTA `lead` and goes on: its record and number of
// parts (0: there is none).  A whole block calls it.
__device__ __forceinline__ int find_parts(const Partial* info, int lead, int nctas, Partial& rec)
{
    int n = 0;
    for (int base = lead + 1; base <= nctas; base += blockDim.x) {
        const int k = base + threadIdx.x;
        const long long seg = k < nctas ? info[2 * k].seg : -1;
        rec = info[2 * lead + 1];
        const int more = __syncthreads_count(seg >= 0 && seg == rec.seg);
        if (rec.seg < 0) return 0;
        n += more;
        if (more < static_cast<int>(blockDim.x)) break;
    }
    return n + 1;
}

// The least units of a share.  A segment cut in n parts costs n reads in its join, one
// CTA's; a worker's share costs its units: with `total` units of `segments` segments and
// `workers` workers to a part, share * 1 + (total / (segments * workers * share)) * ratio
// is least here, ratio being a part's cost in units.
__device__ __forceinline__ int least_share(long long total, int segments, int workers, float ratio)
{
    return max(1, static_cast<int>(sqrtf(ratio * static_cast<float>(total) / (static_cast<float>(segments) * workers)) + 0.5f));
}

// 1 / l; 0 for a row that saw no token, NaN for a NaN.
__device__ __forceinline__ float inv_sum(float l) { return l > 0.0f ? __fdiv_rn(1.0f, l) : (l == 0.0f ? 0.0f : l); }

size_t attend_many_ws_bytes(int D, int sms);
// Sequences of more than `least` packed rows.
cudaError_t launch_attend_many(const AttentionParams& p, int least, int sms, cudaStream_t stream);

}  // namespace w4a8
