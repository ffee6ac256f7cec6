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
constexpr int kFewRows = 32;               // packed query rows of a sequence that attend_few_kernel takes beside attend_many_kernel

// Two int8 codes in bytes 0 and 2 of w (bytes 1 and 3: anything) -> fp16 pair,
// exactly: the bits 0x6400 | (code + 128) are the fp16 number 1024 + code + 128.
__device__ __forceinline__ uint32_t codes_to_f16x2(uint32_t w)
{
    const uint32_t m = (w & 0x00FF00FFu) ^ 0x64806480u;
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&m), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&d);
}

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

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}

// 2^x (one MUFU instruction; results below 2^-126 are 0).
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ------------------------------------------------------------------ the batch

// A sequence as the kernels see it, every value held within the tensors.
struct Seq {
    int q0, n;       // first query token and their number
    int len;         // tokens in the cache
};

__device__ __forceinline__ Seq load_seq(const CacheView& c, int s)
{
    Seq r;
    const int64_t a = min(static_cast<int64_t>(max(c.cu[s], 0)), c.tokens);
    const int64_t b = min(static_cast<int64_t>(max(c.cu[s + 1], 0)), c.tokens);
    r.q0 = static_cast<int>(a);
    r.n = static_cast<int>(max(b - a, static_cast<int64_t>(0)));
    r.len = static_cast<int>(min(static_cast<int64_t>(max(c.kv_lens[s], 0)),
                                 static_cast<int64_t>(c.table_cols) << c.page_log2));
    return r;
}

struct Partial {        // one per CTA and slot, in the workspace
    long long seg;
    int seq, head, tile, pad;
};

// Output row `row` of a sequence's packed rows for one kv head.
__device__ __forceinline__ uint16_t* out_row(const AttentionParams& p, const Seq& s, int head, int row)
{
    const int tok = row / p.group, g = row - tok * p.group;
    return p.out + static_cast<int64_t>(s.q0 + tok) * p.ldo + static_cast<int64_t>(head * p.group + g) * p.c.D;
}

// 1 / l; 0 for a row that saw no token, NaN for a NaN.
__device__ __forceinline__ float inv_sum(float l) { return l > 0.0f ? __fdiv_rn(1.0f, l) : (l == 0.0f ? 0.0f : l); }

size_t attend_many_ws_bytes(int D, int sms);
cudaError_t launch_attend_many(const AttentionParams& p, int sms, cudaStream_t stream);

}  // namespace w4a8
