// w4a8_rotary.cuh -- turning the pairs of a head's row, shared by the cache write
// (w4a8_kvcache.cu) and the rotation alone (w4a8_rotary.cu).
#pragma once

#include "w4a8_common.cuh"
#include "w4a8_kernels.h"

namespace w4a8 {

__device__ __forceinline__ void rotate_pair(float& a, float& b, float c, float s)
{
    const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    a = x;
}

// A work item of a head's row: two vectors of 8 elements.  Items [0, rot / 16)
// are rotated -- half layout: elements [8j, 8j + 8) and the same past rot / 2;
// interleaved: elements [16j, 16j + 16) -- the rest are 16 plain elements.
__device__ __forceinline__ void item_cols(int j, int rot, int interleaved, int& c0, int& c1)
{
    if (j < rot / 16 && !interleaved) {
        c0 = 8 * j;
        c1 = rot / 2 + 8 * j;
    } else {
        c0 = 16 * j;
        c1 = 16 * j + 8;
    }
}

// Cosines and sines of item j's 8 pairs, from a table row.
__device__ __forceinline__ void load_angles(const float* row, int j, int rot, float4 (&cs)[4])
{
    const float4* cp = reinterpret_cast<const float4*>(row + 8 * j);
    const float4* sp = reinterpret_cast<const float4*>(row + rot / 2 + 8 * j);
    cs[0] = cp[0];
    cs[1] = cp[1];
    cs[2] = sp[0];
    cs[3] = sp[1];
}

__device__ __forceinline__ void rotate_item(int interleaved, const float4 (&cs)[4], float (&a)[8], float (&b)[8])
{
    const float c[8] = {cs[0].x, cs[0].y, cs[0].z, cs[0].w, cs[1].x, cs[1].y, cs[1].z, cs[1].w};
    const float s[8] = {cs[2].x, cs[2].y, cs[2].z, cs[2].w, cs[3].x, cs[3].y, cs[3].z, cs[3].w};
    if (!interleaved) {
#pragma unroll
        for (int i = 0; i < 8; ++i) rotate_pair(a[i], b[i], c[i], s[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) rotate_pair(a[2 * i], a[2 * i + 1], c[i], s[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) rotate_pair(b[2 * i], b[2 * i + 1], c[4 + i], s[4 + i]);
    }
}

__device__ __forceinline__ uint4 pack8(const float (&v)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ int64_t clamp_row(int64_t pos, int64_t rows)
{
    return pos < 0 ? 0 : (pos >= rows ? rows - 1 : pos);
}


// rotate_item on the 16 elements as they are stored, two products an instruction.  The sums stay single
// ones: a packed sum of packed products may become a fused one, which rounds once.
__device__ __forceinline__ void turn_item(int interleaved, const float4 (&cs)[4], uint4& v0, uint4& v1)
{
    const uint64_t c[4] = {pair2(cs[0].x, cs[0].y), pair2(cs[0].z, cs[0].w), pair2(cs[1].x, cs[1].y), pair2(cs[1].z, cs[1].w)};
    const uint64_t s[4] = {pair2(cs[2].x, cs[2].y), pair2(cs[2].z, cs[2].w), pair2(cs[3].x, cs[3].y), pair2(cs[3].z, cs[3].w)};
    uint32_t* w[2] = {&v0.x, &v1.x};
    const auto low = [](uint32_t x) { return __uint_as_float(x << 16); };
    const auto high = [](uint32_t x) { return __uint_as_float(x & 0xFFFF0000u); };
    const auto pack = [](float lo, float hi) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&b);
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // pairs 2 i and 2 i + 1: a word of either half, or two words next to each other
        uint32_t &x = interleaved ? w[i >> 1][(2 * i) & 3] : w[0][i], &y = interleaved ? w[i >> 1][(2 * i + 1) & 3] : w[1][i];
        const uint64_t a = interleaved ? pair2(low(x), low(y)) : pair2(low(x), high(x));
        const uint64_t b = interleaved ? pair2(high(x), high(y)) : pair2(low(y), high(y));
        float ac0, ac1, bs0, bs1, bc0, bc1, as0, as1;
        unpair2(f2_mul(a, c[i]), ac0, ac1);
        unpair2(f2_mul(b, s[i]), bs0, bs1);
        unpair2(f2_mul(b, c[i]), bc0, bc1);
        unpair2(f2_mul(a, s[i]), as0, as1);
        const float a0 = __fsub_rn(ac0, bs0), a1 = __fsub_rn(ac1, bs1), b0 = __fadd_rn(bc0, as0), b1 = __fadd_rn(bc1, as1);
        x = interleaved ? pack(a0, b0) : pack(a0, a1);
        y = interleaved ? pack(a1, b1) : pack(b0, b1);
    }
}

// Rows of the table that a token's axes point at.
struct AxisRows {
    int32_t at[kMaxAxes];
};

__device__ __forceinline__ AxisRows axis_rows(const AxesView& v, int64_t t, int64_t rows)
{
    AxisRows r;
#pragma unroll
    for (int a = 0; a < kMaxAxes; ++a) r.at[a] = a < v.axes ? static_cast<int32_t>(clamp_row(v.positions[a * v.ld + t], rows)) : 0;
    return r;
}

// load_angles where each pair has its own axis: one row's vectors where item j's 8 pairs
// share an axis, else those of every axis, pair by pair the right one kept.
__device__ __forceinline__ void load_angles_axes(const float* table, const AxesView& v, const AxisRows& r, int j, int rot,
                                                 float4 (&cs)[4])
{
    const uint32_t bits = static_cast<uint32_t>(v.map[j >> 2] >> (16 * (j & 3))) & 0xFFFFu;
    const int first = bits & 3;
    int32_t row = r.at[0];
#pragma unroll
    for (int a = 1; a < kMaxAxes; ++a) row = first == a ? r.at[a] : row;
    load_angles(table + static_cast<int64_t>(row) * rot, j, rot, cs);
    if (bits == first * 0x5555u) return;
#pragma unroll
    for (int a = 0; a < kMaxAxes; ++a) {
        // the pairs of axis a, a bit each at the even places; the first pair's axis is there already
        const uint32_t x = bits ^ (a * 0x5555u), mine = ~(x | (x >> 1)) & 0x5555u;
        if (a == first || mine == 0) continue;
        float4 o[4];
        load_angles(table + static_cast<int64_t>(r.at[a]) * rot, j, rot, o);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float4 &c = cs[i], &s = cs[2 + i];
            const uint32_t m = mine >> (8 * i);
            if (m & 1u) c.x = o[i].x, s.x = o[2 + i].x;
            if (m & 4u) c.y = o[i].y, s.y = o[2 + i].y;
            if (m & 16u) c.z = o[i].z, s.z = o[2 + i].z;
            if (m & 64u) c.w = o[i].w, s.w = o[2 + i].w;
        }
    }
}

}  // namespace w4a8
