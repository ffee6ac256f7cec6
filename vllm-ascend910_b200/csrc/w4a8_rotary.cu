// w4a8_rotary.cu -- rotary positions with several axes, on q and k alone.
//
//   a' = a c - b s      b' = b c + a s      (fp32, products rounded first, one rounding to bf16)
//
// for each pair (a, b) of a head's first `rot` elements, with the cosine and sine that the
// caller's table holds for the pair in the row of the token's position on the pair's axis
// (time, height, width of an image's or video's patches; one axis: ordinary positions).
//
// A thread owns 16 elements of a head (two vectors of 8 pairs' halves) for one token, so it reads
// the token's positions and its pairs' angles once and turns its part of every
// (threads / (items x tokens))-th head with them, four heads' loads in flight.  Elements past `rot`
// are copied, or left alone in place.
#include <algorithm>

#include "w4a8_rotary.cuh"

namespace w4a8 {

namespace {

constexpr int kThreads = 256;

__global__ void __launch_bounds__(kThreads, 4) rotary_kernel(const RotaryParams p, const int items, const int toks)
{
    pdl_wait();
    const int slot = threadIdx.x / items, j = threadIdx.x - slot * items, slots = kThreads / items;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * toks + slot % toks;
    const int step = slots / toks, h_first = slot / toks;
    if (t >= p.tokens || h_first >= step) return;             // (threads past the last whole set of slots)
    const bool turn = j < p.rot / 16;
    int c0, c1;
    if (turn) {
        item_cols(j, p.rot, p.interleaved, c0, c1);
    } else {
        c0 = p.rot + 16 * (j - p.rot / 16);
        c1 = c0 + 8 < p.D ? c0 + 8 : c0;                     // (the last vector of D = 8 mod 16 twice)
    }
    float4 cs[4] = {};
    constexpr int AHEAD = 4;
    bool have = false;
#pragma unroll 1
    for (int w = 0; w < 2; ++w) {
        if (!p.x[w] || (!turn && p.x[w] == p.out[w] && p.ld[w] == p.ldo[w])) continue;
        const uint16_t* src = p.x[w] + t * p.ld[w];
        uint16_t* dst = p.out[w] + t * p.ldo[w];
        for (int h0 = h_first; h0 < p.heads[w]; h0 += AHEAD * step) {
            uint4 v[AHEAD][2];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int64_t h = min(h0 + k * step, p.heads[w] - 1);
                v[k][0] = *reinterpret_cast<const uint4*>(src + h * p.D + c0);
                v[k][1] = *reinterpret_cast<const uint4*>(src + h * p.D + c1);
            }
            if (turn && !have) {
                load_angles_axes(p.cos_sin, p.axes, axis_rows(p.axes, t, p.table_rows), j, p.rot, cs);
                have = true;
            }
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int64_t h = h0 + k * step;
                if (h >= p.heads[w]) break;
                if (turn) {
                    float a[8], b[8];
                    unpack8_bf16(v[k][0], a);
                    unpack8_bf16(v[k][1], b);
                    rotate_item(p.interleaved, cs, a, b);
                    v[k][0] = pack8(a);
                    v[k][1] = pack8(b);
                }
                *reinterpret_cast<uint4*>(dst + h * p.D + c0) = v[k][0];
                *reinterpret_cast<uint4*>(dst + h * p.D + c1) = v[k][1];
            }
        }
    }
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams& p, cudaStream_t stream)
{
    const int items = p.rot / 16 + (p.D - p.rot + 15) / 16, slots = kThreads / items;
    const int toks = p.tokens < 592 ? 1 : std::min(4, slots);
    const int64_t blocks = (p.tokens + toks - 1) / toks;
    if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, rotary_kernel, p, items, toks);
}

}  // namespace w4a8
