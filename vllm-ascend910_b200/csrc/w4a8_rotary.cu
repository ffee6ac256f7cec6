// w4a8_rotary.cu -- rotary positions with several axes, on q and k alone.
//
//   a' = a c - b s      b' = b c + a s      (fp32, products rounded first, one rounding to bf16)
//
// for each pair (a, b) of a head's first `rot` elements, with the cosine and sine that the
// caller's table holds for the pair in the row of the token's position on the pair's axis
// (time, height, width of an image's or video's patches; one axis: ordinary positions).
//
// A block takes a few tokens.  It finds their cosines and sines first, pair by pair, in shared memory; a
// thread then stays with 16 elements of a head (two vectors of 8 pairs' halves) and one token, keeps their
// angles in registers and turns every (threads / (items x tokens))-th head with them, with several heads' loads in
// flight.  Elements past `rot` are copied, or left alone in place.
//
// Many tokens: memory bounds it (8,191 tokens of 40 + 8 heads of 128 36.0 us, 5.6 TB/s).  Fewer: the chain of position, table
// row, rotation and store (one token 1.9 us; 5,041 of 16 + 16 heads of 80 13.5, a wave of 1,184 blocks and the rest of a second).
#include <algorithm>

#include "w4a8_rotary.cuh"

namespace w4a8 {

namespace {

constexpr int kThreads = 128;
constexpr int kAhead = 2;
constexpr int kManyTokens = 592;

// LOG2 > 0: 2^LOG2 tokens and all their heads; 0: one token and `heads_each` heads of q or, in a token's later blocks, of k.
// (The number is a constant and shared memory sized by it: 8,191 tokens of 40 + 8 heads 36.0 us, 36.9 with room for 16.)
template <bool INTERLEAVED, int LOG2>
__global__ void __launch_bounds__(kThreads, 8) rotary_kernel(const RotaryParams p, const int items, const int heads_each)
{
    constexpr bool MANY = LOG2 > 0;
    constexpr int toks = 1 << LOG2;
    __shared__ __align__(16) float angles[toks][kMaxRotaryDim];
    pdl_wait();
    const int tid = threadIdx.x, half = p.rot / 2;
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) << LOG2;
    const int step = (kThreads / items) >> LOG2, slot = tid / items, j = tid - slot * items;
    const int k_tok = slot & (toks - 1), first = slot >> LOG2;
    const int64_t t = t0 + k_tok;
    const bool on = first < step && t < p.tokens;             // (not the threads past the last whole set)

    const bool turn = j < p.rot / 16;
    int c0, c1;
    if (turn) {
        item_cols(j, p.rot, INTERLEAVED, c0, c1);
    } else {
        c0 = p.rot + 16 * (j - p.rot / 16);
        c1 = c0 + 8 < p.D ? c0 + 8 : c0;                     // (the last vector of D = 8 mod 16 twice)
    }
    const int q_parts = MANY ? 0 : (p.heads[0] + heads_each - 1) / heads_each;
    const int w0 = !MANY && static_cast<int>(blockIdx.y) >= q_parts;
    const int h0 = MANY ? first : (static_cast<int>(blockIdx.y) - (w0 ? q_parts : 0)) * heads_each + first;
    const int end0 = !on ? 0 : MANY ? p.heads[0] : min(h0 - first + heads_each, p.heads[w0]);
    uint4 v[kAhead][2];
    const auto load = [&](const uint16_t* src, int h, int end) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k, h += step)
            if (h < end) {
                const uint16_t* at = src + static_cast<int64_t>(h) * p.D;
                v[k][0] = *reinterpret_cast<const uint4*>(at + c0);
                v[k][1] = *reinterpret_cast<const uint4*>(at + c1);
            }
    };
    load(p.x[w0] + t * p.ld[w0], h0, end0);
    for (int i = tid; i < half << LOG2; i += kThreads) {
        const int k = i / half, pair = i - k * half, a = static_cast<int>(p.axes.map[pair >> 5] >> (2 * (pair & 31))) & 3;
        const int64_t at = min(t0 + k, p.tokens - 1);
        const float* row = p.cos_sin + clamp_row(p.axes.positions[a * p.axes.ld + at], p.table_rows) * p.rot;
        angles[k][pair] = row[pair];
        angles[k][half + pair] = row[half + pair];
    }
    __syncthreads();
    if (!on) return;
    float4 cs[4] = {};
    if (turn) load_angles(angles[k_tok], j, p.rot, cs);
#pragma unroll 1
    for (int w = w0; w < (MANY ? 2 : w0 + 1); ++w) {
        const int end = w == w0 ? end0 : p.heads[1];
        const uint16_t* src = p.x[w] + t * p.ld[w];
        uint16_t* dst = p.out[w] + t * p.ldo[w];
        if (!turn && src == dst) continue;
        if (w != w0) load(src, h0, end);
        for (int h = h0; h < end; h += kAhead * step) {
#pragma unroll
            for (int k = 0, g = h; k < kAhead; ++k, g += step)
                if (g < end) {
                    if (turn) turn_item(INTERLEAVED, cs, v[k][0], v[k][1]);
                    uint16_t* at = dst + static_cast<int64_t>(g) * p.D;
                    *reinterpret_cast<uint4*>(at + c0) = v[k][0];
                    *reinterpret_cast<uint4*>(at + c1) = v[k][1];
                }
            load(src, h + kAhead * step, end);
        }
    }
}

template <int LOG2>
cudaError_t launch(const RotaryParams& p, int items, int heads_each, int parts, cudaStream_t stream)
{
    const int64_t blocks = (p.tokens + (1 << LOG2) - 1) >> LOG2;
    if (blocks > 0x7FFFFFFF || parts > 65535) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(parts));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return p.interleaved ? cudaLaunchKernelEx(&cfg, rotary_kernel<true, LOG2>, p, items, heads_each)
                         : cudaLaunchKernelEx(&cfg, rotary_kernel<false, LOG2>, p, items, heads_each);
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams& p, cudaStream_t stream)
{
    const int items = p.rot / 16 + (p.D - p.rot + 15) / 16, slots = kThreads / items;
    // Few tokens: one a block, its heads spread over blocks.  (40 + 8 heads of 128, one and four tokens a
    // block: 256 tokens 3.5 and 5.6 us, 512 5.6 and 5.7, 1,024 9.5 and 6.8.)
    if (p.tokens < kManyTokens)
        return launch<0>(p, items, slots, (p.heads[0] + slots - 1) / slots + (p.heads[1] + slots - 1) / slots, stream);
    // Many: four a block with all their heads, and more where a block has threads for more heads than there are (62,909
    // tokens of 1 + 1 heads of 96: 44 us by four, 21 by sixteen).
    const int heads = std::max(p.heads[0], p.heads[1]);
    if ((slots >> 3) > heads) return launch<4>(p, items, 0, 1, stream);
    if ((slots >> 2) > heads) return launch<3>(p, items, 0, 1, stream);
    return launch<2>(p, items, 0, 1, stream);
}

}  // namespace w4a8
