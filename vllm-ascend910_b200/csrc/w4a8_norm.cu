// w4a8_norm.cu -- residual addition and root-mean-square norm of bf16 rows,
// with a bf16 or an 8-bit output.
//
//   h = x + r                       (fp32; r' = bf16(h) is the residual stream's new value)
//   n = 1 / sqrt(sum(h^2) / K + eps)
//   y = (h * n) * w
//
//   kNormBf16    y rounded once to bf16
//   kNormCodes   int8 codes [M, K] and scales [G, M], the activation quantiser's
//                rule (w4a8_common.cuh) applied to the fp32 y: one rounding
//                where norm, store and quantise would make two.  A group's maximum
//                is that of |h w|, times n, two fp32 roundings from max|y|: of bf16
//                scales of random rows one in 100,000 is the next one for it
//   kNormTiles   the same codes and scales in the GEMM's operand order, straight
//                into a linear call's workspace (QuantParams' kOutKernel form)
//
// A block holds one row in registers: a thread owns VPT vectors of 8 consecutive
// elements (16-byte loads), so x and r are read once and y, r' are written once.
// (At 64 registers a thread the compiler spills some: up to 56 bytes with two vectors,
// 208 to 560 with four, which rows wider than 8,192 take, and whose weight is read for every row.)
// Blocks stay for several rows when there are many: the weight is read once, and
// the next row's loads are on their way while this one is reduced.  The sum of
// squares takes one warp reduction and one barrier; the fp32 parts are added in a
// fixed order, so repeated calls give the same bits.  A group's amax stays within
// GK / 8 neighbouring vectors: a warp's shuffles, and shared memory for groups of 1024.
// fp32 arithmetic runs in pairs, two elements an instruction; each rounds alone.
//
// Measured (B200, rows of 5120 with a residual): 4096 rows, bf16 out 27.5 us, 6.1 TB/s, 93 %
// of a plain copy's rate; 8191 rows with codes 63 and 64 us in groups of 128 and 1024, 4.6 TB/s:
// about 570 instructions for a thread's 16 elements bound it, not the memory (before the
// pairs, the bodies without bounds tests and groups by vector order 75 and 96 us).  One
// row: 1.9 us, launch and two load latencies.  Rows of 27,648, whose spills and weights pass
// through L1: 2,048 of them 105 us, 4.3 TB/s, and 147 with codes, 2.7 TB/s.
#include <algorithm>

#include "w4a8_common.cuh"
#include "w4a8_kernels.h"

namespace w4a8 {

namespace {

constexpr int kMaxNormThreads = 1024;
// Rows past which a block takes two vectors a thread, bf16 / codes of rows of 5120: 64 rows
// 2.3 / 2.8 us with one, 2.3 / 3.6 with two; 592 rows 4.8 / 6.9 and 4.3 / 6.9; 4,096 rows 33 / 37 and
// 27 / 33.
constexpr int kManyRows = 296;
constexpr int kResident = 1024;            // threads per SM that the kernels' 64 registers allow

// 8 bf16 elements from position pos < K of a row (zeros past K), as they are.  WHOLE:
// rows are 16-byte aligned and K is a multiple of 8.
template <bool WHOLE>
__device__ __forceinline__ uint4 load_row8(const uint16_t* row, int pos, int K, bool vec)
{
    if (WHOLE || (vec && pos + 8 <= K)) return *reinterpret_cast<const uint4*>(row + pos);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = pos + 2 * i < K ? row[pos + 2 * i] : 0u, hi = pos + 2 * i + 1 < K ? row[pos + 2 * i + 1] : 0u;
        w[i] = lo | (hi << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Four pairs of fp32 values from 8 bf16 ones, and back.
__device__ __forceinline__ void unpack_pairs(uint4 v, uint64_t (&x)[4])
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = pair2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
}
__device__ __forceinline__ void unpair8(const uint64_t (&x)[4], float (&v)[8])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) unpair2(x[i], v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ uint4 pack8_bf16(const float (&v)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool WHOLE>
__device__ __forceinline__ void store_row8(uint16_t* row, int pos, int K, bool vec, const uint64_t (&h)[4])
{
    float v[8];
    unpair8(h, v);
    if (WHOLE || (vec && pos + 8 <= K)) {
        *reinterpret_cast<uint4*>(row + pos) = pack8_bf16(v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (pos + i < K) row[pos + i] = f32_to_bf16_bits(v[i]);
    }
}

// The weight's 8 elements from position pos.
__device__ __forceinline__ void load_weight8(const NormParams& p, int pos, uint64_t (&w)[4])
{
    if (p.weight_f32) {
        const float* wf = static_cast<const float*>(p.weight);
#pragma unroll
        for (int i = 0; i < 8; i += 2) w[i / 2] = pair2(pos + i < p.K ? wf[pos + i] : 0.0f, pos + i + 1 < p.K ? wf[pos + i + 1] : 0.0f);
    } else {
        unpack_pairs(load_row8<false>(static_cast<const uint16_t*>(p.weight), pos, p.K, p.vec_w), w);
    }
}

// The largest |h w| 2^-128 of 8 elements, as bits with the sign set.
__device__ __forceinline__ uint32_t far_max(const uint64_t (&h)[4], const uint64_t (&w)[4])
{
    const uint64_t down = pair2(0x1p-64f, 0x1p-64f);
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float lo, hi;
        unpair2(f2_mul(f2_mul(h[i], down), f2_mul(w[i], down)), lo, hi);
        a = max_abs_nan(a, lo, hi);
    }
    return __float_as_uint(a) | 0x80000000u;
}

template <int OUT, int VPT, bool WHOLE>
__global__ void __launch_bounds__(VPT == 2 ? 512 : kMaxNormThreads, VPT == 2 ? 2 : 1) rms_norm_kernel(const NormParams p)
{
    __shared__ float red[2][kMaxNormThreads / 32];
    __shared__ __align__(16) uint32_t red_max[2][VPT * kMaxNormThreads / 32];

    // the next kernel may come early where this one leaves room for it
    if (gridDim.x <= 148) pdl_launch_dependents();
    const int tid = threadIdx.x, T = blockDim.x, nw = T >> 5;
    pdl_wait();

    uint4 xn[VPT], rn[VPT];                        // a row's elements, loaded one row ahead
    auto load = [&](int row) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int pos = (j * T + tid) * 8;
            xn[j] = make_uint4(0, 0, 0, 0);
            rn[j] = xn[j];
            if (row < p.M && pos < p.K) {          // (the tile form has rows past M: zeros)
                xn[j] = load_row8<WHOLE>(p.x + static_cast<int64_t>(row) * p.ldx, pos, p.K, p.vec_x);
                if (p.res) rn[j] = load_row8<WHOLE>(p.res + static_cast<int64_t>(row) * p.ldr, pos, p.K, p.vec_r);
            }
        }
    };
    load(blockIdx.x);
    constexpr bool kKeep = VPT <= 2;               // the weight stays in registers
    uint64_t w[kKeep ? VPT : 1][4];
    if (kKeep)
#pragma unroll
        for (int j = 0; j < VPT; ++j) load_weight8(p, (j * T + tid) * 8, w[kKeep ? j : 0]);

    // (the last group's warps may be fewer than four)
    if (OUT != kNormBf16 && p.gk == 1024 && tid < 4 && VPT * nw + tid < VPT * kMaxNormThreads / 32)
        red_max[0][VPT * nw + tid] = red_max[1][VPT * nw + tid] = 0;

    // a vector that begins a group: the group, and -1 for the others
    int leads[VPT];
    if (OUT != kNormBf16)
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int pos = (j * T + tid) * 8, g = pos / p.gk;
            leads[j] = g < p.G && pos - g * p.gk == 0 ? g : -1;
        }

    int flip = 0;
    for (int row = blockIdx.x; row < p.rows; row += gridDim.x, flip ^= 1) {
        const bool real_row = OUT != kNormTiles || row < p.M;
        uint64_t h[VPT][4], ss2 = 0;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            uint64_t r[4];
            unpack_pairs(xn[j], h[j]);
            unpack_pairs(rn[j], r);
#pragma unroll
            for (int i = 0; i < 4; ++i) h[j][i] = f2_add(h[j][i], r[i]);         // (without a residual, + 0)
        }
        if (row + static_cast<int>(gridDim.x) < p.rows) load(row + gridDim.x);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) ss2 = f2_fma(h[j][i], h[j][i], ss2);
            const int pos = (j * T + tid) * 8;
            if (p.res_out && real_row && pos < p.K)
                store_row8<WHOLE>(p.res_out + static_cast<int64_t>(row) * p.ldro, pos, p.K, p.vec_ro, h[j]);
        }

        // ---- sum of squares over the block; group maxima of |h w| on the way ----
        // max|y| is max|h w| * n up to fp32 rounding, so the maxima need not wait for
        // the sum.  The 2^40 keeps tiny products normal.  Products of 2^88 and more leave
        // fp32's range so: a thread that meets one (or a NaN or infinity) takes its maximum
        // times 2^-128 instead, where no finite product overflows, and says so by the sign
        // bit, which also makes it the larger of any two as bits.
        uint32_t amax[VPT];
        const int tpg = p.gk >> 3;
        if (OUT != kNormBf16) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                if (!kKeep) load_weight8(p, (j * T + tid) * 8, w[0]);
                float a = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float lo, hi;
                    unpair2(f2_mul(f2_mul(h[j][i], pair2(0x1p40f, 0x1p40f)), w[kKeep ? j : 0][i]), lo, hi);
                    a = max_abs_nan(a, lo, hi);
                }
                amax[j] = __float_as_uint(a);          // (as bits, a NaN is the largest)
            }
            uint32_t far = amax[0];
#pragma unroll
            for (int j = 1; j < VPT; ++j) far = max(far, amax[j]);
            if (far >= 0x7F800000u)
#pragma unroll
                for (int j = 0; j < VPT; ++j)
                    if (amax[j] >= 0x7F800000u) {
                        if (!kKeep) load_weight8(p, (j * T + tid) * 8, w[0]);
                        amax[j] = far_max(h[j], w[kKeep ? j : 0]);
                    }
            for (int o = (tpg < 32 ? tpg : 32) >> 1; o > 0; o >>= 1)
#pragma unroll
                for (int j = 0; j < VPT; ++j) amax[j] = max(amax[j], __shfl_xor_sync(0xffffffffu, amax[j], o));
            if (p.gk == 1024 && lane_id() == 0)
#pragma unroll
                for (int j = 0; j < VPT; ++j) red_max[flip][j * nw + warp_id()] = amax[j];
        }
        float ss, ss_odd;
        unpair2(ss2, ss, ss_odd);
        ss += ss_odd;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (lane_id() == 0) red[flip][warp_id()] = ss;
        __syncthreads();
        ss = static_cast<int>(lane_id()) < nw ? red[flip][lane_id()] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float n = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, static_cast<float>(p.K)) + p.eps));

#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            if (!kKeep) load_weight8(p, (j * T + tid) * 8, w[0]);
#pragma unroll
            for (int i = 0; i < 4; ++i) h[j][i] = f2_mul(f2_mul(h[j][i], pair2(n, n)), w[kKeep ? j : 0][i]);
        }

        if (OUT == kNormBf16) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int pos = (j * T + tid) * 8;
                if (pos < p.K) store_row8<WHOLE>(p.y + static_cast<int64_t>(row) * p.ldy, pos, p.K, p.vec_y, h[j]);
            }
            continue;
        }

        if (p.gk == 1024) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) {            // a group of 1024 is four warps' vectors
                const uint4 m = *reinterpret_cast<const uint4*>(&red_max[flip][(j * nw + warp_id()) & ~3u]);
                amax[j] = max(max(m.x, m.y), max(m.z, m.w));
            }
        }
        const float n40 = n * 0x1p-40f;
        float most[VPT];
        uint32_t far = 0;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            most[j] = __uint_as_float(amax[j]) * n40;
            far |= amax[j];
        }
        if (far >> 31)
#pragma unroll
            for (int j = 0; j < VPT; ++j)
                if (amax[j] >> 31) most[j] = __uint_as_float(amax[j] & 0x7FFFFFFFu) * n * 0x1p64f * 0x1p64f;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int pos = (j * T + tid) * 8;
            float y[8];
            unpair8(h[j], y);
            const uint16_t sb = act_scale_bits(most[j]);
            const float s = bf16_bits_to_f32(sb);
            uint2 q;                                   // 8 codes, a byte each
            if (act_scale_fast(sb)) {
                const float rcp = __frcp_rn(s);
                q = make_uint2(codes4(y, s, rcp), codes4(y + 4, s, rcp));
            } else {
                uint32_t b[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) b[i] = static_cast<uint32_t>(quant_exact(y[i], s)) & 0xFFu;
                q = make_uint2(b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24), b[4] | (b[5] << 8) | (b[6] << 16) | (b[7] << 24));
            }
            if (OUT == kNormTiles) {
                if (pos < p.kb_total * 256) {
                    *reinterpret_cast<uint2*>(p.aq + gemm_act_tile_offset(row, pos, p.tt, p.kb_total)) =
                        make_uint2(__byte_perm(q.x, q.y, 0x6420), __byte_perm(q.x, q.y, 0x7531));   // k0 k2 k4 k6 | k1 k3 k5 k7
                    if (leads[j] >= 0)
                        p.as[(static_cast<int64_t>(row / p.tt) * p.G + leads[j]) * p.tt + row % p.tt] = real_row ? s : 0.0f;
                }
            } else if (pos < p.K) {
                int8_t* qr = p.q + static_cast<int64_t>(row) * p.K;
                if (WHOLE || (pos + 8 <= p.K && p.vec_q)) {
                    *reinterpret_cast<uint2*>(qr + pos) = q;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (pos + i < p.K) qr[pos + i] = static_cast<int8_t>((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
                }
                if (leads[j] >= 0) {
                    const int64_t o = static_cast<int64_t>(leads[j]) * p.M + row;
                    if (p.scale_f32) reinterpret_cast<float*>(p.scale)[o] = s;
                    else reinterpret_cast<uint16_t*>(p.scale)[o] = sb;
                }
            }
        }
    }
}

template <int OUT, int VPT>
cudaError_t launch_vpt(const NormParams& p, int threads, cudaStream_t stream)
{
    // What the bodies without bounds and alignment tests take: 1,024 rows of 5120 5.9 us (codes 9.5)
    // without the tests, 6.5 (10.3) with them.
    const bool whole = p.K % 8 == 0 && p.vec_x && (!p.res || p.vec_r) && (!p.res_out || p.vec_ro) &&
                       (OUT != kNormBf16 || p.vec_y) && (OUT != kNormCodes || p.vec_q);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(std::min(p.rows, 148 * std::max(1, kResident / threads)));
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return whole ? cudaLaunchKernelEx(&cfg, rms_norm_kernel<OUT, VPT, true>, p)
                 : cudaLaunchKernelEx(&cfg, rms_norm_kernel<OUT, VPT, false>, p);
}

template <int OUT>
cudaError_t launch_out(const NormParams& p, cudaStream_t stream)
{
    // positions to cover: the tile form writes whole k-blocks
    const int span = OUT == kNormTiles ? p.kb_total * 256 : p.K;
    const int nvec = (span + 7) / 8;
    const auto threads = [&](int vpt) { return ((nvec + vpt - 1) / vpt + 31) / 32 * 32; };
    // One vector a thread is quickest for few rows; for many, two vectors keep more
    // bytes in flight per register (kManyRows below).  Wide rows take what fits.
    const bool one = threads(1) <= kMaxNormThreads;
    if (one && (p.rows <= kManyRows || nvec < 64)) return launch_vpt<OUT, 1>(p, threads(1), stream);
    if (threads(2) <= 512) return launch_vpt<OUT, 2>(p, threads(2), stream);
    if (one) return launch_vpt<OUT, 1>(p, threads(1), stream);
    if (threads(4) > kMaxNormThreads) return cudaErrorInvalidValue;
    return launch_vpt<OUT, 4>(p, threads(4), stream);
}

}  // namespace

cudaError_t launch_rms_norm(const NormParams& p, int out_kind, cudaStream_t stream)
{
    switch (out_kind) {
        case kNormBf16: return launch_out<kNormBf16>(p, stream);
        case kNormCodes: return launch_out<kNormCodes>(p, stream);
        default: return launch_out<kNormTiles>(p, stream);
    }
}

}  // namespace w4a8
