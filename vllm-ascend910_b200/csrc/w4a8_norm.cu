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
//                where norm, store and quantise would make two
//   kNormTiles   the same codes and scales in the GEMM's operand order, straight
//                into a linear call's workspace (QuantParams' kOutKernel form)
//
// One block holds one row in registers: a thread owns VPT vectors of 8
// consecutive elements (16-byte loads), so x and r are read once and y, r' are
// written once.  The sum of squares takes one warp reduction and one barrier;
// the fp32 parts are added in a fixed order, so repeated calls give the same
// bits.  A group's amax stays within GK / 8 neighbouring threads.  Bound by HBM
// for many rows and by the launch and two dependent load latencies for few.
#include "w4a8_common.cuh"
#include "w4a8_kernels.h"

namespace w4a8 {

namespace {

constexpr int kMaxNormThreads = 1024;

__device__ __forceinline__ void load_row8(const uint16_t* row, int pos, int K, bool vec, float (&v)[8])
{
    if (vec && pos + 8 <= K) {
        unpack8_bf16(*reinterpret_cast<const uint4*>(row + pos), v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = pos + i < K ? bf16_bits_to_f32(row[pos + i]) : 0.0f;
    }
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

__device__ __forceinline__ void store_row8(uint16_t* row, int pos, int K, bool vec, const float (&v)[8])
{
    if (vec && pos + 8 <= K) {
        *reinterpret_cast<uint4*>(row + pos) = pack8_bf16(v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (pos + i < K) row[pos + i] = f32_to_bf16_bits(v[i]);
    }
}

template <int OUT, int VPT>
__global__ void __launch_bounds__(kMaxNormThreads) rms_norm_kernel(const NormParams p)
{
    __shared__ float red[kMaxNormThreads / 32];
    __shared__ uint32_t red_max[VPT][kMaxNormThreads / 32];

    pdl_launch_dependents();
    const int row = blockIdx.x, tid = threadIdx.x, T = blockDim.x;
    const bool real_row = OUT != kNormTiles || row < p.M;
    pdl_wait();

    float h[VPT][8];
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int pos = (j * T + tid) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[j][i] = 0.0f;
        if (real_row && pos < p.K) {
            load_row8(p.x + static_cast<int64_t>(row) * p.ldx, pos, p.K, p.vec_x, h[j]);
            if (p.res) {
                float r[8];
                load_row8(p.res + static_cast<int64_t>(row) * p.ldr, pos, p.K, p.vec_r, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[j][i] = __fadd_rn(h[j][i], r[i]);
            }
        }
    }
    // the weight's loads go out with the row's: they do not depend on the sum
    float w[VPT][8];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int pos = (j * T + tid) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[j][i] = 0.0f;
        if (pos < p.K) {
            if (p.weight_f32) {
                const float* wf = static_cast<const float*>(p.weight);
#pragma unroll
                for (int i = 0; i < 8; ++i) w[j][i] = pos + i < p.K ? wf[pos + i] : 0.0f;
            } else {
                load_row8(static_cast<const uint16_t*>(p.weight), pos, p.K, p.vec_w, w[j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(h[j][i], h[j][i], ss);
        const int pos = (j * T + tid) * 8;
        if (p.res_out && real_row && pos < p.K)
            store_row8(p.res_out + static_cast<int64_t>(row) * p.ldro, pos, p.K, p.vec_ro, h[j]);
    }

    // ---- sum of squares over the block ----
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const int nw = T >> 5;
    if (lane_id() == 0) red[warp_id()] = ss;
    __syncthreads();
    ss = static_cast<int>(lane_id()) < nw ? red[lane_id()] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float n = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, static_cast<float>(p.K)) + p.eps));

#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) h[j][i] = __fmul_rn(__fmul_rn(h[j][i], n), w[j][i]);

    if (OUT == kNormBf16) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int pos = (j * T + tid) * 8;
            if (pos < p.K) store_row8(p.y + static_cast<int64_t>(row) * p.ldy, pos, p.K, p.vec_y, h[j]);
        }
        return;
    }

    // ---- group amax (as bits of |y|: a NaN wins over every number) ----
    const int tpg = p.gk >> 3;
    uint32_t amax[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        uint32_t a = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(h[j][i]) & 0x7FFFFFFFu);
        for (int o = (tpg < 32 ? tpg : 32) >> 1; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
        if (tpg > 32 && lane_id() == 0) red_max[j][warp_id()] = a;
        amax[j] = a;
    }
    if (tpg > 32) {
        __syncthreads();
        const int w0 = (warp_id() / (tpg >> 5)) * (tpg >> 5);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            uint32_t a = 0;
            for (int k = 0; k < (tpg >> 5); ++k) a = max(a, red_max[j][w0 + k]);
            amax[j] = a;
        }
    }

#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int pos = (j * T + tid) * 8;
        const int g = pos / p.gk;
        const uint16_t sb = act_scale_bits(__uint_as_float(amax[j]));
        const float s = bf16_bits_to_f32(sb);
        int q[8];
        if (act_scale_fast(sb)) {
            const float rcp = __frcp_rn(s);
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = quant_fast(h[j][i], s, rcp);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = quant_exact(h[j][i], s);
        }
        const bool leader = pos % p.gk == 0;
        if (OUT == kNormTiles) {
            if (pos < p.kb_total * 256) {
                *reinterpret_cast<uint2*>(p.aq + gemm_act_tile_offset(row, pos, p.tt, p.kb_total)) =
                    pack_operand_order(q);
                if (leader && g < p.G)
                    p.as[(static_cast<int64_t>(row / p.tt) * p.G + g) * p.tt + row % p.tt] = real_row ? s : 0.0f;
            }
        } else if (pos < p.K) {
            int8_t* qr = p.q + static_cast<int64_t>(row) * p.K;
            if (pos + 8 <= p.K && p.vec_q) {
                const uint32_t w0 = (q[0] & 0xFF) | ((q[1] & 0xFF) << 8) | ((q[2] & 0xFF) << 16) |
                                    (static_cast<uint32_t>(q[3] & 0xFF) << 24);
                const uint32_t w1 = (q[4] & 0xFF) | ((q[5] & 0xFF) << 8) | ((q[6] & 0xFF) << 16) |
                                    (static_cast<uint32_t>(q[7] & 0xFF) << 24);
                *reinterpret_cast<uint2*>(qr + pos) = make_uint2(w0, w1);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (pos + i < p.K) qr[pos + i] = static_cast<int8_t>(q[i]);
            }
            if (leader) {
                const int64_t o = static_cast<int64_t>(g) * p.M + row;
                if (p.scale_f32) reinterpret_cast<float*>(p.scale)[o] = s;
                else reinterpret_cast<uint16_t*>(p.scale)[o] = sb;
            }
        }
    }
}

template <int OUT>
cudaError_t launch_out(const NormParams& p, cudaStream_t stream)
{
    // positions to cover: the tile form writes whole k-blocks
    const int span = OUT == kNormTiles ? p.kb_total * 256 : p.K;
    const int nvec = (span + 7) / 8;
    // threads per row: a multiple of a warp, and of a 1024-element group's 128 threads
    const int unit = OUT != kNormBf16 && p.gk > 256 ? p.gk / 8 : 32;
    int vpt = 1;
    while (vpt < 4 && (nvec + vpt - 1) / vpt > kMaxNormThreads) vpt *= 2;
    const int threads = ((nvec + vpt - 1) / vpt + unit - 1) / unit * unit;
    if (threads > kMaxNormThreads) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.rows);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    switch (vpt) {
        case 1: return cudaLaunchKernelEx(&cfg, rms_norm_kernel<OUT, 1>, p);
        case 2: return cudaLaunchKernelEx(&cfg, rms_norm_kernel<OUT, 2>, p);
        default: return cudaLaunchKernelEx(&cfg, rms_norm_kernel<OUT, 4>, p);
    }
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
