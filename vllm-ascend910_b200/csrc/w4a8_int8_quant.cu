// w4a8_int8_quant.cu -- activations for the 8-bit linears: int8 codes with one
// scale per token.
//
//   s = max|h| / 127     q = rint(h / s), within +-127     (IEEE fp32, half-even)
//
// of a row h that is x itself, bf16(silu(gate) * up) of x = [gate | up], or the
// root-mean-square norm of x (+ residual) in fp32:
//
//   h = (x + r) / sqrt(sum((x + r)^2) / K + eps) * weight     r' = bf16(x + r)
//
// A row of zeros has s = 0 and codes 0; a row with a value that is not finite has
// s = NaN and codes 0, so that its outputs are NaN.
//
// A block holds its part of a row in registers, 8 elements of 16 bytes a vector (as bf16, or fp32
// behind a norm): x is read once.  A wide row of few is cut over a cluster of eight blocks, whose sums and maxima
// meet in distributed shared memory.  Many wide rows wait for their scale in shared memory.  Rows past 65,536 elements are read twice, the second time out of L2.
//
// Few rows are bound by their chain of loads, sums and a barrier (one row of 5120 1.6 us, 16 of 27,648 3.2, SwiGLU 3.6), many
// by the bytes in flight: 2,048 rows of 5120 7.6 us (4.1 TB/s), 8,192 28, with SwiGLU 12.3 and 49, behind a norm about 15
// (24.4 with a product that takes 9.9 alone); 2,048 of 27,648 43, SwiGLU 61.
//
// Sums and maxima take a warp reduction and a barrier; partial sums are added in a fixed order.
#include <algorithm>

#include "w4a8_common.cuh"
#include "w4a8_kernels.h"

namespace w4a8 {

namespace {

constexpr int kMaxTokThreads = 1024;
constexpr int kMaxRowThreads = 512;
constexpr int kRowBytes = 112 * 1024;      // of a row in shared memory: two blocks an SM at least

// Elements first .. first + 7 of the sixteen in lo, hi (first 0 to 8, the same in the whole warp).
__device__ __forceinline__ uint4 middle8(uint4 lo, uint4 hi, int first)
{
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (first == 8) return hi;
    uint32_t t[6], u[5];
#pragma unroll
    for (int i = 0; i < 6; ++i) t[i] = first & 4 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) u[i] = first & 2 ? t[i + 1] : t[i];
    const int odd = (first & 1) * 16;
    return make_uint4(__funnelshift_r(u[0], u[1], odd), __funnelshift_r(u[1], u[2], odd), __funnelshift_r(u[2], u[3], odd),
                      __funnelshift_r(u[3], u[4], odd));
}

// 8 bf16 elements from position pos < K of a row, zeros past K.  WHOLE: rows are 16-byte aligned and K is a multiple of
// 8.  Otherwise they come out of the two aligned vectors that hold them, each of which is only read where it holds
// an element of the row; by single elements they took eight times the accesses (2,026 rows of 6023
// behind a norm, their product included, 63 us, so 44).
template <bool WHOLE>
__device__ __forceinline__ uint4 load8_raw(const uint16_t* row, int pos, int K, bool vec)
{
    if (WHOLE || (vec && pos + 8 <= K)) return *reinterpret_cast<const uint4*>(row + pos);
    const uintptr_t at = reinterpret_cast<uintptr_t>(row + pos);
    const int mis = static_cast<int>(at & 15) >> 1, left = K - pos;
    const uint4* v = reinterpret_cast<const uint4*>(at & ~static_cast<uintptr_t>(15));
    const uint4 zero = make_uint4(0, 0, 0, 0);
    uint4 r = v[0];
    if (mis) r = middle8(r, left > 8 - mis ? v[1] : zero, mis);
    if (left < 8) {
        uint32_t* w = &r.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (2 * i >= left) w[i] = 0;
            else if (2 * i + 1 >= left) w[i] &= 0xFFFFu;
        }
    }
    return r;
}

template <bool WHOLE>
__device__ __forceinline__ void load8(const uint16_t* row, int pos, int K, bool vec, float (&v)[8])
{
    unpack8_bf16(load8_raw<WHOLE>(row, pos, K, vec), v);
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

__device__ __forceinline__ void store_some(uint16_t* p, uint4 v, int from, int to)
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i >= from && i < to) p[i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
}

// 8 elements at position pos, if below K.  Called by whole warps whose lanes hold neighbouring vectors: where rows suit no
// vectors, a lane stores the aligned one that ends in its own elements and begins in those of the lane before.
template <bool WHOLE>
__device__ __forceinline__ void store8(uint16_t* row, int pos, int K, bool vec, const float (&h)[8])
{
    const uint4 mine = pack8(h);
    const int n = min(K - pos, 8);                            // elements of this lane, maybe none
    if (WHOLE || vec) {
        if (WHOLE ? n > 0 : n == 8) *reinterpret_cast<uint4*>(row + pos) = mine;
        else if (n > 0) store_some(row + pos, mine, 0, n);
        return;
    }
    const int mis = static_cast<int>(reinterpret_cast<uintptr_t>(row + pos) & 15) >> 1, lane = lane_id();
    uint4 prev;
    prev.x = __shfl_up_sync(0xffffffffu, mine.x, 1);
    prev.y = __shfl_up_sync(0xffffffffu, mine.y, 1);
    prev.z = __shfl_up_sync(0xffffffffu, mine.z, 1);
    prev.w = __shfl_up_sync(0xffffffffu, mine.w, 1);
    if (n <= 0) return;
    const int own = 8 - mis;                                  // elements of the vector that are this lane's
    if (lane > 0 && n >= own) {
        *reinterpret_cast<uint4*>(row + pos - mis) = middle8(prev, mine, own);
    } else {
        if (lane > 0 && mis) store_some(row + pos - 8, prev, own, 8);
        store_some(row + pos, mine, 0, min(n, own));
    }
    if (mis && (lane == 31 || pos + 8 >= K)) store_some(row + pos, mine, own, n);
}

__device__ __forceinline__ void load_weight8(const TokenQuantParams& p, int pos, float (&w)[8])
{
    if (p.weight_f32) {
        const float* wf = static_cast<const float*>(p.weight);
        if (p.vec_w && pos + 8 <= p.K) {
            *reinterpret_cast<float4*>(w) = *reinterpret_cast<const float4*>(wf + pos);
            *reinterpret_cast<float4*>(w + 4) = *reinterpret_cast<const float4*>(wf + pos + 4);
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = pos + i < p.K ? wf[pos + i] : 0.0f;
    } else {
        load8<false>(static_cast<const uint16_t*>(p.weight), pos, p.K, p.vec_w, w);
    }
}

// silu(g) u = g / (1 + e^-g) u of two elements, g >= kFarGate (below, nothing of use).  The exponential is the
// hardware's base-2 one, of -g log2(e) as a rounded product and what the rounding left (log2(e) in two parts, after
// Cody and Waite): within 2^-21 of the result.  Above 88 the exponent stays: 1 + e^-88 is 1.
constexpr float kFarGate = -87.0f;         // from about -87.3 on 1 / (1 + e^-g) is below fp32's normal numbers
__device__ __forceinline__ void silu_up2(float g0, float g1, float u0, float u1, float& y0, float& y1)
{
    constexpr float kL = 1.44269502162933349609375f, kLow = 1.925963033500011e-08f;     // log2(e) = kL + kLow
    const uint64_t c = pair2(fminf(g0, 88.0f), fminf(g1, 88.0f));
    const uint64_t t = f2_mul(c, pair2(-kL, -kL)), minus_t = f2_mul(c, pair2(kL, kL));
    const uint64_t low = f2_fma(c, pair2(-kLow, -kLow), f2_fma(c, pair2(-kL, -kL), minus_t));
    float t0, t1, e0, e1, r0, r1;
    unpair2(t, t0, t1);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(t0));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(t1));
    const uint64_t e = pair2(e0, e1);
    constexpr float kLn2 = 0.693147180559945f;
    unpair2(f2_add(f2_fma(e, f2_mul(low, pair2(kLn2, kLn2)), e), pair2(1.0f, 1.0f)), e0, e1);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(e0));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(e1));
    unpair2(f2_mul(f2_mul(pair2(g0, g1), pair2(r0, r1)), pair2(u0, u1)), y0, y1);
}

// The same of one element, g < kFarGate, where 1 / (1 + e^-g) is e^g (1 - e^g) = e^g: its four factors e^(g / 4) one by one
// after u, whose size keeps each product in fp32's range while the last one is in it.
__device__ __forceinline__ float silu_up_far(float g, float u)
{
    const float e = expf(0.25f * g);
    return __fmul_rn(__fmul_rn(__fmul_rn(__fmul_rn(__fmul_rn(g, e), u), e), e), e);
}

// The largest of `most` and of 8 values' bits: above kFarBits where one is below kFarGate (or a NaN of negative sign).
constexpr uint32_t kFarBits = 0xC2AE0000u;
__device__ __forceinline__ uint32_t most_bits(uint32_t most, const float (&g)[8])
{
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(g[i]));
    return most;
}

// The larger of the magnitudes in m and of two bf16 values, each half its own; a NaN wins.
__device__ __forceinline__ uint32_t max_abs2(uint32_t m, uint32_t w)
{
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(w & 0x7FFF7FFFu));
    return r;
}

// What a thread holds of 8 elements: bf16 before the scale is known, fp32 behind a norm.
template <int SRC>
struct Held {
    uint4 v;
    __device__ __forceinline__ void get(float (&x)[8]) const { unpack8_bf16(v, x); }
};
template <>
struct Held<kTokNorm> {
    float v[8];
    __device__ __forceinline__ void get(float (&x)[8]) const
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = v[i];
    }
};

// 8 elements of h; behind a norm, of x + residual.  Gates below kFarGate take a branch of their own (FAR), or are left wrong
// and gathered in `most`, for a thread that met one to take its vectors again: in a loop that waits for its loads the branch
// holds up the next ones (2,048 rows of 27,648 64 to 66 us with it, 60 to 61 without), rows in registers have all theirs
// on the way (8,192 of 5120 48.5 with it, 52.4 the other way).
template <int SRC, bool WHOLE, bool FAR>
__device__ __forceinline__ void row8(const TokenQuantParams& p, const uint16_t* x, const uint16_t* r, int pos, Held<SRC>& h,
                                     uint32_t& most)
{
    if constexpr (SRC == kTokNorm) {
        load8<WHOLE>(x, pos, p.K, p.vec_x, h.v);
        if (r) {
            float u[8];
            load8<WHOLE>(r, pos, p.K, p.vec_r, u);
#pragma unroll
            for (int i = 0; i < 8; ++i) h.v[i] = __fadd_rn(h.v[i], u[i]);
        }
    } else {
        h.v = load8_raw<WHOLE>(x, pos, p.K, p.vec_x);
        if (SRC == kTokSwiglu) {
            float g[8], u[8], y[8];
            const uint4 w = load8_raw<WHOLE>(x + p.K, pos, p.K, p.vec_x && p.K % 8 == 0);
            unpack8_bf16(h.v, g);
            unpack8_bf16(w, u);
#pragma unroll
            for (int i = 0; i < 8; i += 2) silu_up2(g[i], g[i + 1], u[i], u[i + 1], y[i], y[i + 1]);
            if constexpr (!FAR) {
                most = most_bits(most, g);
            } else if (most_bits(0, g) > kFarBits) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (g[i] < kFarGate) y[i] = silu_up_far(g[i], u[i]);
            }
            h.v = pack8(y);
        }
    }
}

// 4 codes, a byte each, by the division alone: scales whose reciprocal fp32 cannot hold.
__device__ __forceinline__ uint32_t codes4_div(const float* x, float s)
{
    uint32_t w = 0;
    if (s > 0.0f)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float q = fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -127.0f), 127.0f);
            w |= (static_cast<uint32_t>(static_cast<int>(q)) & 0xFFu) << (8 * i);
        }
    return w;
}

template <bool WHOLE>
__device__ __forceinline__ void emit8(const TokenQuantParams& p, int8_t* q, int pos, const float (&v)[8], float s, float rcp,
                                      bool fast)
{
    // (|h / s| < 127.5: s is the rounded quotient of the row's maximum and 127)
    const uint32_t lo = fast ? codes4(v, s, rcp) : codes4_div(v, s), hi = fast ? codes4(v + 4, s, rcp) : codes4_div(v + 4, s);
    if (WHOLE || (p.vec_q && pos + 8 <= p.K)) {
        *reinterpret_cast<uint2*>(q + pos) = make_uint2(lo, hi);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (pos + i < p.K) q[pos + i] = static_cast<int8_t>((i < 4 ? lo : hi) >> (8 * (i & 3)));
    }
}

__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// (all threads of all blocks of the cluster)
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A word of this block's shared memory as the cluster's block `rank` has it.
__device__ __forceinline__ uint32_t peer_word(const uint32_t* p, uint32_t rank)
{
    uint32_t at, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

// VPT vectors a thread in registers (0: the row is read twice), a row over CL blocks.
template <int SRC, int VPT, int CL, bool WHOLE>
__global__ void __launch_bounds__(kMaxTokThreads) token_quant_kernel(const TokenQuantParams p)
{
    __shared__ float red_sum[kMaxTokThreads / 32];
    __shared__ uint32_t red_max[kMaxTokThreads / 32];
    __shared__ uint32_t mine[2];                              // the block's sum and maximum, for the cluster's others
    const int tid = threadIdx.x, T = blockDim.x, nw = T >> 5;
    // The product that follows may start once everything before this kernel is done: it reads its weights
    // without waiting for the codes.
    pdl_wait();
    pdl_launch_dependents();

    const int64_t row = blockIdx.x / CL;
    const int rank = CL > 1 ? static_cast<int>(cluster_rank()) : 0;
    const uint16_t* x = p.x + row * p.ldx;
    const uint16_t* r = SRC == kTokNorm && p.res ? p.res + row * p.ldr : nullptr;
    constexpr int HOLD = VPT ? VPT : 1;
    const int vecs = VPT ? VPT : (p.K + 8 * T - 1) / (8 * T);
    const auto at = [&](int j) { return ((j * CL + rank) * T + tid) * 8; };
    Held<SRC> h[HOLD] = {};
    float ss = 0.0f, big = 0.0f;
    uint32_t big2 = 0, most = 0;
#pragma unroll
    for (int j = 0; j < vecs; ++j)
        if (VPT && at(j) < p.K) row8<SRC, WHOLE, true>(p, x, r, at(j), h[j], most);
#pragma unroll
    for (int j = 0; j < vecs; ++j) {
        const int pos = at(j);
        Held<SRC>& e = h[VPT ? j : 0];
        if constexpr (SRC == kTokNorm) {
            if (p.res_out) store8<WHOLE>(p.res_out + row * p.ldro, pos, p.K, p.vec_ro, e.v);     // (whole warps)
            if (pos >= p.K) continue;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(e.v[i], e.v[i], ss);
        } else {
            if (pos >= p.K) continue;
            if (!VPT) row8<SRC, WHOLE, true>(p, x, r, pos, e, most);
            big2 = max_abs2(max_abs2(max_abs2(max_abs2(big2, e.v.x), e.v.y), e.v.z), e.v.w);
        }
    }
    if (SRC != kTokNorm) big = max_abs_nan(0.0f, __uint_as_float(big2 << 16), __uint_as_float(big2 & 0xFFFF0000u));
    if constexpr (SRC == kTokNorm) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (lane_id() == 0) red_sum[warp_id()] = ss;
        __syncthreads();
        ss = static_cast<int>(lane_id()) < nw ? red_sum[lane_id()] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (CL > 1) {
            if (tid == 0) mine[0] = __float_as_uint(ss);
            cluster_sync();
            ss = 0.0f;
#pragma unroll
            for (int c = 0; c < CL; ++c) ss += __uint_as_float(peer_word(&mine[0], c));
        }
        const float n = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, static_cast<float>(p.K)) + p.eps));
#pragma unroll
        for (int j = 0; j < HOLD; ++j) {
            if (at(j) >= p.K) continue;
            float w[8];
            load_weight8(p, at(j), w);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[j].v[i] = __fmul_rn(__fmul_rn(h[j].v[i], n), w[i]);
#pragma unroll
            for (int i = 0; i < 8; i += 2) big = max_abs_nan(big, h[j].v[i], h[j].v[i + 1]);
        }
    }
    uint32_t amax = __reduce_max_sync(0xffffffffu, __float_as_uint(big));     // (as bits, a NaN is the largest)
    if (lane_id() == 0) red_max[warp_id()] = amax;
    __syncthreads();
    amax = __reduce_max_sync(0xffffffffu, static_cast<int>(lane_id()) < nw ? red_max[lane_id()] : 0u);
    if (CL > 1) {
        if (tid == 0) mine[1] = amax;
        cluster_sync();
#pragma unroll
        for (int c = 0; c < CL; ++c) amax = max(amax, peer_word(&mine[1], c));
    }
    const bool finite = amax < 0x7F800000u;
    const float s = finite ? __fdiv_rn(__uint_as_float(amax), 127.0f) : __uint_as_float(0x7FC00000u);
    if (tid == 0 && rank == 0) p.scale[row] = s;
    const bool fast = finite && s >= 1.1754943508222875e-38f;
    const float rcp = fast ? __frcp_rn(s) : 0.0f;
    int8_t* q = p.q + row * p.ldq;
#pragma unroll
    for (int j = 0; j < vecs; ++j) {
        const int pos = at(j);
        if (pos >= p.K) continue;
        Held<SRC>& e = h[VPT ? j : 0];
        if (!VPT) row8<SRC, WHOLE, true>(p, x, r, pos, e, most);
        float v[8];
        e.get(v);
        emit8<WHOLE>(p, q, pos, v, s, rcp, fast);
    }
    if (CL > 1) cluster_sync();                               // (the others read this block's words until here)
}

// Many rows: the row waits for its scale in shared memory (bf16; fp32 behind a norm), which leaves room
// for 48 warps an SM where registers held 28.
template <int SRC, bool WHOLE>
__global__ void __launch_bounds__(kMaxRowThreads, 1536 / kMaxRowThreads) token_quant_rows_kernel(const TokenQuantParams p)
{
    extern __shared__ __align__(16) uint8_t staged[];
    __shared__ float red_sum[kMaxRowThreads / 32];
    __shared__ uint32_t red_max[kMaxRowThreads / 32];
    const int tid = threadIdx.x, T = blockDim.x, nw = T >> 5, nvec = (p.K + 7) / 8, lane = lane_id();
    pdl_wait();
    pdl_launch_dependents();
    const int64_t row = blockIdx.x;
    const uint16_t* x = p.x + row * p.ldx;
    const uint16_t* r = SRC == kTokNorm && p.res ? p.res + row * p.ldr : nullptr;
    Held<SRC>* hold = reinterpret_cast<Held<SRC>*>(staged);
    float big = 0.0f;
    if constexpr (SRC == kTokNorm) {
        // (halves of the 32 bytes a vector apart, so that a warp's accesses are to 16 bytes next to each other)
        float4 *lo = reinterpret_cast<float4*>(staged), *hi = lo + nvec;
        float ss = 0.0f;
#pragma unroll 2
        for (int v = tid; WHOLE ? v < nvec : v - lane < nvec; v += T) {      // (whole warps for store8)
            Held<SRC> h = {};
            uint32_t none = 0;
            if (WHOLE || v < nvec) row8<SRC, WHOLE, false>(p, x, r, 8 * v, h, none);
            if (p.res_out) store8<WHOLE>(p.res_out + row * p.ldro, 8 * v, p.K, p.vec_ro, h.v);
            if (!WHOLE && v >= nvec) break;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(h.v[i], h.v[i], ss);
            lo[v] = make_float4(h.v[0], h.v[1], h.v[2], h.v[3]);
            hi[v] = make_float4(h.v[4], h.v[5], h.v[6], h.v[7]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (lane_id() == 0) red_sum[warp_id()] = ss;
        __syncthreads();
        ss = static_cast<int>(lane_id()) < nw ? red_sum[lane_id()] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float n = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, static_cast<float>(p.K)) + p.eps));
#pragma unroll 2
        for (int v = tid; v < nvec; v += T) {
            float w[8], h[8];
            load_weight8(p, 8 * v, w);
            *reinterpret_cast<float4*>(h) = lo[v];
            *reinterpret_cast<float4*>(h + 4) = hi[v];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = __fmul_rn(__fmul_rn(h[i], n), w[i]);
#pragma unroll
            for (int i = 0; i < 8; i += 2) big = max_abs_nan(big, h[i], h[i + 1]);
            lo[v] = make_float4(h[0], h[1], h[2], h[3]);
            hi[v] = make_float4(h[4], h[5], h[6], h[7]);
        }
    } else {
        uint32_t big2 = 0, most = 0;
#pragma unroll 2
        for (int v = tid; v < nvec; v += T) {
            Held<SRC> h;
            row8<SRC, WHOLE, false>(p, x, r, 8 * v, h, most);
            big2 = max_abs2(max_abs2(max_abs2(max_abs2(big2, h.v.x), h.v.y), h.v.z), h.v.w);
            hold[v] = h;
        }
        if (SRC == kTokSwiglu && most > kFarBits) {
            big2 = 0;
#pragma unroll 1
            for (int v = tid; v < nvec; v += T) {
                Held<SRC> h;
                row8<SRC, WHOLE, true>(p, x, r, 8 * v, h, most);
                big2 = max_abs2(max_abs2(max_abs2(max_abs2(big2, h.v.x), h.v.y), h.v.z), h.v.w);
                hold[v] = h;
            }
        }
        big = max_abs_nan(0.0f, __uint_as_float(big2 << 16), __uint_as_float(big2 & 0xFFFF0000u));
    }
    uint32_t amax = __reduce_max_sync(0xffffffffu, __float_as_uint(big));     // (as bits, a NaN is the largest)
    if (lane_id() == 0) red_max[warp_id()] = amax;
    __syncthreads();
    amax = __reduce_max_sync(0xffffffffu, static_cast<int>(lane_id()) < nw ? red_max[lane_id()] : 0u);
    const bool finite = amax < 0x7F800000u;
    const float s = finite ? __fdiv_rn(__uint_as_float(amax), 127.0f) : __uint_as_float(0x7FC00000u);
    if (tid == 0) p.scale[row] = s;
    const bool fast = finite && s >= 1.1754943508222875e-38f;
    const float rcp = fast ? __frcp_rn(s) : 0.0f;
    int8_t* q = p.q + row * p.ldq;
#pragma unroll 2
    for (int v = tid; v < nvec; v += T) {                     // (a thread's own vectors: no barrier since)
        float h[8];
        if constexpr (SRC == kTokNorm) {
            const float4 *lo = reinterpret_cast<const float4*>(staged), *hi = lo + nvec;
            *reinterpret_cast<float4*>(h) = lo[v];
            *reinterpret_cast<float4*>(h + 4) = hi[v];
        } else {
            hold[v].get(h);
        }
        emit8<WHOLE>(p, q, 8 * v, h, s, rcp, fast);
    }
}

bool whole_rows(const TokenQuantParams& p, int src)
{
    return p.K % 8 == 0 && p.vec_x && p.vec_q && (src != kTokNorm || ((!p.res || p.vec_r) && (!p.res_out || p.vec_ro)));
}

template <int SRC>
cudaError_t launch_rows(const TokenQuantParams& p, cudaStream_t stream)
{
    const int threads = p.K <= 2048 * 8 ? 256 : 512;
    const size_t smem = static_cast<size_t>((p.K + 7) / 8) * (SRC == kTokNorm ? 32 : 16);
    const auto kern = whole_rows(p, SRC) ? token_quant_rows_kernel<SRC, true> : token_quant_rows_kernel<SRC, false>;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowBytes);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.M));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

template <int SRC, int VPT, int CL = 1>
cudaError_t launch(const TokenQuantParams& p, int threads, cudaStream_t stream)
{
    const bool whole = whole_rows(p, SRC);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.M) * CL);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CL;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CL > 1 ? 2 : 1;
    return whole ? cudaLaunchKernelEx(&cfg, token_quant_kernel<SRC, VPT, CL, true>, p)
                 : cudaLaunchKernelEx(&cfg, token_quant_kernel<SRC, VPT, CL, false>, p);
}

constexpr int kFewRows = 64;               // rows that a cluster each is no loss for
constexpr int kManyRows = 296;

template <int SRC>
cudaError_t launch_source(const TokenQuantParams& p, cudaStream_t stream)
{
    const int nvec = (p.K + 7) / 8;
    const auto threads = [&](int vpt) { return ((nvec + vpt - 1) / vpt + 31) / 32 * 32; };
    if (nvec > 1024 && nvec <= 8 * 1024 && p.M <= kFewRows) return launch<SRC, 1, 8>(p, threads(8), stream);
    // Many wide rows through shared memory (2,048 of 27,648: plain 43 us, SwiGLU 61, norm 124; in registers 49, 79 and 128),
    // narrower ones in registers (2,048 of 5120: plain 7.5 us, through shared memory 8.7).
    if (p.M > kManyRows && nvec * (SRC == kTokNorm ? 32 : 16) <= kRowBytes && nvec > 1024)
        return launch_rows<SRC>(p, stream);
    // Many rows: more vectors a thread keep more bytes in flight.
    if (p.M > kManyRows) {
        if constexpr (SRC != kTokNorm)
            if (threads(8) >= 256 && threads(8) <= kMaxTokThreads) return launch<SRC, 8>(p, threads(8), stream);
        if (threads(4) >= 128 && threads(4) <= kMaxTokThreads) return launch<SRC, 4>(p, threads(4), stream);
        if (threads(2) >= 128 && threads(2) <= kMaxTokThreads) return launch<SRC, 2>(p, threads(2), stream);
    }
    if (threads(1) <= kMaxTokThreads) return launch<SRC, 1>(p, threads(1), stream);
    if (threads(2) <= kMaxTokThreads) return launch<SRC, 2>(p, threads(2), stream);
    if (threads(4) <= kMaxTokThreads) return launch<SRC, 4>(p, threads(4), stream);
    if constexpr (SRC == kTokNorm) {
        return cudaErrorInvalidValue;
    } else {
        if (threads(8) <= kMaxTokThreads) return launch<SRC, 8>(p, threads(8), stream);
        return launch<SRC, 0>(p, kMaxTokThreads, stream);
    }
}

}  // namespace

cudaError_t launch_token_quant(const TokenQuantParams& p, int source, cudaStream_t stream)
{
    switch (source) {
        case kTokPlain: return launch_source<kTokPlain>(p, stream);
        case kTokSwiglu: return launch_source<kTokSwiglu>(p, stream);
        default: return launch_source<kTokNorm>(p, stream);
    }
}

}  // namespace w4a8
