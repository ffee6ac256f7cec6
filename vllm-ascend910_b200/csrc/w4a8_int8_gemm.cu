// w4a8_int8_gemm.cu -- product of int8 codes with a scale per token and per channel.
//
//   y[t, n] = bf16( sum_k q[t, k] w[n, k] * s[t] * ws[n] + b[n] )
//
// The sums are exact 32-bit integers (K <= 131071: 128 * 128 * K < 2^31), so that neither
// the order of the products nor how K is cut changes a bit; each sum becomes fp32 once,
// is multiplied by the token's and then the channel's scale, the bias is added, and
// the result is rounded to bf16.
//
// Both operands are K-major bytes, brought by TMA in boxes of 128 bytes x rows with the
// 128-byte swizzle that the MMA's descriptors name; what lies past K, M or N arrives as
// zeros.  tcgen05.mma kind::i8 multiplies 32 bytes of K an instruction.
//
// few (up to kFewTokens tokens): the weights' bytes bound it (64 tokens of 55296 x 5120 45.7 us, 6.2 TB/s; one of
//   7168 x 5120 9.6, 3.8 TB/s, where launch and join weigh).  A tile is 128 channels (the MMA's rows) by 16, 32, 64 or 128
//   tokens (its columns), so that few tokens waste little.  Two CTAs an SM, each with a ring of up to 104 KB in flight.
//   With fewer tiles than CTAs, a cluster cuts a tile's K: each CTA leaves its sums in shared memory and adds up a
//   share of the tokens out of all of them over distributed shared memory.  128 tokens still belong here: 55296 x 5120
//   51.4 us, 57.4 by the other kernel; 7168 x 5120 14.2 and 16.6.
// many: the tensor pipe bounds it (2,048 tokens of 55296 x 5120 349 us for one launch, 3.3 POP/s; 370 in a loop of some, 3.1;
//   438 with the norm in front in a loop of seconds, 2.6 by the clock that the power limit leaves).  A pair of CTAs
//   (cta_group::2) owns 256 tokens x 256 (or 128) channels: each brings 128 tokens and half of the channels, one of them issues
//   for both.  Two accumulators fill tensor memory, one in work while the other is stored.
//
// Each wait for a barrier is bounded; one that runs out ends the CTA's roles and leaves a code in
// the workspace's status word.
#include <algorithm>
#include <atomic>

#include "w4a8_common.cuh"
#include "w4a8_kernels.h"

namespace w4a8 {

namespace {

constexpr int kThreads = 192;              // few: producer, issuer, four epilogue warps
constexpr int kManyThreads = 320;          // many: eight epilogue warps
constexpr int kFewTokens = 128;

// Ids of the waits in the status word (kDevTimeoutBase + id; the other kernels' are smaller).
enum : int { kWaitEmpty = 0x40, kWaitFull, kWaitAccFull, kWaitAccEmpty, kWaitDrain };

// ---------------------------------------------------------------- instructions

// n columns of tensor memory; other CTAs of the SM may then have theirs.
template <int G>
__device__ __forceinline__ void alloc_columns(uint32_t* dst, uint32_t n)
{
    if (G == 1) {
        tmem_alloc(dst, n);
        tmem_relinquish();
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(n) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}

template <int G>
__device__ __forceinline__ void free_columns(uint32_t t, uint32_t n)
{
    if (G == 1) tmem_dealloc(t, n);
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(t), "r"(n) : "memory");
}

// D[tmem] (+)= A[smem] * B[smem], int8 x int8 -> int32, by one CTA or a pair.
template <int G>
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    if (G == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
}

// Arrive on `bar` of both CTAs of the pair once the MMAs issued so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar, uint32_t lead)
{
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(static_cast<uint16_t>(3u << lead))
        : "memory");
}

// Box of a tensor map into this CTA's shared memory, its bytes counted by a barrier that may be the pair's other CTA's.
__device__ __forceinline__ void load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y, uint64_t policy)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar), "l"(policy)
        : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// This CTA's shared address as it is in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// (What the arrival orders is tensor memory, by the fence before it.  A release for the whole cluster would also wait for
// the tile's stores.)
__device__ __forceinline__ void arrive_remote(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// All threads of the cluster (each CTA gets here whatever its waits gave).
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t load_cluster(uint32_t addr)
{
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ void load_columns32(uint32_t taddr, uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, "
        "[%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
// Later uses of r come after the wait for the loads that filled it.
__device__ __forceinline__ void settle32(uint32_t (&r)[32])
{
#pragma unroll
    for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i]));
}

__device__ __forceinline__ float scaled(uint32_t sum, float s, float ws, float b)
{
    return __fadd_rn(__fmul_rn(__fmul_rn(static_cast<float>(static_cast<int32_t>(sum)), s), ws), b);
}
__device__ __forceinline__ uint32_t two(float lo, float hi)
{
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}

// After a wait that ran out: gives what is on its way to a barrier until `deadline` to arrive.
__device__ __forceinline__ void settle(uint64_t* bar, uint32_t parity, uint64_t deadline)
{
    while (!mbar_try_wait(bar, parity) && global_timer_ns() < deadline) {
    }
}

// A warp's 32 rows of 32 outputs from `turn` into y, BYTES an access: 64 / BYTES lanes a row.
template <int BYTES>
__device__ __forceinline__ void put_rows(const Int8GemmParams& p, int n, int64_t row0, const uint16_t (*turn)[40])
{
    constexpr int LANES = 64 / BYTES, ROWS = 32 / LANES, EACH = BYTES / 2;
    const int lane = lane_id(), c = lane % LANES * EACH, first = lane / LANES;
    const int rows = static_cast<int>(min(static_cast<int64_t>(32), p.M - row0));
    uint16_t* y = p.y + (row0 + first) * p.ldy + n + c;
    const int64_t step = ROWS * p.ldy;
    if (n + c + EACH <= p.N) {
#pragma unroll 8
        for (int i = first; i < rows; i += ROWS, y += step) {
            if (BYTES == 16) *reinterpret_cast<uint4*>(y) = *reinterpret_cast<const uint4*>(&turn[i][c]);
            else if (BYTES == 8) *reinterpret_cast<uint2*>(y) = *reinterpret_cast<const uint2*>(&turn[i][c]);
            else if (BYTES == 4) *reinterpret_cast<uint32_t*>(y) = *reinterpret_cast<const uint32_t*>(&turn[i][c]);
            else *y = turn[i][c];
        }
    } else {
        for (int i = first; i < rows; i += ROWS, y += step)
            for (int e = 0; e < EACH && n + c + e < p.N; ++e) y[e] = turn[i][c + e];
    }
}

// 32 sums of a lane's row (channels n .. n + 31) into y: scaled, rounded and stored by the widest access that
// `align` allows, 32 bytes of a row a thread or, turned in shared memory, whole rows of 64.  All lanes of the warp call
// it; `turn` is the warp's; `scale`, `bias`: the channels' in shared memory.
__device__ __forceinline__ void put32(const Int8GemmParams& p, const uint32_t (&r)[32], int n, int64_t row, bool in, float s,
                                      const float* scale, const float* bias, int align, uint16_t (*turn)[40])
{
    const int lane = lane_id();
    if (n >= p.N) return;
    uint32_t o[16];
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
        const float4 ws = *reinterpret_cast<const float4*>(scale + i), b = *reinterpret_cast<const float4*>(bias + i);
        o[i / 2] = two(scaled(r[i], s, ws.x, b.x), scaled(r[i + 1], s, ws.y, b.y));
        o[i / 2 + 1] = two(scaled(r[i + 2], s, ws.z, b.z), scaled(r[i + 3], s, ws.w, b.w));
    }
    if (n + 32 <= p.N && align >= 32) {
        uint16_t* y = p.y + row * p.ldy + n;
        if (in)
#pragma unroll
            for (int i = 0; i < 16; i += 8)                  // 32 bytes: a whole sector a thread
                asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(y + 2 * i), "r"(o[i]), "r"(o[i + 1]),
                             "r"(o[i + 2]), "r"(o[i + 3]), "r"(o[i + 4]), "r"(o[i + 5]), "r"(o[i + 6]), "r"(o[i + 7])
                             : "memory");
        return;
    }
#pragma unroll
    for (int i = 0; i < 16; i += 4) *reinterpret_cast<uint4*>(&turn[lane][2 * i]) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
    __syncwarp();
    if (align >= 16) put_rows<16>(p, n, row - lane, turn);
    else if (align == 8) put_rows<8>(p, n, row - lane, turn);
    else if (align == 4) put_rows<4>(p, n, row - lane, turn);
    else put_rows<2>(p, n, row - lane, turn);
    __syncwarp();
}

// G tokens from c on of a warp's 32 channels (n0 ..; a lane a channel) into y: rounded sums v, turned in `turn` so
// that a lane stores 16 bytes of a token where rows suit that, else a lane its channel.
template <int G>
__device__ __forceinline__ void put_tokens(const Int8GemmParams& p, const float (&v)[G], int c, int n0, bool vec, uint16_t (*turn)[40])
{
    const int lane = lane_id();
    if (vec && n0 + 32 <= p.N) {
#pragma unroll
        for (int i = 0; i < G; ++i) turn[i][lane] = f32_to_bf16_bits(v[i]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < G; i += 8) {
            const int t = i + (lane >> 2), at = (lane & 3) * 8;
            if (t < G && c + t < p.M)
                *reinterpret_cast<uint4*>(p.y + static_cast<int64_t>(c + t) * p.ldy + n0 + at) = *reinterpret_cast<const uint4*>(&turn[t][at]);
        }
        __syncwarp();
    } else if (n0 + lane < p.N) {
#pragma unroll
        for (int i = 0; i < G; ++i)
            if (c + i < p.M) p.y[static_cast<int64_t>(c + i) * p.ldy + n0 + lane] = f32_to_bf16_bits(v[i]);
    }
}

// ---------------------------------------------------------------- few tokens

template <int TT>
struct Few {
    static constexpr int STAGE = 16384 + TT * 128;
    static constexpr int STAGES = 104 * 1024 / STAGE;
    static constexpr int COLUMNS = 2 * TT < 32 ? 32 : 2 * TT;
    static constexpr size_t SMEM = 1024 + static_cast<size_t>(STAGES) * STAGE;
};

template <int TT, int SPLIT>
__global__ void __launch_bounds__(kThreads, 2) int8_few_kernel(const __grid_constant__ Int8GemmParams p, const int vec)
{
    using C = Few<TT>;
    constexpr int S = C::STAGES;
    static_assert(TT * 128 * 4 <= S * C::STAGE, "the sums of a split tile lie where the ring was");
    extern __shared__ uint8_t raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t full[S], empty[S], acc_full[2], acc_empty[2], done;
    __shared__ uint32_t tmem_at;
    __shared__ int abort_flag;
    __shared__ float sh_scale[TT];
    __shared__ __align__(16) uint16_t turn[4][16][40];

    const int warp = warp_id(), lane = lane_id();
    const uint32_t rank = SPLIT > 1 ? cluster_rank() : 0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 4);
        }
        mbar_init(&done, 1);
        abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&p.tm_w);
        tma_prefetch_desc(&p.tm_a);
    }
    if (warp == 1) alloc_columns<1>(&tmem_at, C::COLUMNS);
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    volatile int* quit = &abort_flag;

    const int tiles = (p.N + 127) / 128, KB = (p.K + 127) / 128;
    const int t0 = blockIdx.x / SPLIT, step = gridDim.x / SPLIT;
    const int kb0 = static_cast<int>(rank) * KB / SPLIT, kb1 = (static_cast<int>(rank) + 1) * KB / SPLIT;

    if (warp == 0) {
        if (lane == 0) {
            const uint64_t stream = policy_evict_first(), stay = policy_evict_last();
            // the ring's first weights do not wait for the codes
            const int n0 = t0 < tiles ? kb1 - kb0 : 0, first = min(n0, S);
            for (int i = 0; i < first; ++i) {
                mbar_arrive_expect_tx(&full[i], C::STAGE);
                tma_load_2d_hint(ring + i * C::STAGE, &p.tm_w, &full[i], (kb0 + i) * 128, t0 * 128, stream);
            }
            pdl_wait();
            for (int i = 0; i < first; ++i)
                tma_load_2d_hint(ring + i * C::STAGE + 16384, &p.tm_a, &full[i], (kb0 + i) * 128, 0, stay);
            int it = 0;
            bool ok = true;
            for (int t = t0; t < tiles && ok; t += step)
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    if (it < first) continue;
                    const int s = it % S, round = it / S;
                    if (round > 0 && !mbar_wait(&empty[s], (round - 1) & 1, quit, p.status, kWaitEmpty)) {
                        ok = false;
                        break;
                    }
                    mbar_arrive_expect_tx(&full[s], C::STAGE);
                    tma_load_2d_hint(ring + s * C::STAGE, &p.tm_w, &full[s], kb * 128, t * 128, stream);
                    tma_load_2d_hint(ring + s * C::STAGE + 16384, &p.tm_a, &full[s], kb * 128, 0, stay);
                }
            pdl_launch_dependents();
            // no copy may be on its way when the CTA ends: the last round of each stage has been read
            for (int i = max(it - S, 0); i < it; ++i)
                mbar_wait(&empty[i % S], (i / S) & 1, quit, p.status, kWaitDrain);
            if (*quit) {
                const uint64_t deadline = global_timer_ns() + kWaitLimitNs;
                for (int i = max(it - S, 0); i < it; ++i) settle(&full[i % S], (i / S) & 1, deadline);
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            constexpr uint32_t idesc = idesc_i8(128, TT);
            const uint32_t base = smem_u32(ring);
            int it = 0, tile = 0;
            bool ok = true;
            for (int t = t0; t < tiles && ok; t += step, ++tile) {
                const int a = tile & 1;
                if (tile >= 2 && !mbar_wait(&acc_empty[a], ((tile >> 1) - 1) & 1, quit, p.status, kWaitAccEmpty)) break;
                tc_fence_after();
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    const int s = it % S;
                    if (!mbar_wait(&full[s], (it / S) & 1, quit, p.status, kWaitFull)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t wd = smem_desc_sw128(base + s * C::STAGE), ad = smem_desc_sw128(base + s * C::STAGE + 16384);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_i8<1>(tmem + a * TT, wd + 2 * k, ad + 2 * k, idesc, kb > kb0 || k > 0);
                    tc_commit(&empty[s]);
                }
                if (ok) tc_commit(&acc_full[a]);
            }
            if (*quit) {                   // (tensor memory is given back below)
                tc_commit(&done);
                settle(&done, 0, global_timer_ns() + kWaitLimitNs);
            }
        }
    } else {
        const int quad = warp & 3, ch = quad * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        pdl_wait();
        for (int i = (warp - 2) * 32 + lane; i < TT; i += 128) sh_scale[i] = i < p.M ? p.a_scale[i] : 0.0f;
        asm volatile("bar.sync 1, 128;" ::: "memory");
        int tile = 0;
        for (int t = t0; t < tiles; t += step, ++tile) {
            const int a = tile & 1;
            const int64_t n = static_cast<int64_t>(t) * 128 + ch;
            const bool in = n < p.N;
            const float ws = in ? p.w_scale[n] : 0.0f, b = in && p.bias ? p.bias[n] : 0.0f;
            if (!mbar_wait(&acc_full[a], (tile >> 1) & 1, quit, p.status, kWaitAccFull)) break;
            tc_fence_after();
            // the next columns are on their way while these are stored
            uint32_t r[2][16];
            tc_ld16(tmem + a * TT + lanes, r[0]);
            tc_wait_ld();
            reg_fence16(r[0]);
#pragma unroll
            for (int c = 0; c < TT; c += 16) {
                if (c >= p.M) break;
                uint32_t(&now)[16] = r[(c / 16) & 1];
                uint32_t(&next)[16] = r[(c / 16 + 1) & 1];
                if (c + 16 < TT) tc_ld16(tmem + a * TT + c + 16 + lanes, next);
                if (SPLIT > 1) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) reinterpret_cast<uint32_t*>(ring)[(c + i) * 128 + ch] = now[i];
                } else {
                    float v[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = scaled(now[i], sh_scale[c + i], ws, b);
                    put_tokens<16>(p, v, c, t * 128 + quad * 32, vec, turn[quad]);
                }
                if (c + 16 < TT) {
                    tc_wait_ld();
                    reg_fence16(next);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[a]);
        }
    }
    __syncwarp();
    if (SPLIT > 1) {
        cluster_sync();
        if (warp >= 2) {
            // a share of the tokens out of every CTA's sums, G at a time with all their loads in flight
            constexpr int G = TT == 16 ? 4 : 8;
            const int ch = (warp & 3) * 32 + lane;
            const int64_t n = static_cast<int64_t>(t0) * 128 + ch;
            const bool in = n < p.N;
            const float ws = in ? p.w_scale[n] : 0.0f, b = in && p.bias ? p.bias[n] : 0.0f;
            for (int c = static_cast<int>(rank) * G; c < p.M; c += SPLIT * G) {
                const uint32_t at = smem_u32(ring) + (c * 128 + ch) * 4;
                uint32_t sum[G] = {};
#pragma unroll
                for (int o = 0; o < SPLIT; ++o) {
                    const uint32_t from = map_rank(at, o);
#pragma unroll
                    for (int i = 0; i < G; ++i) sum[i] += load_cluster(from + i * 512);
                }
                float v[G];
#pragma unroll
                for (int i = 0; i < G; ++i) v[i] = scaled(sum[i], sh_scale[c + i], ws, b);
                put_tokens<G>(p, v, c, t0 * 128 + (warp & 3) * 32, vec, turn[warp & 3]);
            }
        }
        __syncwarp();
        cluster_sync();                    // (the others' sums are read until here)
    } else {
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        free_columns<1>(tmem, C::COLUMNS);
    }
}

// ---------------------------------------------------------------- many tokens

template <int NT>
struct Many {
    static constexpr int A = 128 * 128, B = NT / 2 * 128, STAGE = A + B;
    static constexpr int STAGES = 192 * 1024 / STAGE;
    static constexpr int COLUMNS = 2 * NT;
    static constexpr size_t SMEM = 1024 + static_cast<size_t>(STAGES) * STAGE;
};

// Token and channel tile of number i: token tiles innermost within groups of kGroup of them,
// so that what the pairs work on at a time shares few of both.
constexpr int kGroup = 16;
__device__ __forceinline__ void tile_of(int64_t i, int mt, int nt, int& m, int& n)
{
    const int64_t per = static_cast<int64_t>(kGroup) * nt;
    const int g = static_cast<int>(i / per), rest = static_cast<int>(i - g * per);
    const int rows = min(kGroup, mt - g * kGroup);
    n = rest / rows;
    m = g * kGroup + rest - n * rows;
}

// SPLIT > 1: a cluster of that many pairs cuts the K of one tile.
template <int NT, int SPLIT>
__global__ void __launch_bounds__(kManyThreads, 1) int8_many_kernel(const __grid_constant__ Int8GemmParams p, const int align)
{
    using C = Many<NT>;
    constexpr int S = C::STAGES;
    static_assert(SPLIT == 1 || NT * 128 * 4 <= S * C::STAGE, "the sums of a split tile lie where the ring was");
    extern __shared__ uint8_t raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t full[S], empty[S], acc_full[2], acc_empty[2], done;
    __shared__ uint32_t tmem_at;
    __shared__ int abort_flag;
    __shared__ __align__(16) float sh_ws[2][NT], sh_b[2][NT];
    __shared__ __align__(16) uint16_t turn[8][32][40];       // a warp's 32 x 32 outputs on their way to rows

    const int warp = warp_id(), lane = lane_id();
    const uint32_t cta = cluster_rank(), rank = cta & 1, lead = cta & ~1u;       // in the pair; its first CTA
    const int part = static_cast<int>(cta >> 1);
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 16);                    // eight warps of each CTA
        }
        mbar_init(&done, 1);
        abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&p.tm_w);
        tma_prefetch_desc(&p.tm_a);
    }
    if (warp == 1) alloc_columns<2>(&tmem_at, C::COLUMNS);
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    volatile int* quit = &abort_flag;

    const int mt = (p.M + 255) / 256, nt = (p.N + NT - 1) / NT, KB = (p.K + 127) / 128;
    const int64_t tiles = static_cast<int64_t>(mt) * nt;
    const int pairs = gridDim.x / (2 * SPLIT), pair = blockIdx.x / (2 * SPLIT);
    const int kb0 = part * KB / SPLIT, kb1 = (part + 1) * KB / SPLIT;

    if (warp == 0) {
        if (lane == 0) {
            const uint64_t stay = policy_evict_last();
            pdl_wait();
            int64_t it = 0;
            bool ok = true;
            for (int64_t t = pair; t < tiles && ok; t += pairs) {
                int m, n;
                tile_of(t, mt, nt, m, n);
                const int a_row = m * 256 + static_cast<int>(rank) * 128, w_row = n * NT + static_cast<int>(rank) * (NT / 2);
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    const int s = static_cast<int>(it % S);
                    const int64_t round = it / S;
                    if (round > 0 && !mbar_wait(&empty[s], (round - 1) & 1, quit, p.status, kWaitEmpty)) {
                        ok = false;
                        break;
                    }
                    // the pair's first CTA counts the bytes of both
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * C::STAGE);
                    const uint32_t bar = map_rank(smem_u32(&full[s]), lead);
                    load_pair(ring + s * C::STAGE, &p.tm_a, bar, kb * 128, a_row, stay);
                    load_pair(ring + s * C::STAGE + C::A, &p.tm_w, bar, kb * 128, w_row, stay);
                }
            }
            pdl_launch_dependents();
            // every copy and every arrival at this CTA's barriers is in before it ends
            for (int64_t i = it > S ? it - S : 0; i < it; ++i)
                mbar_wait(&empty[i % S], (i / S) & 1, quit, p.status, kWaitDrain);
            if (*quit && rank == 0) {      // (the first CTA's barriers count both CTAs' copies)
                const uint64_t deadline = global_timer_ns() + kWaitLimitNs;
                for (int64_t i = it > S ? it - S : 0; i < it; ++i) settle(&full[i % S], (i / S) & 1, deadline);
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            constexpr uint32_t idesc = idesc_i8(256, NT);
            const uint32_t base = smem_u32(ring);
            int64_t it = 0, tile = 0;
            bool ok = true;
            for (int64_t t = pair; t < tiles && ok; t += pairs, ++tile) {
                const int a = tile & 1;
                if (tile >= 2 && !mbar_wait(&acc_empty[a], ((tile >> 1) - 1) & 1, quit, p.status, kWaitAccEmpty)) break;
                tc_fence_after();
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    const int s = static_cast<int>(it % S);
                    if (!mbar_wait(&full[s], (it / S) & 1, quit, p.status, kWaitFull)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t ad = smem_desc_sw128(base + s * C::STAGE), wd = smem_desc_sw128(base + s * C::STAGE + C::A);
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma_i8<2>(tmem + a * NT, ad + 2 * k, wd + 2 * k, idesc, kb > kb0 || k > 0);
                    commit_pair(&empty[s], lead);
                }
                if (ok) commit_pair(&acc_full[a], lead);
            }
            if (*quit) {                   // (tensor memory is given back below)
                asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&done))
                             : "memory");
                settle(&done, 0, global_timer_ns() + kWaitLimitNs);
            }
        }
    } else {
        const int quad = warp & 3;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        pdl_wait();
        int64_t tile = 0;
        bool ok = true;                    // (a warp whose wait ran out still comes to the others' barrier)
        // the row's scale and, one channel a thread, the channels', loaded a tile ahead
        float row_scale, ws, b;
        const auto load = [&](int64_t t) {
            int m, nn;
            tile_of(t, mt, nt, m, nn);
            const int64_t row = static_cast<int64_t>(m) * 256 + rank * 128 + quad * 32 + lane;
            const int c = threadIdx.x - 64;
            const int64_t n = static_cast<int64_t>(nn) * NT + c;
            const bool there = c < NT && n < p.N;
            row_scale = row < p.M ? p.a_scale[row] : 0.0f;
            ws = there ? p.w_scale[n] : 0.0f;
            b = there && p.bias ? p.bias[n] : 0.0f;
        };
        if (pair < tiles) load(pair);
        for (int64_t t = pair; t < tiles; t += pairs, ++tile) {
            int m, nn;
            tile_of(t, mt, nt, m, nn);
            const int a = tile & 1;
            const int64_t row = static_cast<int64_t>(m) * 256 + rank * 128 + quad * 32 + lane;
            const bool in = row < p.M;
            const float s = row_scale;
            // (the other tile's warps still read the other buffer)
            if (const int c = threadIdx.x - 64; c < NT) {
                sh_ws[a][c] = ws;
                sh_b[a][c] = b;
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (t + pairs < tiles) load(t + pairs);
            ok = ok && mbar_wait(&acc_full[a], (tile >> 1) & 1, quit, p.status, kWaitAccFull);
            if (!ok) continue;
            tc_fence_after();
            // this warp's half of the channels, the next 32 on their way while these are stored
            const int c0 = (warp - 2) / 4 * (NT / 2);
            uint32_t r[2][32];
            load_columns32(tmem + a * NT + c0 + lanes, r[0]);
            tc_wait_ld();
            settle32(r[0]);
#pragma unroll
            for (int k = 0; k < NT / 64; ++k) {
                const int c = c0 + 32 * k;
                uint32_t(&now)[32] = r[k & 1];
                uint32_t(&next)[32] = r[(k + 1) & 1];
                if (k + 1 < NT / 64) {
                    load_columns32(tmem + a * NT + c + 32 + lanes, next);
                } else {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_remote(map_rank(smem_u32(&acc_empty[a]), lead));
                }
                if (SPLIT > 1) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) reinterpret_cast<uint32_t*>(ring)[(c + i) * 128 + quad * 32 + lane] = now[i];
                } else {
                    put32(p, now, nn * NT + c, row, in, s, sh_ws[a] + c, sh_b[a] + c, align, turn[warp - 2]);
                }
                if (k + 1 < NT / 64) {
                    tc_wait_ld();
                    settle32(next);
                }
            }
        }
    }
    __syncwarp();
    cluster_sync();
    if (SPLIT > 1) {
        // a share of the channels out of every pair's sums
        if (warp >= 2) {
            int m, nn;
            tile_of(pair, mt, nt, m, nn);
            const int quad = warp & 3;
            const int64_t row = static_cast<int64_t>(m) * 256 + rank * 128 + quad * 32 + lane;
            const bool in = row < p.M;
            const float s = in ? p.a_scale[row] : 0.0f;
#pragma unroll 1
            for (int k = part * (NT / 32) / SPLIT + (warp - 2) / 4; k < (part + 1) * (NT / 32) / SPLIT; k += 2) {
                const int c = 32 * k;
                uint32_t r[32] = {};
                const uint32_t at = smem_u32(ring) + (c * 128 + quad * 32 + lane) * 4;
#pragma unroll
                for (int o = 0; o < SPLIT; ++o) {
                    const uint32_t from = map_rank(at, 2 * o + rank);
#pragma unroll
                    for (int i = 0; i < 32; ++i) r[i] += load_cluster(from + i * 512);
                }
                put32(p, r, nn * NT + c, row, in, s, sh_ws[0] + c, sh_b[0] + c, align, turn[warp - 2]);
            }
        }
        __syncwarp();
        cluster_sync();                    // (the others' sums are read until here)
    }
    if (warp == 1) {
        tc_fence_after();
        free_columns<2>(tmem, C::COLUMNS);
    }
}

// ---------------------------------------------------------------- launch

template <typename Kern, typename... Args>
cudaError_t launch(Kern kern, int grid, int threads, int cluster, size_t smem, cudaStream_t stream, bool pdl, const Args&... args)
{
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

template <int TT>
cudaError_t launch_few(const Int8GemmParams& p, int split, int sms, cudaStream_t stream, bool pdl)
{
    const int tiles = (p.N + 127) / 128;
    constexpr size_t smem = Few<TT>::SMEM;
    const int vec = reinterpret_cast<uintptr_t>(p.y) % 16 == 0 && p.ldy % 8 == 0;
    switch (split) {
        case 8: return launch(int8_few_kernel<TT, 8>, tiles * 8, kThreads, 8, smem, stream, pdl, p, vec);
        case 6: return launch(int8_few_kernel<TT, 6>, tiles * 6, kThreads, 6, smem, stream, pdl, p, vec);
        case 3: return launch(int8_few_kernel<TT, 3>, tiles * 3, kThreads, 3, smem, stream, pdl, p, vec);
        case 4: return launch(int8_few_kernel<TT, 4>, tiles * 4, kThreads, 4, smem, stream, pdl, p, vec);
        case 2: return launch(int8_few_kernel<TT, 2>, tiles * 2, kThreads, 2, smem, stream, pdl, p, vec);
        default: return launch(int8_few_kernel<TT, 1>, std::min(tiles, 2 * sms), kThreads, 1, smem, stream, pdl, p, vec);
    }
}

template <int NT>
cudaError_t launch_many(const Int8GemmParams& p, int split, int64_t tiles, int align, int sms, cudaStream_t stream, bool pdl)
{
    constexpr size_t smem = Many<NT>::SMEM;
    const int n = static_cast<int>(std::min<int64_t>(tiles, split > 1 ? tiles : sms / 2));
    switch (split) {
        case 4: return launch(int8_many_kernel<NT, 4>, 8 * n, kManyThreads, 8, smem, stream, pdl, p, align);
        case 3: return launch(int8_many_kernel<NT, 3>, 6 * n, kManyThreads, 6, smem, stream, pdl, p, align);
        case 2: return launch(int8_many_kernel<NT, 2>, 4 * n, kManyThreads, 4, smem, stream, pdl, p, align);
        default: return launch(int8_many_kernel<NT, 1>, 2 * n, kManyThreads, 2, smem, stream, pdl, p, align);
    }
}

// Clusters of KERN that the current device holds at a time with `per_sm` CTAs an SM; 0 where that cannot be told.  (For
// kernels with tensor memory the runtime counts one CTA an SM.  Two of the few-token kernel run: 40 clusters of six
// take one wave, 24.5 us, 40 of eight do not, 29.4.)
template <auto KERN>
int resident(int cluster, int threads, size_t smem, int per_sm)
{
    constexpr int kDevices = 64;
    static std::atomic<int> known[kDevices];                  // plus one
    int dev = 0, n = 0, counted = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) return 0;
    if ((n = known[dev].load(std::memory_order_relaxed)) > 0) return n - 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, KERN, &cfg) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&counted, KERN, threads, smem) != cudaSuccess || counted < 1) {
        cudaGetLastError();
        return 0;
    }
    n = n / counted * per_sm;
    known[dev].store(n + 1, std::memory_order_relaxed);
    return n;
}

template <int TT, int SPLIT>
bool few_fits(int64_t tiles)
{
    return tiles <= resident<int8_few_kernel<TT, SPLIT>>(SPLIT, kThreads, Few<TT>::SMEM, 2);
}

// How many CTAs cut a tile's K: as many as are resident with the tiles there are, while each keeps enough blocks of 128
// to be worth its share of the join -- two where the cut still leaves SMs idle, ten where SMs would hold two CTAs (with
// fewer, 12000 x 2048 of one token 8.5 us uncut, 8.2 in two, 11.1 in three; 5120 x 27648 61.5 uncut, 24.8 in four,
// 24.5 in six; 1280 x 5120 13.6 uncut, 5.4 in eight).
template <int TT>
int few_split(int64_t tiles, int64_t kb, int sms)
{
    const auto worth = [&](int s) { return kb >= (tiles * s <= sms ? 2 : 10) * s; };
    if (kb < 8) return 1;
    if (worth(8) && few_fits<TT, 8>(tiles)) return 8;
    if (worth(6) && few_fits<TT, 6>(tiles)) return 6;
    if (worth(4) && few_fits<TT, 4>(tiles)) return 4;
    if (worth(3) && few_fits<TT, 3>(tiles)) return 3;
    if (worth(2) && few_fits<TT, 2>(tiles)) return 2;
    return 1;
}

template <int NT>
bool many_fits(int64_t tiles, int split)
{
    switch (split) {
        case 1: return true;
        case 2: return tiles <= resident<int8_many_kernel<NT, 2>>(4, kManyThreads, Many<NT>::SMEM, 1);
        case 3: return tiles <= resident<int8_many_kernel<NT, 3>>(6, kManyThreads, Many<NT>::SMEM, 1);
        default: return tiles <= resident<int8_many_kernel<NT, 4>>(8, kManyThreads, Many<NT>::SMEM, 1);
    }
}

}  // namespace

Int8Plan int8_plan(int64_t M, int64_t N, int64_t K, int sms)
{
    Int8Plan r{};
    const int64_t kb = (K + 127) / 128;
    r.many = M > kFewTokens;
    if (!r.many) {
        const int64_t tiles = (N + 127) / 128;
        r.tt = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
        r.split = r.tt == 16   ? few_split<16>(tiles, kb, sms)
                  : r.tt == 32 ? few_split<32>(tiles, kb, sms)
                  : r.tt == 64 ? few_split<64>(tiles, kb, sms)
                               : few_split<128>(tiles, kb, sms);
        r.w_rows = 128;
        r.a_rows = r.tt;
        return r;
    }
    // The quickest by what each costs (microseconds measured on B200, 9 shapes of weights x 200 to 1024 tokens, and K 128
    // to 2048 of 4,096 x 8192): starting and storing a tile, 0.26 or 0.31 a block of 128 of K, in every further wave of tiles
    // that or storing the tile before, and a cut tile's join.
    constexpr float kStart[2] = {5.7f, 6.7f}, kBlock[2] = {0.26f, 0.31f}, kStore[2] = {1.7f, 3.2f};
    constexpr float kJoin[2][4] = {{0.0f, 0.9f, 1.8f, 2.0f}, {0.0f, 3.7f, 6.0f, 7.0f}};
    const int64_t mt = (M + 255) / 256;
    float best = 0.0f;
    for (int wide = 1; wide >= 0; --wide)
        for (int split = 1; split <= 4; ++split) {
            const int nt = wide ? 256 : 128;
            const int64_t tiles = mt * ((N + nt - 1) / nt), waves = (tiles * split + sms / 2 - 1) / (sms / 2);
            if (split > 1 && (waves > 1 || kb < 2 * split || !(wide ? many_fits<256>(tiles, split) : many_fits<128>(tiles, split))))
                continue;
            const float blocks = kBlock[wide] * static_cast<float>((kb + split - 1) / split);
            const float cost = kStart[wide] + blocks + static_cast<float>(waves - 1) * std::max(blocks, kStore[wide]) + kJoin[wide][split - 1];
            if (r.nt == 0 || cost < best) {
                best = cost;
                r.nt = nt;
                r.split = split;
            }
        }
    r.w_rows = r.nt / 2;
    r.a_rows = 128;
    return r;
}

cudaError_t launch_int8_gemm(const Int8GemmParams& p, const Int8Plan& plan, int sms, cudaStream_t stream, bool pdl)
{
    if (plan.many) {
        const int64_t mt = (p.M + 255) / 256, nt = (p.N + plan.nt - 1) / plan.nt;
        // the widest store that each row's outputs suit
        const auto fits = [&](uintptr_t a) { return reinterpret_cast<uintptr_t>(p.y) % a == 0 && 2 * p.ldy % a == 0; };
        const int align = fits(32) ? 32 : fits(16) ? 16 : fits(8) ? 8 : fits(4) ? 4 : 2;
        if (plan.nt == 256) return launch_many<256>(p, plan.split, mt * nt, align, sms, stream, pdl);
        return launch_many<128>(p, plan.split, mt * nt, align, sms, stream, pdl);
    }
    switch (plan.tt) {
        case 16: return launch_few<16>(p, plan.split, sms, stream, pdl);
        case 32: return launch_few<32>(p, plan.split, sms, stream, pdl);
        case 64: return launch_few<64>(p, plan.split, sms, stream, pdl);
        default: return launch_few<128>(p, plan.split, sms, stream, pdl);
    }
}

}  // namespace w4a8
