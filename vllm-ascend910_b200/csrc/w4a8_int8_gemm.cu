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
// few (up to kFewTokens tokens): the weights' bytes bound it.  A tile is 128 channels (the
//   MMA's rows) by 16, 32, 64 or 128 tokens (its columns), so that few tokens waste little.
//   Two CTAs an SM, each with a ring of 96 KB in flight.  With fewer tiles than CTAs, a
//   cluster cuts a tile's K: each CTA leaves its sums in shared memory and adds up
//   a share of the tokens out of all of them over distributed shared memory.
// many: the tensor pipe bounds it.  A pair of CTAs (cta_group::2) owns 256 tokens x 256 (or
//   128) channels: each brings 128 tokens and half of the channels, one of them issues for
//   both.  Two accumulators fill tensor memory, one in work while the other is stored.
//
// Each wait for a barrier is bounded; one that runs out ends the CTA's roles and leaves a code in
// the workspace's status word.
#include <algorithm>

#include "w4a8_common.cuh"
#include "w4a8_kernels.h"

namespace w4a8 {

namespace {

constexpr int kThreads = 192;              // producer, issuer, four epilogue warps
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
__device__ __forceinline__ void commit_pair(uint64_t* bar)
{
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
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
__device__ __forceinline__ void arrive_remote(uint32_t bar)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
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

// ---------------------------------------------------------------- few tokens

template <int TT>
struct Few {
    static constexpr int STAGE = 16384 + TT * 128;
    static constexpr int STAGES = 96 * 1024 / STAGE > 6 ? 6 : 96 * 1024 / STAGE;
    static constexpr int COLUMNS = 2 * TT < 32 ? 32 : 2 * TT;
    static constexpr size_t SMEM = 1024 + static_cast<size_t>(STAGES) * STAGE;
};

template <int TT, int SPLIT>
__global__ void __launch_bounds__(kThreads, 2) int8_few_kernel(const __grid_constant__ Int8GemmParams p)
{
    using C = Few<TT>;
    constexpr int S = C::STAGES;
    static_assert(TT * 128 * 4 <= S * C::STAGE, "the sums of a split tile lie where the ring was");
    extern __shared__ uint8_t raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t full[S], empty[S], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_at;
    __shared__ int abort_flag;
    __shared__ float sh_scale[TT];

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
            uint16_t* y = p.y + n;
            for (int c = 0; c < TT && c < p.M; c += 16) {
                uint32_t r[16];
                tc_ld16(tmem + a * TT + c + lanes, r);
                tc_wait_ld();
                reg_fence16(r);
                if (SPLIT > 1) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) reinterpret_cast<uint32_t*>(ring)[(c + i) * 128 + ch] = r[i];
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (in && c + i < p.M)
                            y[(c + i) * p.ldy] = f32_to_bf16_bits(scaled(r[i], sh_scale[c + i], ws, b));
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
            const int ch = (warp & 3) * 32 + lane;
            const int64_t n = static_cast<int64_t>(t0) * 128 + ch;
            if (n < p.N) {
                const float ws = p.w_scale[n], b = p.bias ? p.bias[n] : 0.0f;
                for (int c = rank; c < p.M; c += SPLIT) {
                    const uint32_t at = smem_u32(ring) + (c * 128 + ch) * 4;
                    uint32_t sum = 0;
#pragma unroll
                    for (int o = 0; o < SPLIT; ++o) sum += load_cluster(map_rank(at, o));
                    p.y[c * p.ldy + n] = f32_to_bf16_bits(scaled(sum, sh_scale[c], ws, b));
                }
            }
        }
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

template <int NT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    int8_many_kernel(const __grid_constant__ Int8GemmParams p, const int align)
{
    using C = Many<NT>;
    constexpr int S = C::STAGES;
    extern __shared__ uint8_t raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t full[S], empty[S], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_at;
    __shared__ int abort_flag;
    __shared__ uint16_t turn[4][32][34];                     // a warp's 32 x 32 outputs on their way to rows

    const int warp = warp_id(), lane = lane_id();
    const uint32_t rank = cluster_rank();
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 8);                     // four warps of each CTA
        }
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
    const int pairs = gridDim.x / 2, pair = blockIdx.x / 2;

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
                for (int kb = 0; kb < KB; ++kb, ++it) {
                    const int s = static_cast<int>(it % S);
                    const int64_t round = it / S;
                    if (round > 0 && !mbar_wait(&empty[s], (round - 1) & 1, quit, p.status, kWaitEmpty)) {
                        ok = false;
                        break;
                    }
                    // the pair's first CTA counts the bytes of both
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * C::STAGE);
                    const uint32_t bar = map_rank(smem_u32(&full[s]), 0);
                    load_pair(ring + s * C::STAGE, &p.tm_a, bar, kb * 128, a_row, stay);
                    load_pair(ring + s * C::STAGE + C::A, &p.tm_w, bar, kb * 128, w_row, stay);
                }
            }
            pdl_launch_dependents();
            // every copy and every arrival at this CTA's barriers is in before it ends
            for (int64_t i = it > S ? it - S : 0; i < it; ++i)
                mbar_wait(&empty[i % S], (i / S) & 1, quit, p.status, kWaitDrain);
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
                for (int kb = 0; kb < KB; ++kb, ++it) {
                    const int s = static_cast<int>(it % S);
                    if (!mbar_wait(&full[s], (it / S) & 1, quit, p.status, kWaitFull)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t ad = smem_desc_sw128(base + s * C::STAGE), wd = smem_desc_sw128(base + s * C::STAGE + C::A);
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma_i8<2>(tmem + a * NT, ad + 2 * k, wd + 2 * k, idesc, kb > 0 || k > 0);
                    commit_pair(&empty[s]);
                }
                if (ok) commit_pair(&acc_full[a]);
            }
        }
    } else {
        const int quad = warp & 3;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        pdl_wait();
        int64_t tile = 0;
        for (int64_t t = pair; t < tiles; t += pairs, ++tile) {
            int m, nn;
            tile_of(t, mt, nt, m, nn);
            const int a = tile & 1;
            const int64_t row = static_cast<int64_t>(m) * 256 + rank * 128 + quad * 32 + lane;
            const bool in = row < p.M;
            const float s = in ? p.a_scale[row] : 0.0f;
            uint16_t* y = p.y + row * p.ldy;
            if (!mbar_wait(&acc_full[a], (tile >> 1) & 1, quit, p.status, kWaitAccFull)) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < NT; c += 32) {
                const int n = nn * NT + c;
                uint32_t r[32];
                load_columns32(tmem + a * NT + c + lanes, r);
                tc_wait_ld();
                settle32(r);
                if (c + 32 >= NT) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_remote(map_rank(smem_u32(&acc_empty[a]), 0));
                }
                uint32_t o[16];
                const bool whole = n + 32 <= p.N;
                if (whole && align >= 16) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 ws = *reinterpret_cast<const float4*>(p.w_scale + n + i);
                        const float4 b = p.bias ? *reinterpret_cast<const float4*>(p.bias + n + i) : make_float4(0, 0, 0, 0);
                        o[i / 2] = two(scaled(r[i], s, ws.x, b.x), scaled(r[i + 1], s, ws.y, b.y));
                        o[i / 2 + 1] = two(scaled(r[i + 2], s, ws.z, b.z), scaled(r[i + 3], s, ws.w, b.w));
                    }
                    if (!in) continue;
                    if (align >= 32) {
#pragma unroll
                        for (int i = 0; i < 16; i += 8)      // 32 bytes: a whole sector a thread
                            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(y + n + 2 * i), "r"(o[i]),
                                         "r"(o[i + 1]), "r"(o[i + 2]), "r"(o[i + 3]), "r"(o[i + 4]), "r"(o[i + 5]),
                                         "r"(o[i + 6]), "r"(o[i + 7])
                                         : "memory");
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; i += 4)
                            *reinterpret_cast<uint4*>(y + n + 2 * i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                } else if (n < p.N) {
                    // rows that suit no vector, or their end: a lane a channel, row by row
                    const int col = min(n + lane, p.N - 1);
                    const float mws = p.w_scale[col], mb = p.bias ? p.bias[col] : 0.0f;
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float ws0 = __shfl_sync(0xffffffffu, mws, i), ws1 = __shfl_sync(0xffffffffu, mws, i + 1);
                        const float b0 = __shfl_sync(0xffffffffu, mb, i), b1 = __shfl_sync(0xffffffffu, mb, i + 1);
                        *reinterpret_cast<uint32_t*>(&turn[quad][lane][i]) = two(scaled(r[i], s, ws0, b0), scaled(r[i + 1], s, ws1, b1));
                    }
                    __syncwarp();
                    const int64_t row0 = row - lane;
                    for (int i = 0; i < 32 && row0 + i < p.M; ++i)
                        if (n + lane < p.N) p.y[(row0 + i) * p.ldy + n + lane] = turn[quad][i][lane];
                    __syncwarp();
                }
            }
        }
    }
    __syncwarp();
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        free_columns<2>(tmem, C::COLUMNS);
    }
}

// ---------------------------------------------------------------- launch

template <typename Kern, typename... Args>
cudaError_t launch(Kern kern, int grid, int cluster, size_t smem, cudaStream_t stream, bool pdl, const Args&... args)
{
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
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
    switch (split) {
        case 8: return launch(int8_few_kernel<TT, 8>, tiles * 8, 8, smem, stream, pdl, p);
        case 4: return launch(int8_few_kernel<TT, 4>, tiles * 4, 4, smem, stream, pdl, p);
        case 2: return launch(int8_few_kernel<TT, 2>, tiles * 2, 2, smem, stream, pdl, p);
        default: return launch(int8_few_kernel<TT, 1>, std::min(tiles, 2 * sms), 1, smem, stream, pdl, p);
    }
}

}  // namespace

Int8Plan int8_plan(int64_t M, int64_t N, int64_t K, int sms)
{
    Int8Plan r{};
    r.many = M > kFewTokens;
    if (r.many) {
        r.nt = 256;
        r.w_rows = r.nt / 2;
        r.a_rows = 128;
        return r;
    }
    r.tt = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
    const int64_t tiles = (N + 127) / 128, kb = (K + 127) / 128;
    r.split = 1;
    while (r.split < 8 && tiles * r.split * 2 <= 2 * sms && kb >= 4 * r.split) r.split *= 2;
    r.w_rows = 128;
    r.a_rows = r.tt;
    return r;
}

cudaError_t launch_int8_gemm(const Int8GemmParams& p, const Int8Plan& plan, int sms, cudaStream_t stream, bool pdl)
{
    if (plan.many) {
        const int64_t mt = (p.M + 255) / 256, nt = (p.N + plan.nt - 1) / plan.nt;
        const int pairs = static_cast<int>(std::min<int64_t>(mt * nt, sms / 2));
        // the widest store that each row's outputs suit, where 16-byte loads suit the channels' scales
        const auto fits = [&](uintptr_t a) { return reinterpret_cast<uintptr_t>(p.y) % a == 0 && 2 * p.ldy % a == 0; };
        const bool loads = reinterpret_cast<uintptr_t>(p.w_scale) % 16 == 0 && reinterpret_cast<uintptr_t>(p.bias) % 16 == 0;
        const int align = !loads ? 2 : fits(32) ? 32 : fits(16) ? 16 : 2;
        // (the kernel names its cluster itself)
        return plan.nt == 256 ? launch(int8_many_kernel<256>, 2 * pairs, 1, Many<256>::SMEM, stream, pdl, p, align)
                              : launch(int8_many_kernel<128>, 2 * pairs, 1, Many<128>::SMEM, stream, pdl, p, align);
    }
    switch (plan.tt) {
        case 16: return launch_few<16>(p, plan.split, sms, stream, pdl);
        case 32: return launch_few<32>(p, plan.split, sms, stream, pdl);
        case 64: return launch_few<64>(p, plan.split, sms, stream, pdl);
        default: return launch_few<128>(p, plan.split, sms, stream, pdl);
    }
}

}  // namespace w4a8
