// w4a8_attention_many.cu -- attention over the paged 8-bit cache for sequences
// with many query rows (prompts, chunks), on the 5th-generation tensor core.
// The mathematics and the fp16 operand ranges are those of w4a8_attention.cu.
//
// Rows of one kv head are packed (query token x query head of the group) into
// tiles of 256: two halves A and B of 128 rows, one TMEM lane each.  The cache
// is walked in blocks of 64 tokens:
//
//   S_X = Q_X K^T          tcgen05.mma f16, M 128, N 64, both operands in smem
//   P_X = exp2(...)        softmax warps, a thread per row, from and to TMEM
//   O_X += P_X V           A operand = P_X in TMEM, N = D, V K-row-major in smem
//
// Roles (one CTA per SM):
//   warps 0-3, 4-7   softmax of half A, B: row maximum, exponentials, weights, sum;
//                    their rows' queries to fp16 in smem, and the output rows
//   warps 8-11       converters: a block's codes from smem, exact fp16 into the
//                    swizzled operand layout
//   warps 12, 13     issue the MMAs of half A, B
//   warp 14          fetches: bulk copies of codes three blocks ahead, page scales
//                    (warp 15 fills the warpgroup)
// One issuer for both halves was measured first: its chain of waits and commits
// (about 100 cycles each) set the pace at 1,900 cycles a block with all other work
// taken out.  Converters that loaded codes into registers themselves, one block
// ahead, were the pace at 3,200 cycles a block of a prompt of 8,192 tokens (latency
// of loads, addresses and shuffles beside the conversion); fed from smem it is the
// softmax's, 2,400.
// TMEM holds S of each half (64 columns), two P of each half (32 columns) and O (D
// columns).  S is free as soon as the softmax has it in registers, so Q K^T of block
// j + 1 runs while the softmax of block j works; P of a block is kept until its PV
// has read it, two blocks deep.  Neither product waits for the other (P over S in
// two buffers, measured first, made every Q K^T wait for a PV just issued).
//
// The reference maximum of a row moves only when a block exceeds it by more than
// 2^1.9 (weights stay below 2^15.9, inside fp16), and then to 2^2 above what was
// seen: a rescale of O in TMEM is rare instead of once a block (35 in 547 blocks of
// random data), at the price of two of the 28 binades below the largest weight that
// keep all 11 bits.  Exponentials by the old reference beside the maximum, done again
// where it has to move, were no faster (227 against 219 us for three prompts).
//
// Work: units of (row tile, 64-token block), causally pruned, and a few for each
// tile's beginning and end, in one list; every CTA takes an equal contiguous
// share, so chunks over long contexts and mixed batches fill the machine alike.  Tiles
// split between CTAs leave fp32 parts that attend_many_join_kernel adds in order (a
// join by the last CTA to finish, as attend_few_kernel does, was slower for long
// prompts: 733 against 807 TFLOP/s at 8,192 tokens).
//
// Bounds per 256 x 64 step at D = 128: 1024 tensor cycles, 1024 cycles of the
// exponential unit (16 / clock / SM), about 1,500 cycles of shared memory (128 KB of
// operands, 64 KB of codes and their conversion), about 1,200 issue slots per scheduler.
// Measured (B200, 40 query heads on 8 of 128): 2,400 cycles a step, and 10,000 for a
// tile's queries and output; three prompts of 1,364-1,668 tokens behind 179-791 178 us, 692
// TFLOP/s; one prompt of 2,048, 4,096 and 8,192 tokens 77, 215 and 721 us, 554, 798 and 954
// TFLOP/s.  For three seconds on end 183, 76, 227 and 791 us, at 1,912, 1,965, 1,867 and 1,800 MHz:
// all but the 2,048 reach the board's power limit.
#include <algorithm>

#include "w4a8_attention.cuh"

namespace w4a8 {

namespace {

constexpr int kBlk = 64;                   // tokens per step
constexpr int kRows = 256;                 // packed rows per tile
constexpr int kNS = 3;                     // K and V stages
constexpr int kNR = 3;                     // blocks of codes on their way
static_assert(kNR <= kNS, "the fetching warp arrives on a K stage's barrier for no block but its next");
constexpr int kScaleRing = 16;             // blocks whose page scales are kept
constexpr int kManyThreads = 16 * 32;      // whole warpgroups: setmaxnreg moves registers between them
constexpr int kConvWarp = 8, kMmaWarp = 12, kFetchWarp = 14;
constexpr int kRegsSoft = 184, kRegsRest = 72;      // 2 warpgroups of each
static_assert(2 * kRegsSoft + 2 * kRegsRest <= 4 * 128, "the launch allocates 128 registers a thread");
// What beginning and ending a tile costs, in blocks (work shares).  Three prompts of 1,200
// to 2,000 behind 1,300: 264, 235 and 232 us with 3, 6 and 9; one of 2,048: 95, 81 and 82;
// four times 64 tokens behind 1,000: 30.2, 30.7 and 32.7.
constexpr int kTileUnits = 6;
// A CTA's share is not cut below this.  A prompt of 100: 16.3, 16.8, 17.6 and 24.2 us with 1, 2,
// 4 and 8; 100 tokens behind 400: 21.6, 20.1 and 21.4 with 1, 2 and 4.
constexpr int kMinUnits = 2;
// What a part costs its tile's join, in blocks.  One kv head, 20 tokens at 16,000: 49 us cut to
// kMinUnits, 27.5, 27.3 and 28.0 with 0.2, 0.35 and 0.7; 200 tokens there: 40, 38.5, 37.1 and 39.
constexpr float kPartBlocks = 0.35f;
constexpr float kMargin = 2.0f;            // log2 by which a new reference exceeds the scores seen

// wait-site ids for the status word
enum { kAMmaK = 0x41, kAMmaV, kAMmaQ, kAMmaO, kAMmaP, kAMmaS, kASoftS, kASoftPv, kASoftEnd, kAConvK, kAConvV, kAConvRaw, kAFetch, kADrain };

template <int D_>
struct ManyCfg {
    static constexpr int D = D_;
    static constexpr int CH = D_ / 64;                       // 128-byte column chunks of a row
    static constexpr int Q_CHUNK = 128 * 128;                // one half's rows x 128 B
    static constexpr int Q_HALF = CH * Q_CHUNK;
    static constexpr int KV_CHUNK = kBlk * 128;
    static constexpr int KV_STAGE = CH * KV_CHUNK;
    static constexpr int OFF_K = 2 * Q_HALF;
    static constexpr int OFF_V = OFF_K + kNS * KV_STAGE;
    static constexpr int RAW_STAGE = 2 * kBlk * D_;          // codes of K, then V
    static constexpr int OFF_RAW = OFF_V + kNS * KV_STAGE;
    static constexpr int OFF_PREFIX = OFF_RAW + kNR * RAW_STAGE;
    static constexpr int TM_S = 0;                           // [half] of 64 columns
    static constexpr int TM_P = 128;                         // [half][buffer] of 32 columns
    static constexpr int TM_O = 256;                         // [half] of D columns
    static constexpr int TM_COLS = 512;
    static constexpr int PIECE = kRows * D_ * 4;
};

// P and PV phases have a barrier for each of the two buffers: every wait is for a
// phase whose predecessor on the same barrier (two blocks back) is known to be
// complete and whose successor cannot have completed, so parity tells.
struct ManyBars {
    uint64_t kfull[kNS], kempty[kNS], vfull[kNS], vempty[kNS], rfull[kNR], rempty[kNR];
    uint64_t sfull[2], sfree[2], pready[2][2], pvdone[2][2], qfull[2], ofree[2], drain[2];
    uint32_t tmem_base;
    int abort;
};

// mbar_wait for a whole warp, with one answer for all of its lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int where)
{
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, where));
}

// Page scales of a block's four 16-token granules (-1: no page).
struct __align__(16) BlockScales {
    float k[4], v[4];
    int odd;                 // a k scale is missing, zero, infinite or NaN
    int pad[3];
};

struct Start {           // where the CTA's share begins: unit `unit` of a tile
    int seq, head, tile, unit;
    long long units;
};

__device__ __forceinline__ int many_tiles(const Seq& s, int group, int least)
{
    const int rows = s.n * group;            // (at most 0x7FFF0000: checked on the host)
    return rows > least ? (rows + kRows - 1) / kRows : 0;
}

// a / b, by the several times shorter 32-bit division where that does.
__device__ __forceinline__ long long quotient(long long a, long long b)
{
    return a < 0x7FFFFFFF && b < 0x7FFFFFFF ? static_cast<uint32_t>(a) / static_cast<uint32_t>(b) : a / b;
}

// 64-token blocks that some row of tile t sees (at least one: rows that see
// nothing are written too).
__device__ __forceinline__ int many_blocks(const Seq& s, int group, int t)
{
    const int last = min(s.n - 1, static_cast<int>((static_cast<uint32_t>(t + 1) * kRows - 1) / static_cast<uint32_t>(group)));
    const int lim = min(s.pos + last, s.len - 1);
    return lim < 0 ? 1 : lim / kBlk + 1;
}

// Units of a tile in the work list: kTileUnits for its queries and output, then
// its blocks.
__device__ __forceinline__ int many_units(const Seq& s, int group, int t) { return kTileUnits + many_blocks(s, group, t); }

// A piece: blocks [b0, b1) of a tile that has nb of them.
struct Walk {
    int seq, head, tile, b0, b1, nb;
    Seq s;
    long long left;
    // False when the share has no block.
    __device__ __forceinline__ bool begin(const AttentionParams& p, const Start& st, int least)
    {
        seq = st.seq;
        head = st.head;
        tile = st.tile;
        left = st.units;
        if (left <= 0) return false;
        s = load_seq(p.c, seq);
        return cut(p, st.unit) || next(p, least);
    }
    // The blocks of the current tile from its unit u0 on that are within the share.
    __device__ __forceinline__ bool cut(const AttentionParams& p, int u0)
    {
        nb = many_blocks(s, p.group, tile);
        const int u1 = static_cast<int>(min(static_cast<long long>(kTileUnits + nb), u0 + left));
        left -= u1 - u0;
        b0 = max(u0 - kTileUnits, 0);
        b1 = max(u1 - kTileUnits, 0);
        return b1 > b0;
    }
    // Moves to the next piece; false when the share is done.
    __device__ __forceinline__ bool next(const AttentionParams& p, int least)
    {
        if (left <= 0) return false;
        if (++tile >= many_tiles(s, p.group, least)) {
            tile = 0;
            if (++head >= p.c.kv_heads) {
                head = 0;
                do {
                    if (++seq >= p.c.batch) return false;
                    s = load_seq(p.c, seq);
                } while (many_tiles(s, p.group, least) == 0);
            }
        }
        return cut(p, 0);     // (without a block it is the share's last tile)
    }
    __device__ __forceinline__ bool has_b(int group) const
    {
        return s.n * group - tile * kRows > 128;
    }
};

// Shared-memory descriptor of a row-major operand whose rows are tokens and
// whose contiguous direction is the MMA's M / N direction (128-byte swizzle):
// 64-element chunks `chunk` bytes apart, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t saddr, uint32_t chunk)
{
    uint64_t d = smem_desc_sw128(saddr);
    d &= ~(static_cast<uint64_t>(0x3FFF) << 16);
    d |= static_cast<uint64_t>((chunk >> 4) & 0x3FFFu) << 16;
    return d;
}

// f16 x f16 -> f32; b_mn: B is contiguous along N.
__host__ __device__ constexpr uint32_t idesc_f16(uint32_t M, uint32_t N, bool b_mn)
{
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((N >> 3) << 17) | ((M >> 4) << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}

// 32 lanes x 32 columns, a lane per thread of the warp.
__device__ __forceinline__ void tm_ld32(uint32_t t, uint32_t* r)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(t));
}
__device__ __forceinline__ void tm_st32(uint32_t t, const uint32_t* r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(t),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// Keeps uses of r behind the wait that precedes this call (see reg_fence16).
__device__ __forceinline__ void reg_fence32(uint32_t* r)
{
#pragma unroll
    for (int i = 0; i < 32; i += 4) reg_fence4(r + i);
}

// The largest of three scores (one instruction).
__device__ __forceinline__ float max3(float a, uint32_t b, uint32_t c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
    return r;
}
__device__ __forceinline__ float max3(uint32_t a, uint32_t b, uint32_t c) { return max3(__uint_as_float(a), b, c); }

__device__ __forceinline__ uint32_t cvt_f16x2(float lo, float hi)
{
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w)
{
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Workspace: [grid][2] Partial, [grid][2][2][256] (m, l), [grid][2] O as [D / 4][256] float4.
template <class C>
struct ManyLayout {
    static __host__ __device__ size_t ml(int grid) { return static_cast<size_t>(grid) * 2 * sizeof(Partial); }
    static __host__ __device__ size_t o(int grid) { return ml(grid) + static_cast<size_t>(grid) * 2 * 2 * kRows * 4; }
    static __host__ __device__ size_t total(int grid) { return o(grid) + static_cast<size_t>(grid) * 2 * C::PIECE; }
};

// ------------------------------------------------------------------ converters

// One 16-byte vector of codes -> 16 fp16 values, two 16-byte units at a0 and a1.
__device__ __forceinline__ void put_codes(uint32_t a0, uint32_t a1, const uint4& v)
{
    const uint32_t w[4] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u};
    sts128(a0, biased_lo(w[0]), biased_hi(w[0]), biased_lo(w[1]), biased_hi(w[1]));
    sts128(a1, biased_lo(w[2]), biased_hi(w[2]), biased_lo(w[3]), biased_hi(w[3]));
}

__device__ __forceinline__ void bulk_to(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

// One warp fetches: the codes of a block's four 16-token granules, which lie together in
// their pages, by bulk copies (lanes 0-3 K's, 4-7 V's), and the page scales.
template <class C>
__device__ __forceinline__ void fetch_role(const AttentionParams& p, ManyBars* bars, uint32_t sm, BlockScales* ring,
                                           const Start& st, int least, volatile int* abort_flag)
{
    const CacheView& cv = p.c;
    const int lane = lane_id(), gr = lane & 3, pages = static_cast<int>(cv.pages);
    const bool of_v = lane & 4;
    const int8_t* codes = of_v ? cv.v : cv.k;
    const float* scales = of_v ? cv.v_scale : cv.k_scale;
    const uint32_t to = sm + C::OFF_RAW + (of_v ? C::RAW_STAGE / 2 : 0) + gr * 16 * C::D;
    Walk a;
    bool more = a.begin(p, st, least);
    int ab = a.b0, id = -1, head = 0, base = 0;
    auto load_id = [&]() {               // a block ahead
        head = a.head;
        base = ab * kBlk + gr * 16;
        id = base < a.s.len ? cv.table[a.seq * cv.ld_table + (base >> cv.page_log2)] : -1;
    };
    if (more) load_id();
    uint32_t g = 0;
    for (; more; ++g) {
        const uint32_t sr = g % kNR;
        if (!warp_wait(&bars->rempty[sr], ((g / kNR) & 1) ^ 1, abort_flag, p.status, kAFetch)) break;
        // Where there is no page, codes come from page 0: what they are does not matter,
        // their scores are masked and their weights 0.
        const bool there = static_cast<unsigned>(id) < static_cast<unsigned>(pages);
        const int64_t ph = static_cast<int64_t>(there ? id : 0) * cv.kv_heads + head;
        const int8_t* from = codes + ((ph << cv.page_log2) + (base & (cv.page - 1))) * C::D;
        if (lane == 0) mbar_arrive_expect_tx(&bars->rfull[sr], C::RAW_STAGE);
        __syncwarp();
        if (lane < 8) bulk_to(to + sr * C::RAW_STAGE, from, 16 * C::D, &bars->rfull[sr]);
        const float sc = there ? scales[ph] : -1.0f;
        if (++ab >= a.b1) {
            more = a.next(p, least);
            ab = a.b0;
        }
        if (more) load_id();
        BlockScales& rg = ring[g % kScaleRing];
        if (lane < 8) (of_v ? rg.v : rg.k)[gr] = sc;
        // a block with a scale that is missing, zero, infinite or NaN takes the careful path
        const bool odd = __any_sync(0xffffffffu, !of_v && !(sc >= 1e-30f && sc < 1e30f));
        if (lane == 0) rg.odd = odd;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->kfull[g % kNS]);
    }
    // no copy is in flight when the block ends, whatever became of the other warps
    int own = 0;
    for (uint32_t i = g < kNR ? 0 : g - kNR; i < g; ++i) mbar_wait(&bars->rfull[i % kNR], (i / kNR) & 1, &own, p.status, kADrain);
}

template <class C>
__device__ __forceinline__ void converter_role(const AttentionParams& p, ManyBars* bars, uint32_t sm, const Start& st, int least,
                                               volatile int* abort_flag)
{
    constexpr int PER_ROW = C::D / 16;                              // vectors of a token's row
    constexpr int N = kBlk * PER_ROW / 128;                         // vectors of a thread
    constexpr int TSTEP = 128 / PER_ROW;                            // tokens between them
    static_assert(TSTEP % 8 == 0, "the swizzle is the same for a thread's vectors");
    // Lanes are dealt so that the eight lanes of a phase hit distinct banks reading and
    // writing: a token's first half of vectors and the next one's second half, or two
    // whole rows of four vectors.
    const int lane = lane_id(), w = warp_id() - kConvWarp;
    int tok0, c;
    if (PER_ROW == 8) {
        tok0 = w * 4 + (lane >> 4) * 2 + (((lane >> 2) ^ (lane >> 3)) & 1);
        c = lane & 7;
    } else {
        tok0 = w * 8 + (lane >> 2);
        c = lane & 3;
    }
    const uint32_t from = sm + C::OFF_RAW + tok0 * C::D + c * 16;
    const uint32_t row0 = sm + (c >> 2) * C::KV_CHUNK + tok0 * 128;
    const uint32_t to0 = row0 + ((((c & 3) * 2) ^ (tok0 & 7)) << 4), to1 = row0 + ((((c & 3) * 2 + 1) ^ (tok0 & 7)) << 4);
    Walk a;
    bool more = a.begin(p, st, least);
    int ab = a.b0;
    for (uint32_t g = 0; more; ++g) {
        const uint32_t sg = g % kNS, ph = (g / kNS) & 1, sr = g % kNR;
        uint4 r[N];
        if (!warp_wait(&bars->rfull[sr], (g / kNR) & 1, abort_flag, p.status, kAConvRaw)) return;
#pragma unroll
        for (int k = 0; k < N; ++k) r[k] = lds128(from + sr * C::RAW_STAGE + k * TSTEP * C::D);
        if (!warp_wait(&bars->kempty[sg], ph ^ 1, abort_flag, p.status, kAConvK)) return;
        uint32_t at = C::OFF_K + sg * C::KV_STAGE;
#pragma unroll
        for (int k = 0; k < N; ++k) put_codes(to0 + at + k * TSTEP * 128, to1 + at + k * TSTEP * 128, r[k]);
#pragma unroll
        for (int k = 0; k < N; ++k) r[k] = lds128(from + sr * C::RAW_STAGE + C::RAW_STAGE / 2 + k * TSTEP * C::D);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->kfull[sg]);
        if (!warp_wait(&bars->vempty[sg], ph ^ 1, abort_flag, p.status, kAConvV)) return;
        at = C::OFF_V + sg * C::KV_STAGE;
#pragma unroll
        for (int k = 0; k < N; ++k) put_codes(to0 + at + k * TSTEP * 128, to1 + at + k * TSTEP * 128, r[k]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(&bars->vfull[sg]);
            mbar_arrive(&bars->rempty[sr]);
        }
        if (++ab >= a.b1) {
            more = a.next(p, least);
            ab = a.b0;
        }
    }
}

// ------------------------------------------------------------------ MMA issuer

// Half x.  Stages are handed back when both halves' issuers are done with them; in
// a piece without half B its issuer follows along and hands them back at once.
template <class C>
__device__ __forceinline__ void mma_role(const AttentionParams& p, ManyBars* bars, uint32_t sm, uint32_t tbase, const int x,
                                         const Start& st, int least, volatile int* abort_flag)
{
    constexpr uint32_t idqk = idesc_f16(128, kBlk, false), idpv = idesc_f16(128, C::D, true);
    // Descriptors count 16-byte units.
    const uint64_t q_desc = smem_desc_sw128(sm + x * C::Q_HALF), k_desc = smem_desc_sw128(sm + C::OFF_K);
    const uint64_t v_desc = smem_desc_mn(sm + C::OFF_V, C::KV_CHUNK);
    const uint32_t t_s = tbase + C::TM_S + x * kBlk, t_p = tbase + C::TM_P + x * kBlk, t_o = tbase + C::TM_O + x * C::D;
    Walk a;
    bool more = a.begin(p, st, least), ok = true;
    uint32_t g = 0;                 // blocks of the CTA (K, V stages)
    uint32_t n = 0, piece = 0;      // blocks and pieces of the half
    auto wait = [&](uint64_t* b, uint32_t parity, int where) {
        ok = ok && mbar_wait(b, parity, abort_flag, p.status, where);
        return ok;
    };
    while (more && ok) {
        const int steps = a.b1 - a.b0;
        if (x == 1 && !a.has_b(p.group)) {
            for (int j = 0; j < steps && ok; ++j, ++g) {
                const uint32_t sg = g % kNS, ph = (g / kNS) & 1;
                if (!wait(&bars->kfull[sg], ph, kAMmaK)) break;
                mbar_arrive(&bars->kempty[sg]);
                if (!wait(&bars->vfull[sg], ph, kAMmaV)) break;
                mbar_arrive(&bars->vempty[sg]);
            }
            if (ok) more = a.next(p, least);
            continue;
        }
        if (!wait(&bars->qfull[x], piece & 1, kAMmaQ)) break;
        for (int j = 0; j <= steps; ++j) {
            if (j < steps) {
                const uint32_t sg = (g + j) % kNS, b = n + j;
                if (!wait(&bars->kfull[sg], ((g + j) / kNS) & 1, kAMmaK)) break;
                if (b >= 1 && !wait(&bars->sfree[x], (b - 1) & 1, kAMmaS)) break;     // the scores before have been read
                tc_fence_after();
                const uint64_t kd = k_desc + sg * (C::KV_STAGE / 16);
#pragma unroll
                for (int k = 0; k < C::D / 16; ++k)
                    mma_ss(t_s, q_desc + ((k >> 2) * C::Q_CHUNK + (k & 3) * 32) / 16,
                           kd + ((k >> 2) * C::KV_CHUNK + (k & 3) * 32) / 16, idqk, k == 0 ? 0u : 1u);
                tc_commit(&bars->sfull[x]);
                tc_commit(&bars->kempty[sg]);
            }
            if (j > 0) {
                const uint32_t sg = (g + j - 1) % kNS, b = n + j - 1;
                if (!wait(&bars->vfull[sg], ((g + j - 1) / kNS) & 1, kAMmaV)) break;
                // the piece's first PV overwrites O, whose previous output must have been read
                if (j == 1 && piece > 0 && !wait(&bars->ofree[x], (piece - 1) & 1, kAMmaO)) break;
                if (!wait(&bars->pready[x][b & 1], (b >> 1) & 1, kAMmaP)) break;
                tc_fence_after();
                const uint32_t ap = t_p + (b & 1) * (kBlk / 2);
                const uint64_t vd = v_desc + sg * (C::KV_STAGE / 16);
#pragma unroll
                for (int k = 0; k < kBlk / 16; ++k) mma_ts(t_o, ap + k * 8, vd + k * 128, idpv, j == 1 && k == 0 ? 0u : 1u);
                tc_commit(&bars->pvdone[x][b & 1]);
                tc_commit(&bars->vempty[sg]);
            }
        }
        if (!ok) break;
        g += steps;
        n += steps;
        ++piece;
        more = a.next(p, least);
    }
    // nothing of this thread's is in flight when TMEM is freed
    tc_commit(&bars->drain[x]);
    mbar_wait(&bars->drain[x], 0, abort_flag, p.status, kADrain);
}

// ------------------------------------------------------------------ softmax

template <class C>
__device__ __forceinline__ void softmax_role(const AttentionParams& p, ManyBars* bars, uint32_t sm, uint32_t tbase,
                                             BlockScales* ring, const Start& st, int least, volatile int* abort_flag)
{
    const int x = warp_id() >> 2;                               // half
    const int row = threadIdx.x & 127;                          // row within it, and TMEM lane
    const int lane = lane_id();
    const uint32_t lane_off = static_cast<uint32_t>(row & 96) << 16;
    const uint32_t t_o = tbase + lane_off + C::TM_O + x * C::D;
    const uint32_t half_sm = sm + x * C::Q_HALF;                // its queries; afterwards its output rows on their way
    constexpr int LPR = C::D / 8, RPI = 32 / LPR;               // lanes of a row's 16-byte vectors, rows per access
    const auto q_unit = [&](int r, int u) { return half_sm + (u >> 3) * C::Q_CHUNK + r * 128 + (((u & 7) ^ (r & 7)) << 4); };
    Partial* info = reinterpret_cast<Partial*>(p.ws) + 2 * blockIdx.x;
    float* ml = reinterpret_cast<float*>(p.ws + ManyLayout<C>::ml(gridDim.x)) + static_cast<size_t>(blockIdx.x) * 4 * kRows;
    float* po = reinterpret_cast<float*>(p.ws + ManyLayout<C>::o(gridDim.x) + static_cast<size_t>(blockIdx.x) * 2 * C::PIECE);
    if (threadIdx.x < 2) info[threadIdx.x] = Partial{-1, 0, 0, 0, 0};
    __syncwarp();

    Walk a;
    bool more = a.begin(p, st, least);
    uint32_t g = 0, n = 0;           // blocks of the CTA, of this half
    while (more) {
        const int steps = a.b1 - a.b0;
        if (x == 1 && !a.has_b(p.group)) {
            g += steps;
            more = a.next(p, least);
            continue;
        }
        const int pr = a.tile * kRows + x * 128 + row;          // packed row
        const bool valid = pr < a.s.n * p.group;
        const bool live = __any_sync(0xffffffffu, valid);

        // ---- this warp's 32 queries into the operand: rows come by asynchronous copies
        // (RPI rows a turn, a lane per 16 bytes), then a lane is a row: its largest
        // element to [2^13, 2^14), fp16, in place ----
        float qs = 0.0f;                                        // what turns a raw score into log2 units
        const int limit = valid ? a.s.pos + row_token(p, pr) : 0x7FFFFFFF;   // last token the row sees
        {
            // (a lane finds its own row's place; the lanes that copy the row are told)
            const int tok = valid ? row_token(p, pr) : 0;
            const int64_t place = static_cast<int64_t>(a.s.q0 + tok) * p.ldq +
                                  static_cast<int64_t>(a.head * p.group + (valid ? pr - tok * p.group : 0)) * C::D;
            const int sub = lane / LPR, ch = lane % LPR;
#pragma unroll 4
            for (int i = 0; i < 32 / RPI; ++i) {
                const int rr = i * RPI + sub;
                const uint16_t* src = p.q + __shfl_sync(0xffffffffu, place, rr) + ch * 8;
                const bool ok = pr - lane + rr < a.s.n * p.group;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(q_unit((row & 96) + rr, ch)), "l"(src), "r"(ok ? 16 : 0)
                             : "memory");
            }
            asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
            __syncwarp();
            uint32_t big = 0;
            uint4 v[LPR];
#pragma unroll
            for (int u = 0; u < LPR; ++u) {
                v[u] = lds128(q_unit(row, u));
                const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) big = max(big, max((w[e] << 16) & 0x7FFFFFFFu, w[e] & 0x7FFF0000u));
            }
            const float shrink = row_shrink(__uint_as_float(big));
#pragma unroll
            for (int u = 0; u < LPR; ++u) {
                const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
                uint32_t h[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    h[e] = cvt_f16x2(__uint_as_float(w[e] << 16) * shrink, __uint_as_float(w[e] & 0xFFFF0000u) * shrink);
                sts128(q_unit(row, u), h[0], h[1], h[2], h[3]);
            }
            qs = __fdiv_rn(p.scale_log2, shrink);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->qfull[x]);
        }
        const int min_limit = __reduce_min_sync(0xffffffffu, limit);

        float m = kNegInf, l = 0.0f, vr = kVrMin, vr_inv = kWeightOne / kVrMin;
        for (int j = 0; j < steps; ++j, ++g, ++n) {
            if (!warp_wait(&bars->sfull[x], n & 1, abort_flag, p.status, kASoftS)) return;
            if (!live) {                             // (no row of this warp's: it only keeps step)
                if (lane == 0) {
                    mbar_arrive(&bars->sfree[x]);
                    mbar_arrive(&bars->pready[x][n & 1]);
                }
                continue;
            }
            tc_fence_after();
            uint32_t s[kBlk];
            tm_ld32(tbase + lane_off + C::TM_S + x * kBlk, s);
            tm_ld32(tbase + lane_off + C::TM_S + x * kBlk + 32, s + 32);
            tc_wait_ld();
            reg_fence32(s);
            reg_fence32(s + 32);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->sfree[x]);
            const BlockScales& rg = ring[g % kScaleRing];
            const float4 rk = *reinterpret_cast<const float4*>(rg.k), rv = *reinterpret_cast<const float4*>(rg.v);
            const int t0 = (a.b0 + j) * kBlk;
            // a granule's factors of scores and of weights
            float f[4] = {rk.x * qs, rk.y * qs, rk.z * qs, rk.w * qs}, wv[4] = {rv.x, rv.y, rv.z, rv.w};
            if (rg.odd || t0 + kBlk - 1 > min_limit) {
                // A granule that this row does not see at all takes factors that
                // cannot touch it, whatever its scales are.  A zero factor would turn
                // a masked score into NaN: the smallest one changes no visible score.
                const float ks[4] = {rk.x, rk.y, rk.z, rk.w};
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const bool none = ks[b] < 0.0f || t0 + 16 * b > limit;
                    f[b] = none ? 1.0f : ks[b] != ks[b] ? ks[b] : fmaxf(f[b], 1e-37f);
                    if (none) wv[b] = 0.0f;
                    const int seen = none ? -1 : limit - t0 - 16 * b;
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (i > seen) s[16 * b + i] = 0xFF800000u;
                }
            }
            const float vmax = fmaxf(fmaxf(wv[0], wv[1]), fmaxf(wv[2], wv[3]));
            // ---- reference maximum ----
            float mx = kNegInf;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const uint32_t* x = s + 16 * b;
                float r = max3(x[0], x[1], x[2]), q = max3(x[3], x[4], x[5]);
                r = max3(r, x[6], x[7]);
                q = max3(q, x[8], x[9]);
                r = max3(r, x[10], x[11]);
                q = max3(q, x[12], x[13]);
                r = max3(r, x[14], x[15]);
                mx = fmaxf(mx, fmaxf(r, q) * f[b]);
            }
            if (__any_sync(0xffffffffu, mx > m + kSlack || vmax > vr)) {
                const float mn = fmaxf(m, mx + kMargin), vn = fmaxf(vr, pow2_above(vmax));
                const float al = mn == kNegInf ? 1.0f : ex2(m - mn), av = al * __fdiv_rn(vr, vn);
                m = mn;
                l *= al;
                vr = vn;
                vr_inv = __fdiv_rn(kWeightOne, vr);
                if (j > 0) {
                    if (!warp_wait(&bars->pvdone[x][(n - 1) & 1], ((n - 1) >> 1) & 1, abort_flag, p.status, kASoftPv)) return;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < C::D; c += 64) {
                        uint32_t o[64];
                        tm_ld32(t_o + c, o);
                        tm_ld32(t_o + c + 32, o + 32);
                        tc_wait_ld();
                        reg_fence32(o);
                        reg_fence32(o + 32);
#pragma unroll
                        for (int i = 0; i < 64; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * av);
                        tm_st32(t_o + c, o);
                        tm_st32(t_o + c + 32, o + 32);
                    }
                    tc_wait_st();
                }
            }
            // ---- weights ----
            const float neg_m = m == kNegInf ? 0.0f : -m;
            uint32_t pk[kBlk / 2];
            uint64_t sum[2] = {0, 0};
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const uint64_t f2 = pair2(f[b], f[b]), m2 = pair2(neg_m, neg_m);
                const float w = wv[b] * vr_inv;
                const uint64_t w2 = pair2(w, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int e = 16 * b + 2 * i;
                    float lo, hi;
                    unpair2(f2_fma(pair2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), f2, m2), lo, hi);
                    const uint64_t pp = pair2(ex2(lo), ex2(hi));
                    sum[i & 1] = f2_add(sum[i & 1], pp);
                    unpair2(f2_mul(pp, w2), lo, hi);
                    pk[8 * b + i] = cvt_f16x2(lo, hi);
                }
            }
            float lo, hi;
            unpair2(f2_add(sum[0], sum[1]), lo, hi);
            l += lo + hi;
            // This P buffer is free: the scores' barrier says that every product issued before
            // them is done, the PV of two blocks back among them.
            tm_st32(tbase + lane_off + C::TM_P + (x * 2 + (n & 1)) * (kBlk / 2), pk);
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->pready[x][n & 1]);
        }

        // ---- the piece's output ----
        if (!warp_wait(&bars->pvdone[x][(n - 1) & 1], ((n - 1) >> 1) & 1, abort_flag, p.status, kASoftEnd)) return;
        if (live) {
            tc_fence_after();
            const float back = vr * (1.0f / kWeightOne);
            const bool whole = a.b0 == 0 && a.b1 == a.nb;
            const int slot = a.b0 == 0 ? 1 : 0;
            const float inv = whole ? inv_sum(l) * back : back;
            float4* part = reinterpret_cast<float4*>(po + static_cast<size_t>(slot) * kRows * C::D) + x * 128 + row;
#pragma unroll 1
            for (int c = 0; c < C::D; c += 32) {
                uint32_t o[32];
                tm_ld32(t_o + c, o);
                tc_wait_ld();
                reg_fence32(o);
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(o[i]) * inv;
                if (whole) {
                    // through shared memory (its queries are done with), so that rows leave whole
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        sts128(q_unit(row, (c + i) / 8), pack_bf16(v[i], v[i + 1]), pack_bf16(v[i + 2], v[i + 3]), pack_bf16(v[i + 4], v[i + 5]),
                               pack_bf16(v[i + 6], v[i + 7]));
                    }
                } else if (valid) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        part[static_cast<size_t>((c + i) / 4) * kRows] = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                }
            }
            if (whole) {
                __syncwarp();
                const int sub = lane / LPR, ch = lane % LPR, tok = valid ? row_token(p, pr) : 0;
                const int64_t place = static_cast<int64_t>(a.s.q0 + tok) * p.ldo +
                                      static_cast<int64_t>(a.head * p.group + (valid ? pr - tok * p.group : 0)) * C::D;
#pragma unroll 4
                for (int i = 0; i < 32 / RPI; ++i) {
                    const int rr = i * RPI + sub;
                    const int64_t to = __shfl_sync(0xffffffffu, place, rr);
                    const uint4 v = lds128(q_unit((row & 96) + rr, ch));
                    if (pr - lane + rr < a.s.n * p.group) *reinterpret_cast<uint4*>(p.out + to + ch * 8) = v;
                }
                __syncwarp();
            }
            if (!whole) {
                ml[slot * 2 * kRows + x * 128 + row] = m;
                ml[slot * 2 * kRows + kRows + x * 128 + row] = l;
                if (x == 0 && row == 0)
                    info[slot] = Partial{(static_cast<long long>(a.seq) * p.c.kv_heads + a.head) * 0x1000000LL + a.tile, a.s.q0,
                                         a.s.n * p.group, a.head, a.tile * kRows};
            }
            tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->ofree[x]);
        more = a.next(p, least);
    }
}

// ------------------------------------------------------------------ kernel

template <class C>
__global__ void __launch_bounds__(kManyThreads, 1) attend_many_kernel(const AttentionParams p, const int least)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ ManyBars bars_;
    __shared__ BlockScales ring[kScaleRing];
    __shared__ Start start;
    ManyBars* bars = &bars_;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    long long* prefix = reinterpret_cast<long long*>(smem + C::OFF_PREFIX);
    const int warp = warp_id(), lane = lane_id();
    const CacheView& cv = p.c;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kNS; ++i) {
            mbar_init(&bars->kfull[i], 5);
            mbar_init(&bars->kempty[i], 2);
            mbar_init(&bars->vfull[i], 4);
            mbar_init(&bars->vempty[i], 2);
        }
        for (int i = 0; i < kNR; ++i) {
            mbar_init(&bars->rfull[i], 1);
            mbar_init(&bars->rempty[i], 4);
        }
        for (int x = 0; x < 2; ++x) {
            for (int b = 0; b < 2; ++b) {
                mbar_init(&bars->pready[x][b], 4);
                mbar_init(&bars->pvdone[x][b], 1);
            }
            mbar_init(&bars->sfull[x], 1);
            mbar_init(&bars->sfree[x], 4);
            mbar_init(&bars->qfull[x], 4);
            mbar_init(&bars->ofree[x], 4);
            mbar_init(&bars->drain[x], 1);
        }
        bars->abort = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(&bars->tmem_base, C::TM_COLS);
        tmem_relinquish();
    }
    pdl_wait();

    // ---- units of each sequence: a warp sums its tiles' blocks ----
    for (int s = warp; s < cv.batch; s += kManyThreads / 32) {
        const Seq q = load_seq(cv, s);
        const int tiles = many_tiles(q, p.group, least);
        long long u = 0;
        for (int t = lane; t < tiles; t += 32) u += many_units(q, p.group, t);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
        if (lane == 0) prefix[s] = u * cv.kv_heads;
    }
    __syncthreads();
    if (warp == 0) {
        long long run = 0;
        for (int base = 0; base < cv.batch; base += 32) {
            const int s = base + lane;
            const long long u = s < cv.batch ? prefix[s] : 0;
            long long v = u;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += y;
            }
            if (s < cv.batch) prefix[s] = run + v - u;
            run += __shfl_sync(0xffffffffu, v, 31);
        }
        __syncwarp();
        const int share = max(kMinUnits, least_share(run, p.segments, 1, kPartBlocks));
        const long long W = min(static_cast<long long>(gridDim.x), quotient(run + share - 1, share));
        const long long c = blockIdx.x;
        const long long u0 = c < W ? quotient(run * c, W) : run, u1 = c < W ? quotient(run * (c + 1), W) : run;
        Start st{0, 0, 0, 0, u1 - u0};
        if (u0 < u1) {
            int lo = 0, hi = cv.batch - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (prefix[mid] <= u0) lo = mid;
                else hi = mid - 1;
            }
            const Seq q = load_seq(cv, lo);
            const long long per_head = quotient((lo + 1 < cv.batch ? prefix[lo + 1] : run) - prefix[lo], cv.kv_heads);
            const long long off = u0 - prefix[lo];
            st.seq = lo;
            st.head = static_cast<int>(quotient(off, per_head));
            long long r = off - st.head * per_head;
            // the tile that holds unit r of the head
            const int tiles = many_tiles(q, p.group, least);
            for (int base = 0; base < tiles; base += 32) {
                const int t = base + lane;
                const long long u = t < tiles ? many_units(q, p.group, t) : 0;
                long long v = u;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const long long y = __shfl_up_sync(0xffffffffu, v, o);
                    if (lane >= o) v += y;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, v > r);
                if (hit) {
                    const int w = __ffs(hit) - 1;
                    st.tile = base + w;
                    st.unit = static_cast<int>(r - __shfl_sync(0xffffffffu, v - u, w));
                    break;
                }
                r -= __shfl_sync(0xffffffffu, v, 31);
            }
        }
        if (lane == 0) start = st;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = bars->tmem_base, sm = smem_u32(smem);
    volatile int* abort_flag = &bars->abort;
    const Start st = start;

    if (warp < kConvWarp) {
        regs_inc<kRegsSoft>();
        softmax_role<C>(p, bars, sm, tbase, ring, st, least, abort_flag);
    } else {
        regs_dec<kRegsRest>();
        if (warp < kMmaWarp) converter_role<C>(p, bars, sm, st, least, abort_flag);
        else if (warp == kFetchWarp) fetch_role<C>(p, bars, sm, ring, st, least, abort_flag);
        else if (warp < kFetchWarp && elect_one()) mma_role<C>(p, bars, sm, tbase, warp - kMmaWarp, st, least, abort_flag);
    }
    pdl_launch_dependents();
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tbase, C::TM_COLS);
    }
}

// Joins the parts of tiles that span CTAs: blockIdx.x leads the tile that begins
// in CTA blockIdx.x and goes on; blockIdx.y takes 32 of its rows, a lane each, and a
// warp 16 columns, so that a thread's output is one whole sector.  Almost every tile
// has two parts, whose loads a thread has in flight together.
constexpr int kJoinRows = 32;

template <class C>
__global__ void __launch_bounds__(kJoinRows * C::D / 16) attend_many_join_kernel(const AttentionParams p, const int nctas)
{
    pdl_launch_dependents();
    pdl_wait();
    const float* ml = reinterpret_cast<const float*>(p.ws + ManyLayout<C>::ml(nctas));
    const float4* po = reinterpret_cast<const float4*>(p.ws + ManyLayout<C>::o(nctas));
    const int lead = blockIdx.x;
    Partial rec;
    const int n = find_parts(reinterpret_cast<const Partial*>(p.ws), lead, nctas, rec);
    const int row = blockIdx.y * kJoinRows + lane_id(), d4 = warp_id() * 4;
    if (n == 0 || rec.row0 + row >= rec.rows) return;
    const auto slot = [&](int i) { return 2 * (lead + i) + (i == 0); };
    float4 o[4];
    join_parts<2>(
        n, [&](int i) { const float* v = ml + slot(i) * 2 * kRows + row; return make_float2(v[0], v[kRows]); },
        [&](int i, int v) { return po[static_cast<size_t>(slot(i)) * (kRows * C::D / 4) + static_cast<size_t>(d4 + v) * kRows + row]; },
        o);
    uint4* dst = reinterpret_cast<uint4*>(out_row(p, rec.q0, rec.head, rec.row0 + row) + d4 * 4);
#pragma unroll
    for (int v = 0; v < 2; ++v)
        dst[v] = make_uint4(pack_bf16(o[2 * v].x, o[2 * v].y), pack_bf16(o[2 * v].z, o[2 * v].w),
                            pack_bf16(o[2 * v + 1].x, o[2 * v + 1].y), pack_bf16(o[2 * v + 1].z, o[2 * v + 1].w));
}

template <class C>
cudaError_t launch_many(const AttentionParams& p, int least, int sms, cudaStream_t stream)
{
    const int fixed = C::OFF_PREFIX + 1024;
    static bool ready[64] = {};          // per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        e = cudaFuncSetAttribute(attend_many_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, fixed + kMaxBatch * 8);
        if (e != cudaSuccess) return e;
        // setmaxnreg draws on the launch's registers: a build with fewer than the split needs must not start
        cudaFuncAttributes fa{};
        if ((e = cudaFuncGetAttributes(&fa, attend_many_kernel<C>)) != cudaSuccess) return e;
        if (fa.numRegs * 4 < 2 * kRegsSoft + 2 * kRegsRest) return cudaErrorInvalidConfiguration;
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms);
    cfg.blockDim = dim3(kManyThreads);
    cfg.dynamicSmemBytes = fixed + p.c.batch * 8;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, attend_many_kernel<C>, p, least);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3(sms, kRows / kJoinRows);
    cfg.blockDim = dim3(kJoinRows * C::D / 16);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, attend_many_join_kernel<C>, p, sms);
}

}  // namespace

size_t attend_many_ws_bytes(int D, int sms)
{
    return D == 128 ? ManyLayout<ManyCfg<128>>::total(sms) : ManyLayout<ManyCfg<64>>::total(sms);
}

cudaError_t launch_attend_many(const AttentionParams& p, int least, int sms, cudaStream_t stream)
{
    return p.c.D == 128 ? launch_many<ManyCfg<128>>(p, least, sms, stream) : launch_many<ManyCfg<64>>(p, least, sms, stream);
}

}  // namespace w4a8
