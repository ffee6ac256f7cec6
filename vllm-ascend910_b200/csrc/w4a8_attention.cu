// w4a8_attention.cu -- causal attention over the paged 8-bit cache.
//
// For query token i of a sequence with n query tokens and L tokens in the
// cache (these included), position p = L - n + i, and one kv head:
//
//   s_j = scale * ks(page of j) * (q . kc_j)        j <= p
//   o   = sum_j exp(s_j - max s) * vs(page of j) * vc_j / sum_j exp(s_j - max s)
//
// kc, vc are the cache's int8 codes, ks, vs the page scales.  Codes enter the
// tensor core as fp16, exactly; the page scales multiply scores and
// probabilities in fp32, so a page costs one product per score and none per
// element.  fp16 rather than bf16 for both products: a code takes three
// instructions a pair instead of four to convert, and probabilities keep 11
// bits instead of 8.  Its range is kept by powers of two, which are exact:
//   * a query row is divided by 2^e with its largest element in [2^13, 2^14)
//     before it becomes fp16 (8 significand bits fit; what falls below fp16's
//     range is under 2^-28 of the row's largest element), and scores are
//     multiplied by 2^e;
//   * a probability enters as p * vs / vr * 2^14 with p <= 1 and vr a power of
//     two, at least every vs so far (raised together with the running maximum),
//     so weights down to 2^-28 of the largest possible keep all 11 bits.
// Scores, running maximum and sum, and the output accumulate in fp32; the sum
// is taken before the weights are rounded.  A row that sees no token is zero.
//
// Few query rows (kernel below): one pass over the cache, bound by HBM.
//   * Work is cut in units of 16 tokens of one (sequence, kv head, row tile);
//     a row tile is R = 8 * NT packed rows (query token x query head of the
//     group).  All units of the call form one list; every warp of the grid
//     takes an equal contiguous share, whatever the lengths are.  Lengths are
//     read on the device, so a captured graph follows them.
//   * A warp computes S^T = K Q^T and O^T += V^T P^T with m16n8k16: the cache
//     is the 16-row operand, so 8 query rows fill an instruction and a single
//     token's group of 5 or 8 heads wastes little.  It keeps O^T (D x R), the
//     running maximum and its lanes' part of the sum in registers.
//   * Units arrive by 16-byte asynchronous copies in a ring of its own, three
//     deep: with 16 warps up to 128 KB are on the way to an SM.  Shared memory holds codes with
//     16-byte chunks permuted by token, so fragment reads do not collide.
//   * A warp's share begins and ends inside (sequence, head) segments.  Pieces
//     of one segment are joined in the CTA; parts of CTAs by the last of them to
//     finish (a counter tells which), always in unit order, so the bits do not
//     depend on who is last.  Nothing waits for another CTA.
//   * The counters outlive the call, so what an earlier one left must not matter,
//     not even calls that overlapped on one workspace against its rule.  A word of
//     the workspace counts started CTAs modulo four calls' worth: its quotient by
//     the grid is the call's number modulo 4, the same for all of its CTAs since calls
//     follow one another.  A segment's parts are counted in that byte of its word,
//     and the CTA that owns the word clears the other three for the calls to come.
//
// Measured (B200, 40 query heads on 8 of 128): 64 single tokens at 64 to 8,191 (566 MB
// of codes) 108 us, 5.3 TB/s, 80 % of a plain copy's rate; for three seconds on end 123 us, at
// 996 W and an SM clock of 1,680 MHz instead of 1,965 (sampled, power cap active).  One
// token at 4,000: 14 us, of which
// the codes are 1.3: launch, the lists, a chain of loads and the join.  12 x 2-5 drafted
// tokens at 3,000 to 16,000, one kv head: 28 us for 26 MB: a CTA's warps wait for few units
// each, and 10 to 25 rows take up to four products of 8 rows a unit.
#include <algorithm>

#include "w4a8_attention.cuh"

namespace w4a8 {

namespace {

constexpr int kBlkTok = 16;        // tokens per unit
constexpr int kStages = 3;         // units in a warp's ring

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool ok)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint2 lds64(uint32_t a)
{
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ float lds32f(uint32_t a)
{
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
    return v;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Row tiles of a sequence, and 16-token blocks of each (at least one, so that
// rows which see nothing are written too).
__device__ __forceinline__ int seq_tiles(const Seq& s, int group, int rows, int most)
{
    return s.n * group <= most ? (s.n * group + rows - 1) / rows : 0;
}
__device__ __forceinline__ int seq_blocks(const Seq& s) { return max(1, (s.len + kBlkTok - 1) / kBlkTok); }

// ------------------------------------------------------------------ few rows

template <int D_, int NT_>
struct DecCfg {
    static constexpr int D = D_, NT = NT_, R = 8 * NT_;
    static constexpr int WARPS = NT_ == 1 ? 16 : 8;
    static constexpr int THREADS = WARPS * 32;
    static constexpr int KV_BYTES = kBlkTok * D_;                  // codes of K (or V) in a unit
    static constexpr int STAGE = 2 * KV_BYTES + 16;                // + the page's two scales
    static constexpr int RING = kStages * STAGE;                   // one warp's
    static constexpr int PIECE = R * D_ * 4;                       // fp32 O of one piece
    static constexpr int SLOT = RING > PIECE ? RING : PIECE;       // the ring's memory holds the last piece
    static constexpr int SMEM = WARPS * SLOT;
    // What a part costs its segment's join, in units.  One kv head, 1 token at 64,000: 31 us cut
    // to single units, 25 with 0.15, 30 with 0.6; at 4,000 11.4, 13.2 and 15.3 (so 0.08).  3 tokens
    // at 16,000: 44, 22 and 24; 3 at 4,000: 17.6, 15.1 and 16.8.
    static constexpr float PART_UNITS = NT_ == 1 ? 0.08f : 0.2f;
    static constexpr int CHUNKS = D_ / 16;                         // 16-byte chunks of a token's row
};

// Where chunk ch of token t is in shared memory: permuted so that the reads of
// K (two neighbouring tokens x four chunks) and of V (tokens 2c x chunk) by the
// eight lanes of a phase fall in different banks.
template <int D>
__device__ __forceinline__ uint32_t chunk_off(int t, int ch)
{
    if (D == 128) return t * 128 + ((ch ^ (t & 7)) << 4);
    return t * 64 + ((ch ^ ((t >> 1) & 3)) << 4);
}

// Where 16-byte unit u of row `row` of a piece lies: permuted so that the eight
// lanes of a store phase (four rows 2c + h, two neighbouring r) and of a read
// phase (eight units of one row) hit different banks.
template <int D>
__device__ __forceinline__ int piece_off(int row, int u)
{
    const int c = (row >> 1) & 3;
    return row * D * 4 + ((u ^ (D == 128 ? c : (c & 1) | ((c & 2) << 1))) << 4);
}

// One piece of a segment kept for the join: unit range and softmax state.
struct PieceInfo {
    long long seg, seg_end;          // the segment's units; seg -1: no piece
    int q0, rows, head, tile;        // its sequence's first query token and packed rows, kv head, row tile
    int complete_lo, complete_hi;    // the piece reaches the segment's first / last unit
};

template <class C>
struct Layout {
    // workspace: [grid][2] (m, l)[R], then [grid][2] O, then [grid * WARPS] O of stashed pieces
    static __host__ __device__ size_t ml() { return 0; }
    static __host__ __device__ size_t o(int grid) { return static_cast<size_t>(grid) * 2 * 2 * C::R * 4; }
    static __host__ __device__ size_t stash(int grid) { return o(grid) + static_cast<size_t>(grid) * 2 * C::PIECE; }
    static __host__ __device__ size_t total(int grid)
    {
        return stash(grid) + static_cast<size_t>(grid) * C::WARPS * C::PIECE;
    }
};

// The unit list cut in `workers` contiguous shares: the first `more` of them have
// `each` + 1 units, the others `each`.
struct Shares {
    long long total, each;
    int workers, more;
    __device__ __forceinline__ Shares(long long t, int w) : total(t), workers(w)
    {
        if (t < 0x7FFFFFFF) {                       // (32-bit division is several times shorter)
            each = static_cast<uint32_t>(t) / static_cast<uint32_t>(w);
        } else {
            each = t / w;
        }
        more = static_cast<int>(t - each * w);
    }
    __device__ __forceinline__ long long begin(int w) const { return w >= workers ? total : each * w + min(w, more); }
    // The worker whose share holds unit u.
    __device__ __forceinline__ int of(long long u) const
    {
        const long long first = (each + 1) * more;  // units of the longer shares
        if (u < first) return u < 0x7FFFFFFF ? static_cast<int>(static_cast<uint32_t>(u) / static_cast<uint32_t>(each + 1))
                                             : static_cast<int>(u / (each + 1));
        u -= first;
        return more + (u < 0x7FFFFFFF ? static_cast<int>(static_cast<uint32_t>(u) / static_cast<uint32_t>(each))
                                      : static_cast<int>(u / each));
    }
};

// The position of a warp in the unit list.
template <class C>
struct Cursor {
    int seq, head, tile, blk, blocks;
    Seq s;
    __device__ __forceinline__ void set(const CacheView& c, int group, int most, int sq, long long off)
    {
        seq = sq;
        s = load_seq(c, sq);
        blocks = seq_blocks(s);
        const int tiles = seq_tiles(s, group, C::R, most);
        if (off < 0x7FFFFFFF) {
            const int t = static_cast<int>(static_cast<uint32_t>(off) / static_cast<uint32_t>(blocks));
            blk = static_cast<int>(off) - t * blocks;
            head = t / tiles;
            tile = t - head * tiles;
        } else {
            const long long t = off / blocks;
            blk = static_cast<int>(off - t * blocks);
            head = static_cast<int>(t / tiles);
            tile = static_cast<int>(t - static_cast<long long>(head) * tiles);
        }
    }
    // Next unit; false past the end of the list.
    __device__ __forceinline__ bool next(const CacheView& c, int group, int most)
    {
        if (++blk < blocks) return true;
        blk = 0;
        if (++tile < seq_tiles(s, group, C::R, most)) return true;
        tile = 0;
        if (++head < c.kv_heads) return true;
        head = 0;
        do {
            if (++seq >= c.batch) return false;
            s = load_seq(c, seq);
        } while (seq_tiles(s, group, C::R, most) == 0);
        blocks = seq_blocks(s);
        return true;
    }
};

// Writes rows of O^T that a warp holds: out[row] = acc / l for the valid rows.
template <class C>
__device__ __forceinline__ void store_rows(const AttentionParams& p, const Seq& s, int head, int tile,
                                           const float (&acc)[C::NT][C::D / 16][4], const float (&l)[C::NT][2])
{
    const int r = lane_id() >> 2, c = lane_id() & 3;
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = tile * C::R + nt * 8 + 2 * c + h;
            if (row >= s.n * p.group) continue;
            const float inv = inv_sum(l[nt][h]);
            uint16_t* o = out_row(p, s.q0, head, row) + r * (C::D / 8);
            uint32_t w[C::D / 16];
#pragma unroll
            for (int i = 0; i < C::D / 16; ++i) w[i] = pack_bf16(acc[nt][i][h] * inv, acc[nt][i][2 + h] * inv);
#pragma unroll
            for (int i = 0; i < C::D / 16; i += 4)
                *reinterpret_cast<uint4*>(o + 2 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        }
}

template <class C>
__global__ void __launch_bounds__(C::THREADS, 1) attend_few_kernel(const AttentionParams p)
{
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ PieceInfo pieces[2 * C::WARPS];
    __shared__ float piece_m[2 * C::WARPS][C::R], piece_l[2 * C::WARPS][C::R];
    __shared__ long long warp_sum[C::WARPS];
    __shared__ long long running;
    __shared__ uint32_t byte_shift;                   // 8 * (the call's number modulo 4): the counters' byte
    __shared__ bool is_last[2];
    __shared__ int seg_cta0[2], seg_parts[2];
    long long* prefix = reinterpret_cast<long long*>(smem + C::SMEM);   // [batch + 1] units before each sequence

    const int tid = threadIdx.x, warp = warp_id(), lane = lane_id();
    const CacheView& cv = p.c;
    if (tid < 2 * C::WARPS) pieces[tid].seg = -1;
    if (tid == 0) running = 0;
    pdl_wait();
    const uint32_t started = tid == 0 ? atomicInc(p.calls, 4 * gridDim.x - 1) : 0;     // (in flight during the scan)

    // ---- units before each sequence ----
    __syncthreads();
    for (int base = 0; base < cv.batch; base += C::THREADS) {
        const int s = base + tid;
        long long u = 0;
        if (s < cv.batch) {
            const Seq q = load_seq(cv, s);
            u = static_cast<long long>(cv.kv_heads) * seq_tiles(q, p.group, C::R, p.few_most) * seq_blocks(q);
        }
        long long x = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) warp_sum[warp] = x;
        __syncthreads();
        long long before = running;
        for (int w = 0; w < warp; ++w) before += warp_sum[w];
        if (s < cv.batch) prefix[s] = before + x - u;
        __syncthreads();
        if (tid == C::THREADS - 1) running = before + x;
        __syncthreads();
    }
    if (tid == 0) {
        byte_shift = 8 * (started / gridDim.x);
        atomicAnd(p.tickets + blockIdx.x, 0xFFu << byte_shift);
    }
    const long long total = running;
    // equal contiguous shares, none below the least: a short list leaves the last
    // CTAs without work, none between working ones
    const int wk = static_cast<int>(blockIdx.x) * C::WARPS + warp;
    const int least = least_share(total, p.segments, C::WARPS, C::PART_UNITS), most = static_cast<int>(gridDim.x) * C::WARPS;
    const Shares sh(total, total >= static_cast<long long>(most) * least ? most : max(1u, static_cast<uint32_t>(total) / least));
    const long long u0 = sh.begin(wk), u1 = sh.begin(wk + 1);

    float acc[C::NT][C::D / 16][4];
    float m[C::NT][2], negm[C::NT][2], l[C::NT][2];
    const int r = lane >> 2, c = lane & 3;
    const uint32_t ring = smem_u32(smem + warp * C::SLOT);

    if (u0 < u1) {
        // last sequence whose first unit is at or before u0
        int lo = 0, hi = cv.batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (prefix[mid] <= u0) lo = mid;
            else hi = mid - 1;
        }
        Cursor<C> cur, pre;
        cur.set(cv, p.group, p.few_most, lo, u0 - prefix[lo]);
        pre = cur;

        // Where this lane's copies and fragment reads lie in a stage.  chunk_off swizzles
        // by the token's low bits, so offsets of further copies and tokens are constants:
        // tokens 8 apart keep their swizzle, and a copy's neighbour 4 tokens on flips one bit.
        const uint32_t cp0 = chunk_off<C::D>(lane / C::CHUNKS, lane % C::CHUNKS);
        const uint32_t cp1 = chunk_off<C::D>(lane / C::CHUNKS + 32 / C::CHUNKS, lane % C::CHUNKS) - 512;
        const uint32_t k0 = chunk_off<C::D>(r, c * (C::D / 64)), k1 = chunk_off<C::D>(r, c * (C::D / 64) + (C::D / 64 - 1));
        const uint32_t v0 = C::D == 128 ? chunk_off<C::D>(2 * c, r) : chunk_off<C::D>(2 * c, r >> 1) + (r & 1) * 8;
        const uint32_t v1 = C::D == 128 ? chunk_off<C::D>(2 * c + 1, r) : chunk_off<C::D>(2 * c + 1, r >> 1) + (r & 1) * 8;
        const int pages = static_cast<int>(cv.pages);
        int ahead = static_cast<int>(u1 - u0);    // units of the share still to be fetched
        // Page ids of a sequence, 32 at a time: lane i holds that of page id_page + i.
        int ids = -1, id_seq = -1, id_page = 0;

        // Brings the unit under `pre` into ring stage st and moves on.
        auto fetch = [&](int st) {
            if (ahead > 0) {
                const int tok = pre.blk * kBlkTok, pg = tok >> cv.page_log2;
                if (pre.seq != id_seq || pg < id_page || pg >= id_page + 32) {
                    id_seq = pre.seq;
                    id_page = pg;
                    ids = pg + lane <= (pre.s.len - 1) >> cv.page_log2 ? cv.table[pre.seq * cv.ld_table + pg + lane] : -1;
                }
                const int id = __shfl_sync(0xffffffffu, ids, pg - id_page);
                const bool ok = static_cast<unsigned>(id) < static_cast<unsigned>(pages);
                const int64_t ph = ok ? static_cast<int64_t>(id) * cv.kv_heads + pre.head : 0;
                const int64_t at = ((ph << cv.page_log2) + (ok ? tok & (cv.page - 1) : 0)) * C::D + lane * 16;
                const int8_t *kp = cv.k + at, *vp = cv.v + at;
                const uint32_t d = ring + st * C::STAGE;
#pragma unroll
                for (int i = 0; i < C::KV_BYTES / 512; ++i) {
                    const uint32_t off = d + ((i & 1) ? cp1 : cp0) + i * 512;
                    cp_async16(off, kp + i * 512, ok);
                    cp_async16(off + C::KV_BYTES, vp + i * 512, ok);
                }
                // a page that is not there has no tokens: its scale is marked with -1
                if (lane < 2) {
                    if (ok) cp_async4(d + 2 * C::KV_BYTES + lane * 4, (lane ? cv.v_scale : cv.k_scale) + ph, true);
                    else asm volatile("st.shared.f32 [%0], %1;" ::"r"(d + 2 * C::KV_BYTES + lane * 4), "f"(-1.0f));
                }
                if (--ahead > 0) pre.next(cv, p.group, p.few_most);
            }
            cp_commit();
        };

        uint32_t qf[C::NT][C::D / 16][2];
        int limit[C::NT][2];
        float qs[C::NT][2];
        float vr = kVrMin;                        // power of two at or above every vs of the segment so far
        float vr_inv = kWeightOne / kVrMin;       // 2^14 / vr
        int min_limit = 0;
        // The segment's query rows as they are, this lane's elements of row r.
        auto load_queries = [&]() {
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) {
                const int row = cur.tile * C::R + nt * 8 + r;
                const bool ok = row < cur.s.n * p.group;
                const int tok = ok ? row_token(p, row) : 0, g = ok ? row - tok * p.group : 0;
                const uint16_t* q = p.q + static_cast<int64_t>(cur.s.q0 + tok) * p.ldq +
                                    static_cast<int64_t>(cur.head * p.group + g) * C::D + c * (C::D / 4);
#pragma unroll
                for (int i = 0; i < C::D / 32; ++i) {
                    const uint4 v = ok ? *reinterpret_cast<const uint4*>(q + 8 * i) : make_uint4(0, 0, 0, 0);
                    qf[nt][2 * i][0] = v.x;
                    qf[nt][2 * i][1] = v.y;
                    qf[nt][2 * i + 1][0] = v.z;
                    qf[nt][2 * i + 1][1] = v.w;
                }
            }
        };
        // The rows in fp16, and a fresh softmax state.
        auto begin_segment = [&]() {
            min_limit = 0x7FFFFFFF;
            vr = kVrMin;
            vr_inv = kWeightOne / kVrMin;
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) {
                // the row's largest magnitude, as bits: its elements are in the four lanes of r
                uint32_t big = 0;
#pragma unroll
                for (int i = 0; i < C::D / 16; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        big = max(big, max((qf[nt][i][e] << 16) & 0x7FFFFFFFu, qf[nt][i][e] & 0x7FFF0000u));
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
                const float shrink = row_shrink(__uint_as_float(big));
#pragma unroll
                for (int i = 0; i < C::D / 16; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        qf[nt][i][e] = pack_f16(__uint_as_float(qf[nt][i][e] << 16) * shrink,
                                                __uint_as_float(qf[nt][i][e] & 0xFFFF0000u) * shrink);
                // scores of columns 2c, 2c + 1: their rows' factor lies with lanes r = 2c, 2c + 1
                const float grow_back = __fdiv_rn(p.scale_log2, shrink);
#pragma unroll
                for (int h = 0; h < 2; ++h) qs[nt][h] = __shfl_sync(0xffffffffu, grow_back, (2 * c + h) * 4);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int qr = cur.tile * C::R + nt * 8 + 2 * c + h;
                    // rows past the sequence's last are computed on zero queries and not stored
                    limit[nt][h] = qr < cur.s.n * p.group ? cur.s.pos + row_token(p, qr) : 0x7FFFFFFF;
                    min_limit = min(min_limit, limit[nt][h]);
                    m[nt][h] = kNegInf;
                    negm[nt][h] = first_reference(kNegInf);
                    l[nt][h] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < C::D / 16; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[nt][i][e] = 0.0f;
            }
            min_limit = __reduce_min_sync(0xffffffffu, min_limit);
        };

        load_queries();
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) fetch(i);
        begin_segment();
        long long seg_lo = u0 - cur.blk;          // first unit of the segment under `cur`
        int piece_blk = cur.blk;                  // the piece's first block
        int st = 0;
        for (int left = static_cast<int>(u1 - u0); left > 0; --left) {
            cp_wait<kStages - 2>();
            __syncwarp();
            fetch(st == 0 ? kStages - 1 : st - 1);     // the stage consumed in the previous pass
            const uint32_t kb = ring + st * C::STAGE, vb = kb + C::KV_BYTES;
            const float ks = lds32f(kb + 2 * C::KV_BYTES), vs = lds32f(kb + 2 * C::KV_BYTES + 4);

            // ---- S^T = K Q^T ----
            float sc[C::NT][4];
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[nt][e] = 0.0f;
            uint32_t kw[2][C::D / 16];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < C::D / 64; ++i) {
                    const uint4 v = lds128(kb + (i ? k1 : k0) + t * (8 * C::D));
                    kw[t][4 * i] = v.x ^ 0x80808080u;
                    kw[t][4 * i + 1] = v.y ^ 0x80808080u;
                    kw[t][4 * i + 2] = v.z ^ 0x80808080u;
                    kw[t][4 * i + 3] = v.w ^ 0x80808080u;
                }
#pragma unroll
            for (int ks_ = 0; ks_ < C::D / 16; ++ks_) {
                uint32_t a[4];
                a[0] = biased_lo(kw[0][ks_]);
                a[1] = biased_lo(kw[1][ks_]);
                a[2] = biased_hi(kw[0][ks_]);
                a[3] = biased_hi(kw[1][ks_]);
#pragma unroll
                for (int nt = 0; nt < C::NT; ++nt) mma_f16(sc[nt], a, qf[nt][ks_][0], qf[nt][ks_][1]);
            }

            // ---- scores less the reference, in log2 units ----
            float f[C::NT][2], wv[C::NT][2];
            const float vsr = vs * vr_inv;
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    f[nt][h] = ks * qs[nt][h];
                    wv[nt][h] = vsr;
                }
            const int t0 = cur.blk * kBlkTok;
            const bool there = !(ks < 0.0f);             // (a NaN scale passes on; -1: no page)
            float vsu = there ? vs : 0.0f;               // what vr has to cover
            if (t0 + kBlkTok - 1 > min_limit || !there) {
                // Masked scores become -inf; a row that sees nothing of the unit takes
                // factors that cannot touch it, and no factor is 0 (0 * inf).
                bool seen = false;
#pragma unroll
                for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const bool none = !there || t0 > limit[nt][h];
                        f[nt][h] = none ? 1.0f : (ks != ks ? ks : fmaxf(f[nt][h], 1e-37f));
                        if (none) wv[nt][h] = 0.0f;
                        seen = seen || !none;
                        if (none || t0 + r > limit[nt][h]) sc[nt][h] = kNegInf;
                        if (none || t0 + r + 8 > limit[nt][h]) sc[nt][2 + h] = kNegInf;
                    }
                if (!__any_sync(0xffffffffu, seen)) vsu = 0.0f;
            }
            float raise = vsu > vr ? INFINITY : 0.0f;
            float d[C::NT][4];
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    d[nt][e] = fmaf(sc[nt][e], f[nt][e & 1], negm[nt][e & 1]);
                    raise = fmaxf(raise, d[nt][e]);
                }
            if (__any_sync(0xffffffffu, raise > kSlack)) {
                // ---- the references move: m to the scores' maximum, vr over vs ----
                const float vn = fmaxf(vr, pow2_above(vsu));
                const float va = __fdiv_rn(vr, vn);
                vr = vn;
                vr_inv = __fdiv_rn(kWeightOne, vr);
#pragma unroll
                for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float x = fmaxf(sc[nt][h], sc[nt][2 + h]) * f[nt][h];
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        const float mn = fmaxf(m[nt][h], x);
                        const float a = mn == kNegInf ? 1.0f : ex2(m[nt][h] - mn);
                        m[nt][h] = mn;
                        negm[nt][h] = first_reference(mn);
                        l[nt][h] *= a;
                        const float av = a * va;
#pragma unroll
                        for (int i = 0; i < C::D / 16; ++i) {
                            acc[nt][i][h] *= av;
                            acc[nt][i][2 + h] *= av;
                        }
                        d[nt][h] = fmaf(sc[nt][h], f[nt][h], negm[nt][h]);
                        d[nt][2 + h] = fmaf(sc[nt][2 + h], f[nt][h], negm[nt][h]);
                        if (wv[nt][h] != 0.0f) wv[nt][h] = vs * vr_inv;
                    }
            }

            // ---- P, its sum, and the weights P * vs / vr * 2^14 as the second product's operand ----
            uint32_t pb[C::NT][2];
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) {
                const float x0 = ex2(d[nt][0]), x1 = ex2(d[nt][1]), x2 = ex2(d[nt][2]), x3 = ex2(d[nt][3]);
                l[nt][0] += x0 + x2;
                l[nt][1] += x1 + x3;
                pb[nt][0] = movmatrix_trans(pack_f16(x0 * wv[nt][0], x1 * wv[nt][1]));
                pb[nt][1] = movmatrix_trans(pack_f16(x2 * wv[nt][0], x3 * wv[nt][1]));
            }

            // ---- O^T += V^T P^T ----
            uint32_t vw[4][C::D / 32];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint32_t at = vb + ((t & 1) ? v1 : v0) + (t >> 1) * (8 * C::D);
                if (C::D == 128) {
                    const uint4 v = lds128(at);
                    vw[t][0] = v.x;
                    vw[t][1] = v.y;
                    vw[t][2 % (C::D / 32)] = v.z;
                    vw[t][3 % (C::D / 32)] = v.w;
                } else {
                    const uint2 v = lds64(at);
                    vw[t][0] = v.x;
                    vw[t][1] = v.y;
                }
            }
#pragma unroll
            for (int i = 0; i < C::D / 16; ++i) {
                const int w = i >> 1;
                const uint32_t s0 = (i & 1) ? 0x0602 : 0x0400, s1 = (i & 1) ? 0x0703 : 0x0501;
                uint32_t a[4];
                a[0] = codes_to_f16x2(__byte_perm(vw[0][w], vw[1][w], s0));
                a[1] = codes_to_f16x2(__byte_perm(vw[0][w], vw[1][w], s1));
                a[2] = codes_to_f16x2(__byte_perm(vw[2][w], vw[3][w], s0));
                a[3] = codes_to_f16x2(__byte_perm(vw[2][w], vw[3][w], s1));
#pragma unroll
                for (int nt = 0; nt < C::NT; ++nt) mma_f16(acc[nt][i], a, pb[nt][0], pb[nt][1]);
            }
            st = st == kStages - 1 ? 0 : st + 1;

            // ---- end of a piece ----
            const bool seg_end = cur.blk == cur.blocks - 1;
            if (seg_end || left == 1) {
#pragma unroll
                for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float x = l[nt][h];
                        x += __shfl_xor_sync(0xffffffffu, x, 4);
                        x += __shfl_xor_sync(0xffffffffu, x, 8);
                        x += __shfl_xor_sync(0xffffffffu, x, 16);
                        l[nt][h] = x;
                    }
                const float back = vr * (1.0f / kWeightOne);
#pragma unroll
                for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
                    for (int i = 0; i < C::D / 16; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[nt][i][e] *= back;
                if (seg_end && piece_blk == 0) {
                    store_rows<C>(p, cur.s, cur.head, cur.tile, acc, l);
                } else {
                    const bool last = left == 1;
                    const int pi = 2 * warp + (last ? 1 : 0);
                    uint8_t* dst;
                    if (last) {
                        cp_wait<0>();
                        __syncwarp();
                        dst = smem + warp * C::SLOT;
                    } else {
                        dst = p.ws + Layout<C>::stash(gridDim.x) + static_cast<size_t>(wk) * C::PIECE;
                    }
#pragma unroll
                    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int row = nt * 8 + 2 * c + h;
#pragma unroll
                            for (int i = 0; i < C::D / 16; i += 2)
                                *reinterpret_cast<float4*>(dst + piece_off<C::D>(row, r * (C::D / 32) + i / 2)) =
                                    make_float4(acc[nt][i][h], acc[nt][i][2 + h], acc[nt][i + 1][h], acc[nt][i + 1][2 + h]);
                            if (r == 0) {
                                piece_m[pi][row] = m[nt][h];
                                piece_l[pi][row] = l[nt][h];
                            }
                        }
                    if (lane == 0) {
                        PieceInfo& q = pieces[pi];
                        q.seg = seg_lo;
                        q.seg_end = seg_lo + cur.blocks;
                        q.q0 = cur.s.q0;
                        q.rows = cur.s.n * p.group;
                        q.head = cur.head;
                        q.tile = cur.tile;
                        q.complete_lo = piece_blk == 0;
                        q.complete_hi = seg_end;
                    }
                }
            }
            if (left > 1) {
                cur.next(cv, p.group, p.few_most);
                if (seg_end) {
                    seg_lo = u1 - left + 1;
                    piece_blk = 0;
                    load_queries();
                    begin_segment();
                }
            }
        }
        cp_wait<0>();
    }
    pdl_launch_dependents();
    __syncthreads();

    // ---- join the CTA's pieces, in unit order ----
    float* all_ml = reinterpret_cast<float*>(p.ws + Layout<C>::ml());
    float* all_o = reinterpret_cast<float*>(p.ws + Layout<C>::o(gridDim.x));
    float* ml = all_ml + static_cast<size_t>(blockIdx.x) * 2 * 2 * C::R;
    float* po = all_o + static_cast<size_t>(blockIdx.x) * 2 * C::R * C::D;
    const long long my_seg = lane < 2 * C::WARPS ? pieces[lane].seg : -1;
    constexpr int ITEMS = C::R * C::D / 4;          // a segment's rows, 4 elements each
    int open[2] = {-1, -1};                         // first pieces of the segments that other CTAs have parts of
    int turn = 0;
    for (unsigned todo = __ballot_sync(0xffffffffu, my_seg >= 0); todo; ++turn) {
        // the pieces of one segment, a bit each
        const int i = __ffs(todo) - 1;
        const unsigned mask = __ballot_sync(0xffffffffu, my_seg == __shfl_sync(0xffffffffu, my_seg, i));
        const int e = 31 - __clz(mask);
        todo &= ~mask;
        const PieceInfo first = pieces[i];
        const bool whole = first.complete_lo && pieces[e].complete_hi;
        const int slot = first.complete_lo ? 1 : 0;
        if (!whole) open[slot] = i;
        // segments go round the thread groups that hold one each
        constexpr int GROUPS = C::THREADS >= ITEMS ? C::THREADS / ITEMS : 1;
        if (GROUPS > 1 && tid / ITEMS != turn % GROUPS) continue;
        for (int idx = GROUPS > 1 ? tid % ITEMS : tid; idx < ITEMS; idx += GROUPS > 1 ? ITEMS : C::THREADS) {
            // a warp has one row (or two): lane k finds the factor of piece k
            constexpr int RPW = 128 / C::D;
            const int row = idx / (C::D / 4), d4 = idx % (C::D / 4), row0 = row & ~(RPW - 1);
            const bool in = (mask >> lane) & 1;
            float a[RPW], mx[RPW], ls[RPW];
#pragma unroll
            for (int k = 0; k < RPW; ++k) {
                const float pm = in ? piece_m[lane][row0 + k] : kNegInf;
                mx[k] = pm;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], o));
                a[k] = in ? (mx[k] == kNegInf ? 1.0f : ex2(pm - mx[k])) : 0.0f;
                ls[k] = in ? a[k] * piece_l[lane][row0 + k] : 0.0f;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) ls[k] += __shfl_xor_sync(0xffffffffu, ls[k], o);
            }
            const int mine = RPW > 1 ? row - row0 : 0;
            const int off = piece_off<C::D>(row, d4);
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const auto add = [&](int k, const float4& x) {
                float f = __shfl_sync(0xffffffffu, a[0], k);
                if (RPW > 1) {
                    const float f1 = __shfl_sync(0xffffffffu, a[RPW - 1], k);
                    f = mine ? f1 : f;
                }
                o.x += f * x.x;
                o.y += f * x.y;
                o.z += f * x.z;
                o.w += f * x.w;
            };
            const uint8_t* stash = p.ws + Layout<C>::stash(gridDim.x) + static_cast<size_t>(blockIdx.x) * C::WARPS * C::PIECE + off;
            // in unit order: the only stashed piece of a segment is its last one's warp's
            // first, all others are in shared memory
#pragma unroll 4
            for (unsigned left = mask & 0xAAAAAAAAu; left; left &= left - 1) {
                const int k = __ffs(left) - 1;
                add(k, *reinterpret_cast<const float4*>(smem + (k >> 1) * C::SLOT + off));
            }
            if (mask & 0x55555555u) add(e, __ldcg(reinterpret_cast<const float4*>(stash + static_cast<size_t>(e >> 1) * C::PIECE)));
            if (whole) {
                if (first.tile * C::R + row < first.rows) {
                    const float inv = inv_sum(ls[mine]);
                    uint16_t* dst = out_row(p, first.q0, first.head, first.tile * C::R + row) + d4 * 4;
                    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
                }
            } else {
                *reinterpret_cast<float4*>(po + slot * (C::R * C::D) + row * C::D + d4 * 4) = o;
                if (d4 == 0) {
                    ml[slot * 2 * C::R + row] = mx[mine];
                    ml[slot * 2 * C::R + C::R + row] = ls[mine];
                }
            }
        }
    }
    if (open[0] < 0 && open[1] < 0) return;
    // ---- the last of a segment's CTAs to come here joins their parts ----
    __syncthreads();                                // the CTA's parts have been written
    if (warp < 2 && lane == 0) is_last[warp] = false;
    if (warp < 2 && lane == 0 && open[warp] >= 0) {
        const PieceInfo& first = pieces[open[warp]];
        const int cta0 = sh.of(first.seg) / C::WARPS, n = sh.of(first.seg_end - 1) / C::WARPS - cta0 + 1;
        seg_cta0[warp] = cta0;
        seg_parts[warp] = n;
        uint32_t ticket;
        asm volatile("fence.acq_rel.gpu;\n\tatom.relaxed.gpu.global.add.u32 %0, [%1], %2;\n\tfence.acq_rel.gpu;"
                     : "=r"(ticket)
                     : "l"(p.tickets + cta0), "r"(1u << byte_shift)
                     : "memory");
        is_last[warp] = ((ticket >> byte_shift) & 0xFFu) == static_cast<uint32_t>(n - 1);
    }
    __syncthreads();
    for (int sl = 0; sl < 2; ++sl) {
        if (open[sl] < 0 || !is_last[sl]) continue;
        const PieceInfo first = pieces[open[sl]];
        const int cta0 = seg_cta0[sl], n = seg_parts[sl];
        for (int idx = tid; idx < ITEMS; idx += C::THREADS) {
            const int row = idx / (C::D / 4), d4 = idx % (C::D / 4);
            if (first.tile * C::R + row >= first.rows) continue;
            // part k is slot 1 of the segment's first CTA, slot 0 of the others
            const auto at = [&](int k) { return static_cast<size_t>(2 * (cta0 + k) + (k == 0)); };
            float4 o[1];
            join_parts<8>(
                n,
                [&](int k) {
                    const float* v = all_ml + at(k) * 2 * C::R + row;
                    return make_float2(__ldcg(v), __ldcg(v + C::R));
                },
                [&](int k, int) { return __ldcg(reinterpret_cast<const float4*>(all_o + at(k) * C::R * C::D + row * C::D + d4 * 4)); },
                o);
            uint16_t* dst = out_row(p, first.q0, first.head, first.tile * C::R + row) + d4 * 4;
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(o[0].x, o[0].y), pack_bf16(o[0].z, o[0].w));
        }
    }
}

template <class C>
cudaError_t launch_few(const AttentionParams& p, int sms, cudaStream_t stream)
{
    const int smem = C::SMEM + (p.c.batch + 1) * 8;
    static bool ready[64] = {};          // per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        e = cudaFuncSetAttribute(attend_few_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 C::SMEM + (kMaxBatch + 1) * 8);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms);
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attend_few_kernel<C>, p);
}

// Row tile of 8 * NT packed rows: the smallest that holds the rows of any sequence
// the kernel takes, at most 16.  64 single tokens of 5 rows at 1,000: 36 us in tiles of 8,
// 48 in tiles of 16; 64 times 3 tokens of 15 rows: 51 us in tiles of 16, 58 in two of 8.
int few_nt(int64_t rows) { return rows <= 8 ? 1 : 2; }

template <class F>
auto with_few(int D, int nt, const F& f)
{
    if (D == 128) {
        if (nt == 1) return f(DecCfg<128, 1>{});
        return f(DecCfg<128, 2>{});
    }
    if (nt == 1) return f(DecCfg<64, 1>{});
    return f(DecCfg<64, 2>{});
}

}  // namespace

size_t attention_ws_bytes(int batch, int64_t tokens, int q_heads, int kv_heads, int D, int max_q, int sms)
{
    (void)batch;
    (void)tokens;
    const int64_t rows = static_cast<int64_t>(max_q) * (q_heads / kv_heads);
    const size_t few = with_few(D, few_nt(rows), [&](auto c) { return Layout<decltype(c)>::total(sms); });
    return rows <= kFewRows ? few : std::max(few, attend_many_ws_bytes(D, sms));
}

cudaError_t launch_attention(const AttentionParams& p0, int sms, cudaStream_t stream)
{
    AttentionParams p = p0;
    const int64_t rows = static_cast<int64_t>(p.max_q) * p.group;
    p.few_most = 0x7FFFFFFF;
    const int tile = rows <= kFewRows ? 8 * few_nt(rows) : 256;
    p.segments = static_cast<int>(std::min<int64_t>(
        0x7FFFFFFF, static_cast<int64_t>(p.c.kv_heads) * std::max<int64_t>(p.c.batch, p.c.tokens * p.group / tile)));
    if (rows > kFewRows) {
        // A sequence has more rows than attend_few_kernel is made for.  Many sequences of
        // uneven lengths are single tokens beside prompts as a rule: each kernel takes its
        // kind.  32 single tokens at 2,000 and a prompt of 256, 1,024 or three of 1,024: 68,
        // 88 and 130 us against 103, 123 and 165 by attend_many_kernel alone.  With few or
        // even sequences the second launch costs more than it saves: 8 tokens and a prompt
        // of 1,024 62 against 59 us, one token and a prompt of 512 42 against 28, four
        // prompts of 64 33.8 against 30.7.
        const bool mixed = p.c.batch >= 16 && 2 * p.c.tokens <= static_cast<int64_t>(p.c.batch) * p.max_q;
        const cudaError_t e = launch_attend_many(p, mixed ? kFewRows : 0, sms, stream);
        if (e != cudaSuccess || !mixed) return e;
        p.few_most = kFewRows;
    }
    return with_few(p.c.D, few_nt(rows), [&](auto c) { return launch_few<decltype(c)>(p, sms, stream); });
}

}  // namespace w4a8
