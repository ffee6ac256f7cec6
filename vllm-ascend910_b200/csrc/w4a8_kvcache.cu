// w4a8_kvcache.cu -- writing one step's tokens into the paged 8-bit cache, with
// rotary positions applied on the way, and reading cached tokens back.
//
// Rotary: the first `rot` elements of a head are pairs (a, b) -- (x[i], x[i +
// rot/2]) or, interleaved, (x[2i], x[2i+1]) -- turned by the angle whose cosine
// and sine the caller's table holds for the token's position:
//
//   a' = a c - b s        b' = b c + a s          (fp32, products rounded first)
//
// Cache: int8 codes with one scale per (page, kv head), so the attention kernel
// multiplies a page's scores by one number.  A page fills over many calls and
// its scale can only grow:
//
//   s' = max(s if the page holds earlier tokens, max|new| / 127)
//   earlier codes <- rint(code * (s / s'))      new codes <- rint(x / s'), within +-127
//
// (IEEE division and rounding, so a plain fp32 implementation gives the same
// codes.)  A page of zeros has s' = 0 and codes 0; a non-finite value makes the
// page's scale non-finite and the page reads back as NaN.
//
// The write is one launch.  Some blocks turn query heads: a thread stays with
// its token and its elements of a head, so it reads the table once for all the
// heads it turns.  The other blocks own eight warps' worth of one touched page's
// (kv head, K or V) items: a warp holds 4 rows of 128 elements in registers (a page
// of 32 rows is eight warps), so k and v are read once -- rotated, their maximum found, and
// written as codes.  All loads of a warp are in flight together, and four blocks an SM
// (64 registers, for 56 bytes of spills) hide more than three or five do: 7,543 tokens
// 53 us against 58 and 69.
// A loop over several items a block was slower too (68 us).  Dividing by the scale is a
// product with its reciprocal except next to half-integers, where the true division
// decides (the activation quantiser's rule).
//
// Measured (B200): 7,543 tokens of 40 + 8 + 8 heads of 128, pages of 32: write 50 us, of
// which the queries' 155 MB alone take 24 at the memory's rate and the pages, by a chain of
// dependent loads (lengths, rows and page id, scale) and some 650 instructions a warp in each
// of 3,800 blocks, 27; read back 9 us (47 MB).  One token of 64 sequences written: 5.2 us; 530
// tokens read back: 2.9 us: launch and latency.
#include <algorithm>

#include "w4a8_common.cuh"
#include "w4a8_kernels.h"

namespace w4a8 {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
// Tokens whose query heads a block turns.  One a block: 4.3, 7.2 and 37 us for 64, 512 and
// 4,096 tokens of 40 + 8 + 8 heads of 128; four: 4.2, 5.6 and 30.
constexpr int kQTok = 4;
__host__ __device__ constexpr int chunk_rows(int D) { return 512 / D; }   // rows that a warp holds: 16 elements a lane

__device__ __forceinline__ void rotate_pair(float& a, float& b, float c, float s)
{
    const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    a = x;
}

// Bounds of sequence s: its first token in the call, their number, its length
// after the call.  The length may pass what the page table has columns for
// (capacity): tokens there have a position and no page.
__device__ __forceinline__ void seq_bounds(const CacheView& c, int s, int64_t& t0, int& n, int& len)
{
    t0 = min(static_cast<int64_t>(max(c.cu[s], 0)), c.tokens);
    const int64_t t1 = min(static_cast<int64_t>(max(c.cu[s + 1], 0)), c.tokens);
    n = static_cast<int>(max(t1 - t0, static_cast<int64_t>(0)));
    len = max(c.kv_lens[s], 0);
}
__device__ __forceinline__ int capacity(const CacheView& c) { return c.table_cols << c.page_log2; }     // (checked on the host)

// The sequence that token t belongs to: the last s with cu[s] <= t.  The whole
// warp searches for its first token t0 (32 probes a step, so two dependent loads
// for 1024 sequences), then each lane moves on to its own t >= t0.
__device__ __forceinline__ int seq_of(const int32_t* cu, int batch, int64_t t0, int64_t t)
{
    int lo = 0;
    for (int n = batch; n > 1;) {
        const int step = (n + 31) / 32, at = static_cast<int>(lane_id()) * step;
        const unsigned hit = __ballot_sync(0xffffffffu, at < n && cu[lo + at] <= t0) | 1u;
        const int k = (31 - __clz(hit)) * step;
        lo += k;
        n = min(step, n - k);
    }
    while (lo + 1 < batch && cu[lo + 1] <= t) ++lo;
    return lo;
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

// codes4 by the division alone, within +-127, for scales whose reciprocal fp32
// cannot hold; 0 for a zero or non-finite scale.
__device__ __forceinline__ uint32_t codes4_slow(const float* x, float s)
{
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -127.0f), 127.0f);
        if (s > 0.0f && s < INFINITY) w |= (static_cast<uint32_t>(static_cast<int>(q)) & 0xFFu) << (8 * i);
    }
    return w;
}

// Number of pages of sequence s that the call writes; 0 past the last sequence
// (the loads do not wait for that test).
__device__ __forceinline__ int touched_pages(const CacheView& cv, int s)
{
    int64_t t0;
    int n, len;
    seq_bounds(cv, min(s, cv.batch - 1), t0, n, len);
    const int lo = max(len - n, 0);          // tokens before position 0 are not written, nor those past the table
    const int hi = min(len, capacity(cv));
    return s < cv.batch && hi > lo ? ((hi - 1) >> cv.page_log2) - (lo >> cv.page_log2) + 1 : 0;
}

// Query heads of kQTok tokens.
template <int D>
__device__ __forceinline__ void rotate_queries(const KvWriteParams& p, int64_t t0)
{
    constexpr int LPH = D / 16;                          // threads of a head
    const CacheView& cv = p.c;
    const int j = threadIdx.x % LPH, slot = threadIdx.x / LPH;
    const int64_t t = t0 + slot % kQTok;
    const int s = p.rot ? seq_of(cv.cu, cv.batch, t0, min(t, cv.tokens - 1)) : 0;
    if (t >= cv.tokens) return;
    int c0, c1;
    item_cols(j, p.rot, p.interleaved, c0, c1);
    // the first heads' elements are on their way while the token's angles are found
    constexpr int STEP = kThreads / LPH / kQTok, AHEAD = 4;
    const uint16_t* src = p.q + t * p.ldq;
    uint16_t* dst = p.q_out + t * p.ldqo;
    const bool turn = j < p.rot / 16;
    float4 cs[4] = {};
    for (int h0 = slot / kQTok; h0 < p.q_heads; h0 += AHEAD * STEP) {
        uint4 w[AHEAD][2];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int64_t h = min(h0 + k * STEP, p.q_heads - 1);
            w[k][0] = *reinterpret_cast<const uint4*>(src + h * D + c0);
            w[k][1] = *reinterpret_cast<const uint4*>(src + h * D + c1);
        }
        if (turn && h0 == slot / kQTok) {
            int64_t first;
            int n, len;
            seq_bounds(cv, s, first, n, len);
            load_angles(p.cos_sin + clamp_row(static_cast<int64_t>(len) - n + (t - first), p.table_rows) * p.rot, j, p.rot, cs);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int64_t h = h0 + k * STEP;
            if (h >= p.q_heads) break;
            float a[8], b[8];
            unpack8_bf16(w[k][0], a);
            unpack8_bf16(w[k][1], b);
            if (turn) rotate_item(p.interleaved, cs, a, b);
            *reinterpret_cast<uint4*>(dst + h * D + c0) = pack8(a);
            *reinterpret_cast<uint4*>(dst + h * D + c1) = pack8(b);
        }
    }
}

// A touched page: its sequence (-1: nothing to do), the sequence's first token, number
// of tokens and length, and the page's number in it.
struct Job {
    int64_t t0;
    int s, n, len, pg;
};

template <int D, bool ONE>
__global__ void __launch_bounds__(kThreads, 4) kv_write_kernel(const KvWriteParams p, const int q_blocks, const int groups)
{
    __shared__ uint32_t sh_max[kWarps];
    __shared__ Job sh_job;

    const CacheView& cv = p.c;
    const int lane = lane_id(), warp = warp_id();
    pdl_wait();

    // Query blocks (bound by bandwidth) and page blocks (by latency) alternate in
    // proportion, so that both kinds are resident together.
    const int64_t qi = static_cast<int64_t>(blockIdx.x) * q_blocks / gridDim.x;
    if ((static_cast<int64_t>(blockIdx.x) + 1) * q_blocks / gridDim.x > qi) {
        rotate_queries<D>(p, qi * kQTok);
        return;
    }

    // ---- one touched page: the first warp finds (sequence, page) number `job`, four
    // sequences a lane ----
    const uint32_t bid = blockIdx.x - static_cast<uint32_t>(qi);
    const int64_t job = bid / static_cast<uint32_t>(groups);
    const int group = static_cast<int>(bid - static_cast<uint32_t>(job) * groups);
    if (warp == 0) {
        int s = -1, local = 0;
        int64_t run = 0;                                     // touched pages before the current 128 sequences
        for (int base = 0; base < cv.batch && s < 0; base += 128) {
            int np[4];
            int64_t sum = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int q = base + lane * 4 + k;
                np[k] = touched_pages(cv, q);
                sum += np[k];
            }
            int64_t x = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, run + x > job);
            if (hit) {
                int64_t r = job - (run + x - sum);           // the page's number among the lane's sequences
                int k = 0;
                while (k < 3 && r >= np[k]) r -= np[k++];
                const int w = __ffs(hit) - 1;
                s = base + w * 4 + __shfl_sync(0xffffffffu, k, w);
                local = __shfl_sync(0xffffffffu, static_cast<int>(r), w);
            }
            run += __shfl_sync(0xffffffffu, x, 31);
        }
        Job j{0, s, 0, 0, 0};
        if (s >= 0) {
            seq_bounds(cv, s, j.t0, j.n, j.len);
            j.pg = (max(j.len - j.n, 0) >> cv.page_log2) + local;
        }
        if (lane == 0) sh_job = j;
    }
    __syncthreads();
    const int64_t t0 = sh_job.t0;
    const int n = sh_job.n, len = sh_job.len, pg = sh_job.pg;
    if (sh_job.s < 0) return;
    const int id = cv.table[static_cast<int64_t>(sh_job.s) * cv.ld_table + pg];     // (the rows' loads do not wait for it)
    const int start = len - n;                               // position of the call's first token (may be < 0)
    const int page_at = pg << cv.page_log2;
    const int lo = max(start - page_at, 0);                  // rows [0, lo): earlier tokens
    const int hi = min(len - page_at, cv.page);              // rows [lo, hi): this call's

    // This warp's item (kv head, K or V) and its chunks of the page's rows: chunk
    // `part`, part + 8, ... where a page has more than eight.
    constexpr int CHUNK = chunk_rows(D), LPR = D / 16, RPI = 32 / LPR;     // lanes of a row, rows at a time
    static_assert(CHUNK == RPI, "a lane holds 16 elements of one row");
    const int wpi_log2 = min(cv.page_log2 - (D == 128 ? 2 : 3), 3), wpi = 1 << wpi_log2;     // page / CHUNK, at most kWarps
    const int part = warp & (wpi - 1), sub = lane / LPR, j = lane % LPR;
    const int item = group * (kWarps >> wpi_log2) + (warp >> wpi_log2);
    const bool on = item < 2 * cv.kv_heads;
    const bool is_v = on && item >= cv.kv_heads;
    const int h = !on ? 0 : is_v ? item - cv.kv_heads : item;
    const int64_t ld = is_v ? p.ldv : p.ldk;
    const uint16_t* src = (is_v ? p.v : p.k) + (t0 - start + page_at) * ld + static_cast<int64_t>(h) * D;   // of row 0
    const int rot = is_v ? 0 : p.rot;
    int c0, c1;
    item_cols(j, rot, p.interleaved, c0, c1);
    float v[16];
    auto load = [&](int chunk) {
        const int row = chunk * CHUNK + sub;
        const int64_t from = min(max(row, lo), hi - 1);                // a row that is there
        const uint4 w0 = *reinterpret_cast<const uint4*>(src + from * ld + c0);
        const uint4 w1 = *reinterpret_cast<const uint4*>(src + from * ld + c1);
        float4 cs[4];
        if (rot) load_angles(p.cos_sin + clamp_row(page_at + row, p.table_rows) * rot, min(j, rot / 16 - 1), rot, cs);
        float a[8], b[8];
        unpack8_bf16(w0, a);
        unpack8_bf16(w1, b);
        if (j < rot / 16) rotate_item(p.interleaved, cs, a, b);
        const bool there = row >= lo && row < hi;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = there ? a[e] : 0.0f;
            v[8 + e] = there ? b[e] : 0.0f;
        }
    };

    // this call's largest magnitude
    float big = 0.0f;
    const int chunks = cv.page / CHUNK;
    int held = part;
    for (int c = part; c < chunks; c += ONE ? 1 << 20 : wpi) {
        load(c);
        held = c;
#pragma unroll
        for (int e = 0; e < 16; e += 2) big = max_abs_nan(big, v[e], v[e + 1]);
    }
    if (id < 0 || id >= cv.pages) return;                    // (the whole block's page)
    const int64_t ph = static_cast<int64_t>(id) * cv.kv_heads + h;
    int8_t* codes = (is_v ? cv.v : cv.k) + (ph << cv.page_log2) * D;
    float* scale = (is_v ? cv.v_scale : cv.k_scale) + ph;
    uint32_t amax = __reduce_max_sync(0xffffffffu, __float_as_uint(big));   // (as bits, a NaN is the largest)
    const float was = lo > 0 ? *scale : 0.0f;
    if (wpi > 1) {
        if (lane == 0) sh_max[warp] = amax;
        __syncthreads();
        amax = __reduce_max_sync(0xffffffffu, sh_max[warp - part + (lane & (wpi - 1))]);
    }
    if (!on) return;
    const float mine = __fdiv_rn(__uint_as_float(amax), 127.0f);
    // the larger of the two; a NaN of either stays
    const float now = was >= mine || was != was ? was : mine;

    if (lo > 0 && now != was) {
        const float ratio = __fdiv_rn(was, now);
        for (int i = part * 32 + lane; i < lo * D / 4; i += wpi * 32) {
            uint32_t w = reinterpret_cast<const uint32_t*>(codes)[i], o = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float c = static_cast<float>(static_cast<int8_t>(w >> (8 * e)));
                const float q = rintf(__fmul_rn(c, ratio));
                o |= (static_cast<uint32_t>(static_cast<int>(q)) & 0xFFu) << (8 * e);
            }
            reinterpret_cast<uint32_t*>(codes)[i] = o;
        }
    }
    const bool fast = now >= 1.1754943508222875e-38f && now < INFINITY;
    const float rcp = fast ? __frcp_rn(now) : 0.0f;
    for (int c = held; c >= 0; c -= ONE ? 1 << 20 : wpi) {
        if (!ONE && c != held) load(c);
        const int row = c * CHUNK + sub;
        if (row < lo || row >= hi) continue;
        int8_t* d = codes + row * D;
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = fast ? codes4(v + 4 * q, now, rcp) : codes4_slow(v + 4 * q, now);
        *reinterpret_cast<uint2*>(d + c0) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(d + c1) = make_uint2(w[2], w[3]);
    }
    __syncwarp();
    if (lane == 0 && part == 0) *scale = now;
}

// ------------------------------------------------------------------ reading back

constexpr int kRTok = 16;          // most tokens of one block

// bf16(code * scale) of each sequence's last cu[s + 1] - cu[s] tokens.  A token
// without a page (or before position 0, or past the table) reads as zeros.
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const KvReadParams p, const int per)
{
    __shared__ int64_t sh_ph[kRTok];       // page * kv_heads, or -1
    __shared__ int sh_row[kRTok];
    const CacheView& cv = p.c;
    pdl_wait();
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * per;
    const int tid = threadIdx.x;
    const int s = tid < 32 ? seq_of(cv.cu, cv.batch, t0, min(t0 + min(tid, per - 1), cv.tokens - 1)) : 0;
    if (tid < per && t0 + tid < cv.tokens) {
        int64_t first;
        int n, len;
        seq_bounds(cv, s, first, n, len);
        const int64_t pos = static_cast<int64_t>(len) - n + (t0 + tid - first);
        int id = -1;
        if (pos >= 0 && pos < min(len, capacity(cv))) id = cv.table[static_cast<int64_t>(s) * cv.ld_table + (pos >> cv.page_log2)];
        sh_ph[tid] = id >= 0 && id < cv.pages ? static_cast<int64_t>(id) * cv.kv_heads : -1;
        sh_row[tid] = static_cast<int>(pos & (cv.page - 1));
    }
    __syncthreads();
    const int per_head = cv.D / 16, per_tok = cv.kv_heads * per_head;
    const int n = static_cast<int>(min(static_cast<int64_t>(per), cv.tokens - t0)) * per_tok;
    for (int i = tid; i < n; i += kThreads) {
        const int k = i / per_tok, rest = i - k * per_tok;
        const int h = rest / per_head, j = rest - h * per_head;
        const int64_t o = ((t0 + k) * cv.kv_heads + h) * cv.D + 16 * j;
        const int64_t ph = sh_ph[k] < 0 ? 0 : sh_ph[k] + h;
        const int64_t at = ((ph << cv.page_log2) + sh_row[k]) * cv.D + 16 * j;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            uint16_t* out = (kv ? p.v : p.k) + o;
            uint4 w0 = make_uint4(0, 0, 0, 0), w1 = w0;
            if (sh_ph[k] >= 0) {
                const uint4 c = *reinterpret_cast<const uint4*>((kv ? cv.v : cv.k) + at);
                const float sc = (kv ? cv.v_scale : cv.k_scale)[ph];
                const uint32_t w[4] = {c.x, c.y, c.z, c.w};
                float a[8], b[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    a[e] = static_cast<float>(static_cast<int8_t>(w[e >> 2] >> (8 * (e & 3)))) * sc;
                    b[e] = static_cast<float>(static_cast<int8_t>(w[2 + (e >> 2)] >> (8 * (e & 3)))) * sc;
                }
                w0 = pack8(a);
                w1 = pack8(b);
            }
            reinterpret_cast<uint4*>(out)[0] = w0;
            reinterpret_cast<uint4*>(out)[1] = w1;
        }
    }
}

template <typename Kern, typename... Args>
cudaError_t launch(Kern kern, int64_t blocks, cudaStream_t stream, const Args&... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace

cudaError_t launch_kv_write(const KvWriteParams& p, cudaStream_t stream)
{
    const int64_t q_blocks = p.q ? (p.c.tokens + kQTok - 1) / kQTok : 0;
    // n tokens of a sequence touch at most n pages, and at most (n - 1) / page + 2
    const int64_t jobs = std::min<int64_t>(p.c.tokens, p.c.tokens / p.c.page + 2 * static_cast<int64_t>(p.c.batch));
    const int per_block = kWarps / std::min(p.c.page / chunk_rows(p.c.D), kWarps);       // items
    const int groups = (2 * p.c.kv_heads + per_block - 1) / per_block;
    const int64_t blocks = q_blocks + jobs * groups;
    if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
    const int qb = static_cast<int>(q_blocks);
    // Pages that eight warps hold (up to 32 rows of 128 or 64 of 64) need no loop over
    // chunks: without it 7,543 tokens in pages of 32 take 53 us, with it 57.
    const bool one = p.c.page / chunk_rows(p.c.D) <= kWarps;
    if (p.c.D == 128)
        return one ? launch(kv_write_kernel<128, true>, blocks, stream, p, qb, groups)
                   : launch(kv_write_kernel<128, false>, blocks, stream, p, qb, groups);
    return one ? launch(kv_write_kernel<64, true>, blocks, stream, p, qb, groups)
               : launch(kv_write_kernel<64, false>, blocks, stream, p, qb, groups);
}

cudaError_t launch_kv_read(const KvReadParams& p, cudaStream_t stream)
{
    // As many tokens a block as give each thread one vector.  8 heads of 128: 2.9 and 9.1 us
    // for 530 and 7,584 tokens by four a block, 5.4 and 10.8 by sixteen, 2.8 and 12.4 by one;
    // one head of 128: 3.0 us for 7,584 by sixteen, 4.3 by four.
    const int per = std::max(1, std::min(kRTok, kThreads / (p.c.kv_heads * p.c.D / 16)));
    return launch(kv_read_kernel, (p.c.tokens + per - 1) / per, stream, p, per);
}

}  // namespace w4a8
