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
// The write is one launch: some blocks turn the query heads of a few tokens
// each, the others each own one touched page (so no two blocks write one
// scale), a warp per (kv head, K or V).  Bound by HBM for prompts: q is read and
// written, k and v read, a byte per element written.
#include <algorithm>

#include "w4a8_common.cuh"
#include "w4a8_kernels.h"

namespace w4a8 {

namespace {

constexpr int kThreads = 256;
constexpr int kQTok = 4;           // tokens of one query block

__device__ __forceinline__ void rotate_pair(float& a, float& b, float c, float s)
{
    const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    a = x;
}

// Bounds of sequence s: its first token in the call, their number, its length
// after the call (kept inside the tensors).
__device__ __forceinline__ void seq_bounds(const CacheView& c, int s, int64_t& t0, int& n, int& len)
{
    t0 = min(static_cast<int64_t>(max(c.cu[s], 0)), c.tokens);
    const int64_t t1 = min(static_cast<int64_t>(max(c.cu[s + 1], 0)), c.tokens);
    n = static_cast<int>(max(t1 - t0, static_cast<int64_t>(0)));
    len = static_cast<int>(min(static_cast<int64_t>(max(c.kv_lens[s], 0)), static_cast<int64_t>(c.table_cols) << c.page_log2));
}

// The sequence that token t belongs to: the last s with cu[s] <= t (t >= cu[0]).
__device__ __forceinline__ int seq_of(const int32_t* cu, int batch, int64_t t)
{
    int lo = 0, hi = batch - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
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

__device__ __forceinline__ void rotate_item(int j, int rot, int interleaved, const float* cs, float (&a)[8], float (&b)[8])
{
    if (j >= rot / 16) return;
    const float4* cp = reinterpret_cast<const float4*>(cs + 8 * j);
    const float4* sp = reinterpret_cast<const float4*>(cs + rot / 2 + 8 * j);
    const float4 c0 = cp[0], c1 = cp[1], s0 = sp[0], s1 = sp[1];
    const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
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

// One code: rint(x / s) within +-127; 0 for a zero or non-finite scale.
__device__ __forceinline__ uint32_t code_of(float x, float s)
{
    const float q = fminf(fmaxf(rintf(__fdiv_rn(x, s)), -127.0f), 127.0f);
    return s > 0.0f && s < INFINITY ? static_cast<uint32_t>(static_cast<int>(q)) & 0xFFu : 0u;
}

__device__ __forceinline__ uint2 codes8(const float (&v)[8], float s)
{
    uint2 w;
    w.x = code_of(v[0], s) | (code_of(v[1], s) << 8) | (code_of(v[2], s) << 16) | (code_of(v[3], s) << 24);
    w.y = code_of(v[4], s) | (code_of(v[5], s) << 8) | (code_of(v[6], s) << 16) | (code_of(v[7], s) << 24);
    return w;
}

__global__ void __launch_bounds__(kThreads) kv_write_kernel(const KvWriteParams p, const int q_blocks)
{
    __shared__ int64_t sh_pos[kQTok];
    __shared__ int64_t sh_warp[kThreads / 32];
    __shared__ int64_t sh_run;
    __shared__ int sh_found, sh_local;

    const CacheView& cv = p.c;
    const int tid = threadIdx.x;
    pdl_launch_dependents();
    pdl_wait();

    if (static_cast<int>(blockIdx.x) < q_blocks) {
        // ---- query heads of kQTok tokens ----
        const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kQTok;
        if (tid < kQTok && t0 + tid < cv.tokens) {
            const int s = seq_of(cv.cu, cv.batch, t0 + tid);
            int64_t first;
            int n, len;
            seq_bounds(cv, s, first, n, len);
            sh_pos[tid] = clamp_row(static_cast<int64_t>(len) - n + (t0 + tid - first), p.table_rows);
        }
        __syncthreads();
        const int per_head = cv.D / 16, per_tok = p.q_heads * per_head;
        for (int i = tid; i < kQTok * per_tok; i += kThreads) {
            const int k = i / per_tok, rest = i - k * per_tok;
            const int64_t t = t0 + k;
            if (t >= cv.tokens) break;
            const int h = rest / per_head, j = rest - h * per_head;
            int c0, c1;
            item_cols(j, p.rot, p.interleaved, c0, c1);
            const uint16_t* src = p.q + t * p.ldq + static_cast<int64_t>(h) * cv.D;
            uint16_t* dst = p.q_out + t * p.ldqo + static_cast<int64_t>(h) * cv.D;
            float a[8], b[8];
            unpack8_bf16(*reinterpret_cast<const uint4*>(src + c0), a);
            unpack8_bf16(*reinterpret_cast<const uint4*>(src + c1), b);
            if (p.cos_sin) rotate_item(j, p.rot, p.interleaved, p.cos_sin + sh_pos[k] * p.rot, a, b);
            *reinterpret_cast<uint4*>(dst + c0) = pack8(a);
            *reinterpret_cast<uint4*>(dst + c1) = pack8(b);
        }
        return;
    }

    // ---- one touched page: find (sequence, page) number `job` ----
    const int64_t job = blockIdx.x - q_blocks;
    if (tid == 0) {
        sh_run = 0;
        sh_found = -1;
    }
    __syncthreads();
    for (int base = 0; base < cv.batch; base += kThreads) {
        const int s = base + tid;
        int64_t np = 0;
        if (s < cv.batch) {
            int64_t t0;
            int n, len;
            seq_bounds(cv, s, t0, n, len);
            const int lo = max(len - n, 0);          // tokens before position 0 are not written
            if (len > lo) np = ((len - 1) >> cv.page_log2) - (lo >> cv.page_log2) + 1;
        }
        int64_t x = np;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (static_cast<int>(lane_id()) >= o) x += y;
        }
        if (lane_id() == 31) sh_warp[warp_id()] = x;
        __syncthreads();
        int64_t before = sh_run;
        for (int w = 0; w < static_cast<int>(warp_id()); ++w) before += sh_warp[w];
        if (job >= before + x - np && job < before + x) {
            sh_found = s;
            sh_local = static_cast<int>(job - (before + x - np));
        }
        __syncthreads();
        if (tid == kThreads - 1) sh_run = before + x;
        __syncthreads();
        if (sh_found >= 0) break;
    }
    if (sh_found < 0) return;
    const int s = sh_found;
    int64_t t0;
    int n, len;
    seq_bounds(cv, s, t0, n, len);
    const int start = len - n;                               // position of the call's first token (may be < 0)
    const int pg = (max(start, 0) >> cv.page_log2) + sh_local;
    const int page_at = pg << cv.page_log2;
    const int lo = max(start - page_at, 0);                  // rows [0, lo): earlier tokens
    const int hi = min(len - page_at, cv.page);              // rows [max(lo, -start), hi): this call's
    const int first = max(lo, max(-page_at, 0));
    const int id = cv.table[static_cast<int64_t>(s) * cv.ld_table + pg];
    if (id < 0 || id >= cv.pages) return;

    const int per_row = cv.D / 16, rows = hi - first;
    for (int it = warp_id(); it < 2 * cv.kv_heads; it += kThreads / 32) {
        const int h = it >> 1;
        const bool is_v = it & 1;
        const int64_t ph = static_cast<int64_t>(id) * cv.kv_heads + h;
        int8_t* codes = (is_v ? cv.v : cv.k) + (ph << cv.page_log2) * cv.D;
        float* scale = (is_v ? cv.v_scale : cv.k_scale) + ph;
        const int64_t ld = is_v ? p.ldv : p.ldk;
        const uint16_t* src = (is_v ? p.v : p.k) + (t0 + (page_at + first - start)) * ld + static_cast<int64_t>(h) * cv.D;
        const bool turn = !is_v && p.cos_sin != nullptr;
        const int rot = is_v ? 0 : p.rot;

        // this call's largest magnitude, as bits (a NaN wins)
        uint32_t amax = 0;
        for (int i = lane_id(); i < rows * per_row; i += 32) {
            const int rw = i / per_row, j = i - rw * per_row;
            int c0, c1;
            item_cols(j, rot, p.interleaved, c0, c1);
            float a[8], b[8];
            unpack8_bf16(*reinterpret_cast<const uint4*>(src + rw * ld + c0), a);
            unpack8_bf16(*reinterpret_cast<const uint4*>(src + rw * ld + c1), b);
            if (turn)
                rotate_item(j, rot, p.interleaved, p.cos_sin + clamp_row(page_at + first + rw, p.table_rows) * rot, a, b);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                amax = max(amax, max(__float_as_uint(a[e]) & 0x7FFFFFFFu, __float_as_uint(b[e]) & 0x7FFFFFFFu));
        }
        amax = __reduce_max_sync(0xffffffffu, amax);
        const float mine = __fdiv_rn(__uint_as_float(amax), 127.0f);
        const float was = lo > 0 ? *scale : 0.0f;
        __syncwarp();
        // the larger of the two; a NaN of either stays
        const float now = was >= mine || was != was ? was : mine;

        if (lo > 0 && now != was) {
            const float ratio = __fdiv_rn(was, now);
            for (int i = lane_id(); i < lo * cv.D / 4; i += 32) {
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
        for (int i = lane_id(); i < rows * per_row; i += 32) {
            const int rw = i / per_row, j = i - rw * per_row;
            int c0, c1;
            item_cols(j, rot, p.interleaved, c0, c1);
            float a[8], b[8];
            unpack8_bf16(*reinterpret_cast<const uint4*>(src + rw * ld + c0), a);
            unpack8_bf16(*reinterpret_cast<const uint4*>(src + rw * ld + c1), b);
            if (turn)
                rotate_item(j, rot, p.interleaved, p.cos_sin + clamp_row(page_at + first + rw, p.table_rows) * rot, a, b);
            int8_t* d = codes + (first + rw) * cv.D;
            *reinterpret_cast<uint2*>(d + c0) = codes8(a, now);
            *reinterpret_cast<uint2*>(d + c1) = codes8(b, now);
        }
        if (lane_id() == 0) *scale = now;
    }
}

// ------------------------------------------------------------------ reading back

constexpr int kRTok = 16;          // tokens of one block

// bf16(code * scale) of each sequence's last cu[s + 1] - cu[s] tokens.  A token
// without a page (or before position 0) reads as zeros.
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const KvReadParams p)
{
    __shared__ int64_t sh_ph[kRTok];       // page * kv_heads, or -1
    __shared__ int sh_row[kRTok];
    const CacheView& cv = p.c;
    pdl_launch_dependents();
    pdl_wait();
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kRTok;
    const int tid = threadIdx.x;
    if (tid < kRTok && t0 + tid < cv.tokens) {
        const int s = seq_of(cv.cu, cv.batch, t0 + tid);
        int64_t first;
        int n, len;
        seq_bounds(cv, s, first, n, len);
        const int64_t pos = static_cast<int64_t>(len) - n + (t0 + tid - first);
        int id = -1;
        if (pos >= 0 && pos < len) id = cv.table[static_cast<int64_t>(s) * cv.ld_table + (pos >> cv.page_log2)];
        sh_ph[tid] = id >= 0 && id < cv.pages ? static_cast<int64_t>(id) * cv.kv_heads : -1;
        sh_row[tid] = static_cast<int>(pos & (cv.page - 1));
    }
    __syncthreads();
    const int per_head = cv.D / 16, per_tok = cv.kv_heads * per_head;
    const int n = static_cast<int>(min(static_cast<int64_t>(kRTok), cv.tokens - t0)) * per_tok;
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
    const int64_t jobs = p.k ? std::min<int64_t>(p.c.tokens, p.c.tokens / p.c.page + 2 * static_cast<int64_t>(p.c.batch)) : 0;
    if (q_blocks + jobs == 0) return cudaSuccess;
    return launch(kv_write_kernel, q_blocks + jobs, stream, p, static_cast<int>(q_blocks));
}

cudaError_t launch_kv_read(const KvReadParams& p, cudaStream_t stream)
{
    return launch(kv_read_kernel, (p.c.tokens + kRTok - 1) / kRTok, stream, p);
}

}  // namespace w4a8
