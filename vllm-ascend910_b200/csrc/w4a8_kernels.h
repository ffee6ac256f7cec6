// w4a8_kernels.h -- parameter blocks and launchers shared by the .cu files of
// libw4a8_b200.so (internal; the public C ABI is include/w4a8_b200.h).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace w4a8 {

enum QuantOutKind { kOutKernel = 0, kOutPublic = 1, kOutMsd = 2 };

struct QuantParams {
    const uint16_t* x;   // bf16 bits [M, ldx]
    int64_t ldx;
    int M, K, Kpad, G, gk;
    int swiglu;          // x holds [gate | up] ([M, 2K] within ldx): quantise bf16(silu(gate) * up)
    int rows;            // rows to emit: M, or Mp for the MSD form
    int vec_ok;          // 16-byte vector loads are legal for this x
    // kOutKernel: the GEMM's activation tiles (see gemm_act_tile_offset)
    int8_t* aq;          // [n_tt][kb_total][TT * 256] bytes, 128-byte swizzled
    float* as;           // [n_tt][G][TT]
    int tt, kb_total;
    // kOutPublic
    int8_t* q;           // [M, K]
    void* scale;         // [G, M] bf16 bits or fp32
    int scale_f32;
    int32_t* ksum;       // [G, M] or null
    // kOutMsd
    int8_t* a_hi;        // [rows, Kpad/2]
    int8_t* a_lo;
    uint16_t* a_scale;   // [G, rows]
    int32_t* a_ksum;     // [G, rows]
};

struct MsdToKernelParams {
    const int8_t* a_hi;      // [M, Kpad/2]
    const int8_t* a_lo;
    const uint16_t* a_scale; // [G, scale_ld] bf16 bits
    int scale_ld;
    int M, Kpad, G, gk;
    int rows;                // n_tt * tt: rows of the tile layout (>= M)
    int8_t* aq;              // activation tiles, as in QuantParams
    float* as;
    int tt, kb_total;
};

// Byte offset of activation code (row, padded position) inside the GEMM's
// activation tiles: tile (row / tt, pos / 256) holds tt rows x 256 codes as two
// halves of tt x 128 bytes, each in the 128-byte-swizzled order the MMA's
// shared-memory descriptor expects (16-byte chunk c of row r stored at chunk
// c ^ (r % 8)).  One 1-D bulk copy moves a tile.
__host__ __device__ inline int64_t gemm_act_tile_offset(int row, int pos, int tt, int kb_total)
{
    const int r = row % tt, t = row / tt, kb = pos >> 8, w = pos & 255;
    const int h = w >> 7, c = (w & 127) >> 4, b = w & 15;
    return (static_cast<int64_t>(t) * kb_total + kb) * (tt * 256) + h * (tt * 128) + r * 128 +
           ((c ^ (r & 7)) << 4) + b;
}

// Row-parallel output pushed to every rank (the fused GEMM + all-reduce): the
// bf16 result tile goes straight into slot [bank][rank] of every rank's
// one-shot all-reduce buffer instead of into y.  world == 0: no push.
struct PushParams {
    uint8_t* base[8];          // every rank's buffer as mapped in this process (own included)
    const uint32_t* counter;   // this rank's call counter of the all-reduce (block 0's)
    size_t slot_bytes, bank_bytes;
    int world, rank;
};

// The GEMM's view of one call.  Tensor maps are built on the host.
// k-blocks (256 K positions) per pipeline stage and stream-K unit when
// GK <= 256: two for 16-token tiles (32 KB of int4 weights per unit), one for
// wider tiles.  The host plan and the kernel's Cfg both take it from here.
__host__ __device__ constexpr int stage_kblocks(int tt) { return tt <= 16 ? 2 : 1; }

struct alignas(64) GemmParams {
    // raw (reference-layout) weights, read with 2-D tensor copies
    CUtensorMap tm_w;    // packed int4 weights [N, Kpad/2] bytes, box {128 B, 128 rows}, SW128
    CUtensorMap tm_ws;   // weight scales [G, N] (fp32 or bf16), box {128, GPK}
    CUtensorMap tm_wz;   // weight zero points [G, N] bf16, box {128, GPK} (asymmetric only)
    // prepared weights (w4a8_prepare_weights), read with 1-D bulk copies; null = raw path
    const uint8_t* w_tiles;   // [n_wt][kb_total][16384] swizzled packed int4 tiles
    const uint8_t* ws_tiles;  // [n_wt][G][128] scales (fp32 or bf16)
    const uint8_t* wz_tiles;  // [n_wt][G][128] bf16 zero points (asymmetric only)
    // activations from the quantiser, read with 1-D bulk copies
    const uint8_t* a_tiles;   // [n_tt][kb_total][TT * 256] (gemm_act_tile_offset)
    const float* as_tiles;    // [n_tt][G][TT]
    // fused quantisation (GemmConfig::fq): the bf16 activation itself, read with
    // 2-D tensor copies of 256 positions x TT rows (rows >= M and positions >= K
    // arrive as zeros) and quantised inside the GEMM
    CUtensorMap tm_x;    // x bf16 [M, K] (row stride ldx), box {256, TT}, no swizzle
    void* out;           // y bf16 [M, N] (row stride ldy), or int32 partials [G, M, N]
    float* partials;     // stream-K partial tiles: [2 * grid][TT][128] fp32
    int* status;         // device status word
    PushParams push;     // (fused all-reduce) where finished bf16 tiles go instead of out
    int M, N, Kpad, G;
    int64_t ldy;
    int n_wt, n_tt, units_per_tile, total_units, kb_total;
};

// Prepared weight layout: the packed int4 weights regrouped into one
// contiguous, pre-swizzled 16 KB tile per (128-row tile, 256-element k-block),
// followed by the scales and zero points regrouped per row tile.
struct PreparedLayout {
    int64_t off_tiles, off_ws, off_wz, total;
};

__host__ __device__ inline PreparedLayout prepared_layout(int64_t N, int64_t G, int kb_total, int ws_elt, bool zero)
{
    const int64_t n_wt = (N + 127) / 128;
    PreparedLayout L;
    L.off_tiles = 0;
    L.off_ws = n_wt * kb_total * 16384;
    L.off_wz = L.off_ws + ((n_wt * G * 128 * ws_elt + 255) / 256) * 256;
    L.total = L.off_wz + (zero ? ((n_wt * G * 128 * 2 + 255) / 256) * 256 : 0);
    return L;
}

struct PrepareParams {
    const uint8_t* w_packed;   // [N, Kpad/2]
    const uint8_t* w_scale;    // [G, N]
    const uint16_t* w_zero;    // [G, N] or null
    uint8_t* out;
    int N, Kpad, G, kb_total, ws_elt;
};

struct GemmConfig {
    int tt;        // token tile (MMA N): 16, 32, 64 or 128
    int gk;        // 64, 128, 256 or 1024
    bool asym;
    bool ws_bf16;
    bool partials; // debug mode: write int32 group partials instead of y
    bool fq;       // quantise the activation inside the GEMM (one token tile of 16, GK <= 256)
};

cudaError_t launch_quant_act(const QuantParams& p, int out_kind, cudaStream_t stream, bool pdl);
cudaError_t launch_prepare_weights(const PrepareParams& p, cudaStream_t stream);
cudaError_t launch_msd_to_kernel(const MsdToKernelParams& p, cudaStream_t stream, bool pdl);

// Launches the GEMM on `grid` persistent CTAs.  Returns cudaErrorInvalidValue
// for an unsupported configuration.
cudaError_t launch_gemm(const GemmParams& p, const GemmConfig& cfg, int grid, cudaStream_t stream,
                        bool pdl);
size_t gemm_smem_bytes(const GemmConfig& cfg);

// Sums the parts of output tiles split across GEMM CTAs (a programmatic
// dependent of the GEMM launched with the same parameters and grid).
cudaError_t launch_splitk_reduce(const GemmParams& p, int tt, int grid, cudaStream_t stream);


// ---- residual addition + root-mean-square norm (w4a8_norm.cu) ----
enum NormOutKind { kNormBf16 = 0, kNormCodes = 1, kNormTiles = 2 };

struct NormParams {
    const uint16_t* x;        // bf16 [M, ldx]
    const uint16_t* res;      // bf16 [M, ldr], or null
    const void* weight;       // [K] bf16 or fp32
    uint16_t* res_out;        // bf16 [M, ldro]: bf16(x + res), or null
    int64_t ldx, ldr, ldro;
    float eps;
    int weight_f32;
    int M, K;
    int rows;                 // rows to emit: M, or whole token tiles (kNormTiles)
    int vec_x, vec_r, vec_ro, vec_w, vec_y, vec_q;   // 16-byte (codes: 8-byte) accesses are legal
    // kNormBf16
    uint16_t* y;              // bf16 [M, ldy]
    int64_t ldy;
    // kNormCodes
    int gk, G;
    int8_t* q;                // [M, K]
    void* scale;              // [G, M] bf16 bits or fp32
    int scale_f32;
    // kNormTiles: as QuantParams' kOutKernel form
    int8_t* aq;
    float* as;
    int tt, kb_total;
};

cudaError_t launch_rms_norm(const NormParams& p, int out_kind, cudaStream_t stream);

// ---- paged 8-bit cache (w4a8_kvcache.cu) and attention over it (w4a8_attention.cu) ----

// One layer's cache and the batch of sequences that a call works on.
struct CacheView {
    int8_t* k;                // [pages][kv_heads][page][D]
    int8_t* v;
    float* k_scale;           // [pages][kv_heads]
    float* v_scale;
    const int32_t* table;     // page ids [batch][ld_table]
    const int32_t* kv_lens;   // [batch] tokens in the cache, this call's included
    const int32_t* cu;        // [batch + 1] offsets of each sequence's tokens in this call
    int64_t ld_table, pages, tokens;
    int table_cols, batch, kv_heads, page, page_log2, D;
};

// Rotary positions of their own on up to kMaxAxes axes: row positions[a * ld + t] of the table for
// the pairs of axis a; pair i's axis is bits 2 (i % 32) of map[i / 32].
constexpr int kMaxAxes = 4;
constexpr int kMaxRotaryDim = 256;
struct AxesView {
    const int32_t* positions;
    int64_t ld;
    int axes;                 // 0: by the token's place in its sequence
    uint64_t map[4];
};

struct KvWriteParams {
    CacheView c;
    const uint16_t* q;        // bf16 [tokens, ldq] of q_heads * D, or null
    const uint16_t* k;        // bf16 [tokens, ldk] of kv_heads * D
    const uint16_t* v;
    uint16_t* q_out;          // bf16 [tokens, ldqo]
    const float* cos_sin;     // [table_rows, rot]: cos of rot / 2 angles, then sin; null: no rotation
    int64_t ldq, ldk, ldv, ldqo, table_rows;
    int q_heads, rot, interleaved;
    AxesView axes;
};

struct RotaryParams {
    const uint16_t* x[2];     // q and k: bf16 [tokens, ld] of heads * D; k may be null
    uint16_t* out[2];
    int64_t ld[2], ldo[2];
    int heads[2];
    const float* cos_sin;     // as in KvWriteParams
    int64_t tokens, table_rows;
    int D, rot, interleaved;
    AxesView axes;
};

struct KvReadParams {
    CacheView c;              // cu: offsets of the tokens to read (each sequence's last ones)
    uint16_t* k;              // bf16 [tokens, kv_heads, D]
    uint16_t* v;
};

struct AttentionParams {
    CacheView c;
    const uint16_t* q;        // bf16 [tokens, ldq] of q_heads * D
    uint16_t* out;            // bf16 [tokens, ldo]
    int64_t ldq, ldo;
    int q_heads, group;       // group: query heads per kv head
    uint64_t group_magic;     // floor(2^64 / group) + 1 (0 for group 1): see row_token
    int max_q;                // no sequence has more query tokens (host's knowledge)
    float scale_log2;         // softmax scale * log2(e)
    int segments;             // about how many row tiles there are, of all heads and sequences (host's estimate)
    int few_most;             // attend_few_kernel takes sequences of at most this many packed rows
    int* status;              // workspace: status word
    uint32_t* calls;          // workspace: CTAs of attend_few_kernel that have started, modulo four calls' worth
    uint32_t* tickets;        // workspace: counters beside it, a word per CTA, a byte of it per call (modulo four)
    uint8_t* ws;              // workspace past the status block
};

cudaError_t launch_kv_write(const KvWriteParams& p, cudaStream_t stream);
cudaError_t launch_kv_read(const KvReadParams& p, cudaStream_t stream);
cudaError_t launch_rotary(const RotaryParams& p, cudaStream_t stream);
// Bytes of p.ws that a call of these sizes needs.
size_t attention_ws_bytes(int batch, int64_t tokens, int q_heads, int kv_heads, int D, int max_q, int sms);
cudaError_t launch_attention(const AttentionParams& p, int sms, cudaStream_t stream);

// ---- pages kept on the device (w4a8_pages.cu) ----
constexpr int kMaxPlanBatch = 2048;        // sequences of a step
constexpr int kMaxPlanRows = 65536;        // sequences of a state

// Why a step was refused: bits of the state's status word (W4A8_PLAN_* of the C ABI).
enum : int { kPlanRow = 1, kPlanCount = 2, kPlanTokens = 4, kPlanPages = 8, kPlanColumns = 16, kPlanState = 32 };

struct PagesParams {
    int32_t* free;            // stack of free pages [pages]
    int32_t* free_count;      // its height
    int32_t* table;           // pages held [sequences][columns]
    int32_t* lens;            // tokens held [sequences]
    int* status;
    uint32_t* ticket;         // blocks of the running call that are done; 0 between calls
    int pages, sequences, columns, page_log2;
    const int32_t* rows;      // [batch] the step's sequences
    const int32_t* counts;    // [batch] tokens that each brings; shrink: tokens it keeps, or null
    int batch, axes, n_segs;
    int64_t tokens;           // room of slots and positions
    const int32_t* seg_cu;    // [batch + 1] grids of each sequence, or null
    const int32_t* segs;      // [n_segs] of start, t, h, w
    int32_t* page_table;      // [batch][columns]
    int32_t* kv_lens;         // [batch]
    int32_t* cu;              // [batch + 1]
    int32_t* slots;           // [tokens], or null
    int32_t* positions;       // [axes][tokens], or null
};

cudaError_t launch_pages_plan(const PagesParams& p, cudaStream_t stream);
cudaError_t launch_pages_shrink(const PagesParams& p, cudaStream_t stream);

// ---- linears in 8-bit integers: token quantiser (w4a8_int8_quant.cu), product (w4a8_int8_gemm.cu) ----
enum TokenSource { kTokPlain = 0, kTokSwiglu = 1, kTokNorm = 2 };

struct TokenQuantParams {
    const uint16_t* x;        // bf16 [M, ldx]; kTokSwiglu: [gate | up], 2 K used
    int64_t ldx;
    int M, K;
    int vec_x, vec_r, vec_ro, vec_w, vec_q;   // 16-byte (codes: 8-byte) accesses are legal
    int8_t* q;                // [M, ldq]
    int64_t ldq;
    float* scale;             // [M]
    // kTokNorm
    const uint16_t* res;      // bf16 [M, ldr], or null
    uint16_t* res_out;        // bf16 [M, ldro], or null
    int64_t ldr, ldro;
    const void* weight;       // [K] bf16 or fp32
    int weight_f32;
    float eps;
};

cudaError_t launch_token_quant(const TokenQuantParams& p, int source, cudaStream_t stream);

struct alignas(64) Int8GemmParams {
    CUtensorMap tm_w;         // int8 weights [N, K], boxes of 128 bytes x the kernel's rows, SW128
    CUtensorMap tm_a;         // int8 codes [M, K], likewise
    const float* a_scale;     // [M]
    const float* w_scale;     // [N]
    const float* bias;        // [N] or null
    uint16_t* y;              // bf16 [M, ldy]
    int64_t ldy;
    int* status;              // device status word
    int M, N, K;
};

// How a call runs: tiles of one CTA with 128 channels x tt tokens, K cut over a cluster of
// `split` CTAs (few), or of a pair of CTAs with nt channels x 256 tokens (many).
struct Int8Plan {
    bool many;
    int tt, split, nt;
    int w_rows, a_rows;       // rows of the tensor maps' boxes
};
Int8Plan int8_plan(int64_t M, int64_t N, int64_t K, int sms);
cudaError_t launch_int8_gemm(const Int8GemmParams& p, const Int8Plan& plan, int sms, cudaStream_t stream, bool pdl);

// Host helpers of the C entry points (w4a8_capi.cu).
int capi_device_sms(int* sms);
int capi_fail_cuda(cudaError_t e);
// Tensor map of bytes [rows, cols] with row_bytes from row to row, boxes of box_rows x 128 bytes,
// 128-byte swizzled; zeros outside.
int capi_bytes_map(CUtensorMap* m, const void* base, int64_t cols, int64_t rows, int64_t row_bytes, int box_rows);

// The one-shot all-reduce's side of the fused row-parallel linear
// (w4a8_allreduce.cu): where a GEMM must push a message of `bytes`, and the
// reduction that follows the pushes (flags, bounded waits, rank-order sum).
}  // namespace w4a8
struct w4a8_ar;
namespace w4a8 {
// pull: the GEMM stores into this rank's own slot only and the reduction reads
// the peers' slots; otherwise the GEMM stores into every rank's slot.
int ar_push_params(const w4a8_ar* h, size_t bytes, bool pull, PushParams* out);
cudaError_t ar_launch_reduce_pushed(w4a8_ar* h, void* out, int64_t count, bool pull, cudaStream_t stream);

}  // namespace w4a8
