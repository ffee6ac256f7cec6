/*
 * w4a8_b200.h -- C ABI of libw4a8_b200.so, the B200 (sm_100a) mid-group W4A8
 * linear layer.
 *
 * All tensor arguments are raw device pointers to densely packed row-major
 * arrays; bf16 values are 16-bit patterns.  `stream` is a cudaStream_t (NULL =
 * legacy default stream).  Every call is asynchronous on `stream`, allocates
 * no memory, and returns W4A8_OK or a negative status.  Asynchronous failures
 * inside a kernel (a pipeline wait that ran out) are recorded in the
 * workspace's status word: read it with w4a8_workspace_status().
 *
 * Layout conventions (the reference's; mg_kgeom.h in the reference project):
 *   G    = ceil(K / group_size)                       -- w4a8_num_groups()
 *   Kpad = group-padded row length (each group padded to 64 elements;
 *          only the last group can pad when group_size % 64 == 0)
 *   packed int4 weights: [N, Kpad/2] bytes, two codes per byte, even k in the
 *          low nibble, codes in [-8, 7]
 *   scales / zero points: group-major [G, N] (weights), [G, M] (activations)
 *   zero points: integers in code units held in bf16 (asymmetric weights)
 *
 * Each entry point cites the reference interface it replaces.
 */
#ifndef W4A8_B200_H
#define W4A8_B200_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define W4A8_API __attribute__((visibility("default")))
#else
#define W4A8_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

#define W4A8_OK 0
#define W4A8_ERR_INVALID (-1)     /* bad shape, null or misaligned pointer       */
#define W4A8_ERR_UNSUPPORTED (-2) /* group size / dtype not built                */
#define W4A8_ERR_CUDA (-3)        /* a CUDA call failed: w4a8_last_cuda_error()  */
#define W4A8_ERR_WORKSPACE (-4)   /* workspace missing or smaller than required  */
#define W4A8_ERR_DEVICE (-5)      /* current device is not an sm_100 part         */
#define W4A8_ERR_TIMEOUT (-6)     /* a device-side wait on a peer ran out          */

#define W4A8_DTYPE_BF16 0
#define W4A8_DTYPE_F32 1

/* ---- geometry (npu_ops/python/w4a8_ops.py:63-82,160-178; mg_kgeom.h:64-101) ---- */
W4A8_API int64_t w4a8_num_groups(int64_t K, int32_t group_size);
W4A8_API int64_t w4a8_k_pad_elems(int64_t K, int32_t group_size);
/* Rows `midgroup_quant_a` emits for M rows: M rounded up to 16 / 64 / 128
 * (TileMFor, npu_ops/host/midgroup_quant_a.cpp:37). */
W4A8_API int64_t w4a8_pad_rows(int64_t M);

/* ---- fused linear: y = x @ W^T, activation quantised per (token, group) ----
 * Replaces MidGroupW4A8LinearMethod.apply's quant_a -> gemm pair
 * (npu_ops/python/midgroup_quant.py:163-178, w4a8_ops.py:243-252).
 *   x        bf16 [M, ldx] (ldx >= K)
 *   w_packed int8 [N, Kpad/2]            (16-byte aligned)
 *   w_scale  [G, N] bf16 or f32 (w_scale_dtype)
 *   w_zero   [G, N] bf16, or NULL for symmetric weights
 *   y        bf16 [M, ldy] (ldy >= N)
 * group_size in {64, 128, 256, 1024}; N % 8 == 0.
 * The workspace (w4a8_linear_workspace_size bytes, 1024-byte aligned) must be
 * zero-filled before its first use; calls leave it reusable.  Calls that share
 * a workspace must not overlap in time (use one workspace per stream). */
W4A8_API size_t w4a8_linear_workspace_size(int64_t M, int64_t N, int64_t K, int32_t group_size);
W4A8_API int w4a8_linear(const void* x, int64_t M, int64_t K, int64_t ldx, int64_t N, int32_t group_size,
                const void* w_packed, const void* w_scale, int32_t w_scale_dtype,
                const void* w_zero, void* y, int64_t ldy, void* workspace, size_t workspace_bytes,
                void* stream);

/* ---- the down projection with the SwiGLU activation applied to its input ----
 * y = bf16(silu(gate) * up) @ W^T for gu = [gate | up], bf16 [M, ldx] with
 * ldx >= 2K: gate = columns [0, K), up = columns [K, 2K) (vLLM's
 * MergedColumnParallelLinear output order).  silu(g) = g / (1 + exp(-g)) and
 * the product are computed in fp32 and rounded to bf16 before quantisation,
 * as the reference's layer does in torch before its quant op
 * (F.silu(g) * u in npu_ops/python/bench_decode_layer.py:81; torch_npu.npu_swiglu
 * in npu_ops/python/bench_decode_graph.py:64), so no [M, K] activation tensor
 * and no elementwise kernel sit between gate_up and down.  Otherwise as
 * w4a8_linear (same weights, workspace and rules; K is the down projection's). */
W4A8_API int w4a8_linear_swiglu(const void* gu, int64_t M, int64_t K, int64_t ldx, int64_t N, int32_t group_size,
                                const void* w_packed, const void* w_scale, int32_t w_scale_dtype,
                                const void* w_zero, void* y, int64_t ldy, void* workspace, size_t workspace_bytes,
                                void* stream);

/* The two halves of w4a8_linear, for callers that quantise once and reuse the
 * quantised activation, or time the GEMM alone.  w4a8_linear_gemm reads the
 * activation w4a8_linear_quant left in the same workspace (same M, K). */
W4A8_API int w4a8_linear_quant(const void* x, int64_t M, int64_t K, int64_t ldx, int64_t N,
                      int32_t group_size, void* workspace, size_t workspace_bytes, void* stream);
W4A8_API int w4a8_linear_gemm(int64_t M, int64_t K, int64_t N, int32_t group_size, const void* w_packed,
                     const void* w_scale, int32_t w_scale_dtype, const void* w_zero, void* y,
                     int64_t ldy, void* workspace, size_t workspace_bytes, void* stream);

/* ---- prepared weights: the fast path for weights that are used many times ----
 * One-time regrouping of the reference layout (packed int4 [N, Kpad/2], scales
 * and zero points [G, N]) into contiguous, pre-swizzled 16 KB tiles plus
 * per-row-tile scale rows, so each pipeline stage is filled by one bulk copy.
 * Plays the part of MidGroupW4A8LinearMethod.process_weights_after_loading
 * (npu_ops/python/midgroup_quant.py:148-161), which also re-lays scales once
 * after loading.  `prepared` must be 256-byte aligned. */
W4A8_API size_t w4a8_prepared_weights_size(int64_t N, int64_t K, int32_t group_size, int32_t w_scale_dtype,
                                           int32_t has_zero);
W4A8_API int w4a8_prepare_weights(const void* w_packed, const void* w_scale, int32_t w_scale_dtype,
                                  const void* w_zero, int64_t N, int64_t K, int32_t group_size, void* prepared,
                                  size_t prepared_bytes, void* stream);
/* w4a8_linear on prepared weights (same workspace rules). */
W4A8_API int w4a8_linear_prepared(const void* x, int64_t M, int64_t K, int64_t ldx, int64_t N, int32_t group_size,
                                  const void* prepared, int32_t w_scale_dtype, int32_t has_zero, void* y,
                                  int64_t ldy, void* workspace, size_t workspace_bytes, void* stream);
/* w4a8_linear_swiglu on prepared weights. */
W4A8_API int w4a8_linear_prepared_swiglu(const void* gu, int64_t M, int64_t K, int64_t ldx, int64_t N,
                                         int32_t group_size, const void* prepared, int32_t w_scale_dtype,
                                         int32_t has_zero, void* y, int64_t ldy, void* workspace,
                                         size_t workspace_bytes, void* stream);
/* The GEMM half of w4a8_linear_prepared (after w4a8_linear_quant on the same workspace). */
W4A8_API int w4a8_linear_gemm_prepared(int64_t M, int64_t K, int64_t N, int32_t group_size, const void* prepared,
                                       int32_t w_scale_dtype, int32_t has_zero, void* y, int64_t ldy,
                                       void* workspace, size_t workspace_bytes, void* stream);

/* ---- w4a8_linear without a caller-provided workspace ----
 * No counterpart in the reference.  Same arguments, checks and results as
 * w4a8_linear minus the workspace: its scratch is one fixed
 * W4A8_FIXED_SCRATCH_BYTES array of device memory per device, declared in the
 * library itself, so the call allocates nothing.  For callers that cannot
 * allocate device memory at the call site: foreign-language hosts that hold
 * no device allocator, and serving loops whose allocator must not be entered
 * (cudaMalloc synchronises the device; a caching allocator may be in a
 * no-growth phase).
 *   - Returns W4A8_ERR_WORKSPACE when the call would need more scratch than
 *     the array holds (16 MiB covers M <= 64 on 27648 x 7168 weights).
 *   - The first call on a device looks the array up, clears it and waits for
 *     the clear on `stream`: make that first call before any stream capture.
 *     The same happens again on the first call after the device's context
 *     was reset (the module, and with it the array, is loaded anew).
 *   - Every call on a device shares the one array: calls that overlap in time
 *     (different streams, threads) race on it and must be serialised by the
 *     caller.
 *   - A kernel wait that runs out is recorded in the array's status word:
 *     read (and clear) it with w4a8_fixed_scratch_status. */
#define W4A8_FIXED_SCRATCH_BYTES ((size_t)16 << 20)
W4A8_API int w4a8_linear_fixed_scratch(const void* x, int64_t M, int64_t K, int64_t ldx, int64_t N,
                                       int32_t group_size, const void* w_packed, const void* w_scale,
                                       int32_t w_scale_dtype, const void* w_zero, void* y, int64_t ldy,
                                       void* stream);
/* Status word of the current device's fixed scratch, as w4a8_workspace_status
 * returns it for a workspace (synchronises `stream`; reset != 0 clears it).
 * No counterpart in the reference.  W4A8_ERR_WORKSPACE when no
 * w4a8_linear_fixed_scratch call has run in the current context yet. */
W4A8_API int w4a8_fixed_scratch_status(int32_t reset, void* stream);

/* ---- activation quantiser (fakequant_lab/quant.py:89-141 semantics) ----
 *   a_q       int8 [M, K] natural order
 *   a_scale   [G, M] bf16 bits or f32 (scale_dtype)
 *   a_ksum    int32 [G, M] NEGATED per-group code sums, or NULL */
W4A8_API int w4a8_quant_act(const void* x, int64_t M, int64_t K, int64_t ldx, int32_t group_size,
                   int8_t* a_q, void* a_scale, int32_t scale_dtype, int32_t* a_ksum, void* stream);

/* ---- the reference op torch.ops.npu.midgroup_quant_a ----
 * (npu_ops/host/midgroup_quant_a.cpp:40-78; schema :87-90).  Emits Mp rows
 * (Mp >= M; rows [M, Mp) encode zero with scale = bf16 tiny):
 *   a_hi, a_lo int8 [Mp, Kpad/2]   MSD int4 planes: q = 16*hi + lo + 8
 *   a_scale    bf16 [G, Mp]
 *   a_ksum     int32 [G, Mp]       negated code sums */
W4A8_API int w4a8_midgroup_quant_a(const void* x, int64_t M, int64_t K, int32_t group_size, int64_t Mp,
                          int8_t* a_hi, int8_t* a_lo, void* a_scale, int32_t* a_ksum, void* stream);

/* ---- the reference op torch.ops.npu.midgroup_w4a8_gemm ----
 * (npu_ops/host/midgroup_w4a8_gemm.cpp:143-238; schema :249-250).  Computes the
 * definition form y = sum_g as*ws*sum_k A*(W - wz) from the MSD planes
 * (ReferenceMidGroupGemm, int4_cube_lab/host/gemm_ref.cpp:199-240); a_ksum and
 * w_ksum are the MSD bookkeeping of the reference kernel and are not needed by
 * this path (they may be NULL).  M = rows of a_hi; y bf16 [M, N].
 * Workspace: w4a8_midgroup_gemm_workspace_size bytes, zero-filled before first use. */
W4A8_API size_t w4a8_midgroup_gemm_workspace_size(int64_t M, int64_t N, int64_t K, int32_t group_size);
W4A8_API int w4a8_midgroup_w4a8_gemm(const int8_t* a_hi, const int8_t* a_lo, const void* a_scale,
                            const int32_t* a_ksum, int64_t M, const int8_t* w_q,
                            const void* w_scale, const int32_t* w_ksum, const void* w_zero,
                            int64_t N, int64_t K, int32_t group_size, void* y, void* workspace,
                            size_t workspace_bytes, void* stream);

/* ---- int32 per-group partials P[g, m, n] = sum_{k in g} A_q*(W - wz) ----
 * The exactness contract of the reference (fakequant_lab/run_selftest.py:104-141,
 * int4_cube_lab/host/ragged_layout_test.cpp:112-148), computed by the same
 * tensor-core path as w4a8_linear.  partials int32 [G, M, N].  Test-sized
 * problems; workspace as for w4a8_linear. */
W4A8_API int w4a8_group_partials(const void* x, int64_t M, int64_t K, int64_t ldx, int64_t N,
                        int32_t group_size, const void* w_packed, const void* w_zero,
                        int32_t* partials, void* workspace, size_t workspace_bytes, void* stream);

/* ---- one-shot all-reduce over peer memory (tensor-parallel row reductions) ----
 * Replaces the reference's peer-read all-reduce (npu_ops/kernel/peer_allreduce_f32.cpp:127-270,
 * driven from npu_ops/python/peer_allreduce.py) for small bf16 messages.  One
 * handle per rank and device; every rank of the group calls
 * w4a8_ar_allreduce_bf16 in the same order with the same count.
 *   create:     allocates one buffer of two message slots of max_bytes plus flags
 *               (max_bytes a multiple of 16); world <= 8.
 *   ipc_handle: this rank's CUDA IPC handle (w4a8_ar_ipc_handle_size() bytes);
 *   open_peers: `handles` = world handles concatenated in rank order (own ignored).
 *   allreduce:  out[i] = bf16(sum over ranks, in rank order, of in[i] in fp32);
 *               count a multiple of 8 elements, count * 2 <= max_bytes, in / out
 *               16-byte aligned, in == out allowed.  Graph-capturable.  A wait for
 *               a peer is bounded (1 s): on expiry the call leaves its output
 *               untouched and records the failure, which w4a8_ar_status returns
 *               as W4A8_ERR_TIMEOUT (after the stream's work is done).
 * This entry point allocates device memory in create (nothing at call time). */
typedef struct w4a8_ar w4a8_ar;
W4A8_API size_t w4a8_ar_ipc_handle_size(void);
W4A8_API int w4a8_ar_create(int32_t rank, int32_t world, size_t max_bytes, w4a8_ar** out);
W4A8_API int w4a8_ar_ipc_handle(w4a8_ar* h, void* handle_out);
W4A8_API int w4a8_ar_open_peers(w4a8_ar* h, const void* handles);
/* Same, for ranks driven from this process (peers[r] = rank r's handle, own
 * ignored; on other devices peer access is enabled). */
W4A8_API int w4a8_ar_open_local(w4a8_ar* h, w4a8_ar* const* peers);
W4A8_API size_t w4a8_ar_max_bytes(const w4a8_ar* h);
W4A8_API int w4a8_ar_allreduce_bf16(w4a8_ar* h, const void* in, void* out, int64_t count, void* stream);
W4A8_API int w4a8_ar_status(w4a8_ar* h, int32_t reset);
W4A8_API int w4a8_ar_destroy(w4a8_ar* h);

/* ---- row-parallel linear fused with its all-reduce (tensor parallelism) ----
 * y = sum over the ranks of ar's group, in rank order in fp32 and rounded once
 * to bf16, of this rank's w4a8_linear_prepared result (x: the rank's K shard;
 * act = W4A8_ACT_SWIGLU takes x = [gate | up] as w4a8_linear_prepared_swiglu).
 * Every rank calls it in the same order with the same M and N, like
 * w4a8_ar_allreduce_bf16; M * N * 2 <= w4a8_ar_max_bytes(ar), (M * N) % 8 == 0,
 * y dense [M, N] and 16-byte aligned.  The GEMM's epilogue (and its stream-K
 * fix-up, for output tiles split between CTAs) stores each finished bf16 tile
 * straight into this rank's receive slot of the all-reduce buffer, and one
 * reduction kernel then publishes this rank's flags, waits (bounded, 1 s) for
 * the others' and sums every rank's slot in place with peer loads: the
 * partial output's own buffer and the all-reduce's copy pass are gone
 * (W4A8_OPT_AR_PUSH: the epilogue stores into every rank's slot instead).  The same bits as w4a8_linear_prepared
 * followed by w4a8_ar_allreduce_bf16.  A wait that runs out leaves y
 * untouched and is reported by w4a8_ar_status.  Replaces the reference's
 * row-parallel GEMM + peer all-reduce pair, fused as its design notes
 * propose (MGCKPT/P6.5_TP.md:900-957; npu_ops/kernel/peer_allreduce_f32.cpp:127-270). */
#define W4A8_ACT_NONE 0
#define W4A8_ACT_SWIGLU 1
W4A8_API int w4a8_linear_prepared_allreduce(const void* x, int64_t M, int64_t K, int64_t ldx, int64_t N,
                                            int32_t group_size, const void* prepared, int32_t w_scale_dtype,
                                            int32_t has_zero, int32_t act, void* y, void* workspace,
                                            size_t workspace_bytes, w4a8_ar* ar, void* stream);

/* ---- residual addition + root-mean-square norm ----
 *   h = x + residual (fp32; residual NULL: h = x), residual_out = bf16(h)
 *   y = h / sqrt(sum(h^2) / K + eps) * weight    (fp32, rounded once to bf16)
 * The step between a decoder layer's linears, which the reference leaves to its
 * host framework; no counterpart in its operator surface.
 *   x, residual, residual_out, y   bf16 [M, ld] (ld >= K); residual_out may be
 *                                  NULL, and may be x or residual itself
 *   weight                         [K] bf16 or f32 (weight_dtype)
 * 1 <= K <= W4A8_NORM_MAX_K. */
#define W4A8_NORM_MAX_K 32768
W4A8_API int w4a8_rms_norm(const void* x, int64_t M, int64_t K, int64_t ldx, const void* residual, int64_t ldr,
                           void* residual_out, int64_t ldro, const void* weight, int32_t weight_dtype, float eps,
                           void* y, int64_t ldy, void* stream);
/* The same norm with the output quantised by the activation quantiser's rule
 * (w4a8_quant_act) from its fp32 values, without a rounding to bf16 between:
 * a_q int8 [M, K], a_scale [G, M] bf16 or f32. */
W4A8_API int w4a8_rms_norm_quant(const void* x, int64_t M, int64_t K, int64_t ldx, const void* residual, int64_t ldr,
                                 void* residual_out, int64_t ldro, const void* weight, int32_t weight_dtype, float eps,
                                 int32_t group_size, int8_t* a_q, void* a_scale, int32_t scale_dtype, void* stream);
/* w4a8_linear_prepared on the norm's quantised output: the norm kernel writes
 * codes and scales straight into the GEMM's operand tiles in the workspace
 * (those of w4a8_rms_norm_quant), in place of the activation quantiser. */
W4A8_API int w4a8_linear_prepared_rms_norm(const void* x, int64_t M, int64_t K, int64_t ldx, const void* residual,
                                           int64_t ldr, void* residual_out, int64_t ldro, const void* weight,
                                           int32_t weight_dtype, float eps, int64_t N, int32_t group_size,
                                           const void* prepared, int32_t w_scale_dtype, int32_t has_zero, void* y,
                                           int64_t ldy, void* workspace, size_t workspace_bytes, void* stream);

/* ---- linears in 8-bit integers ----
 * One scale per token, one per output channel (the vendor's W8A8_DYNAMIC projections;
 * the reference has such a linear as its comparison arm, npu_ops/python/vllm_engine_patch.py:107-158):
 *   s[t] = max|h[t]| / 127,  q[t, k] = rint(h[t, k] / s[t])     (IEEE fp32, half-even)
 *   y[t, n] = bf16(sum_k q[t, k] w[n, k] * s[t] * w_scale[n] + bias[n])
 * with exact 32-bit integer sums, the sum's scales and bias applied in fp32 in this order.
 * A token of zeros has scale 0; one with a value that is not finite has scale NaN, and its row of
 * y is NaN.  h is x; bf16(silu(gate) * up) of x = [gate | up] with act = W4A8_ACT_SWIGLU
 * (ldx >= 2 K); or the root-mean-square norm of x (+ residual) as w4a8_rms_norm, in fp32.
 *   x          bf16 [M, ldx]
 *   w          int8 [N, ldw], ldw >= K a multiple of 16, 16-byte aligned
 *   w_scale    f32 [N];  bias f32 [N] or NULL
 *   y          bf16 [M, ldy]
 * 1 <= K <= W4A8_INT8_MAX_K (with a norm: W4A8_NORM_MAX_K); M, N <= 2^24.
 * Workspace: w4a8_int8_workspace_size bytes, rules as for the linear calls, with which it
 * may be shared in stream order. */
#define W4A8_INT8_MAX_K 131071
W4A8_API size_t w4a8_int8_workspace_size(int64_t M, int64_t K);
/* The token quantiser alone: q int8 [M, ldq], scale f32 [M]. */
W4A8_API int w4a8_int8_quant(const void* x, int64_t M, int64_t K, int64_t ldx, int32_t act, int8_t* q, int64_t ldq,
                             float* scale, void* stream);
/* The product alone, on codes q int8 [M, ldq] (16-byte aligned, ldq a multiple of 16) and their scales.
 * Codes may be -128..127.  workspace: 1024 bytes for the status word. */
W4A8_API int w4a8_int8_gemm(const int8_t* q, int64_t ldq, const float* scale, int64_t M, int64_t K, const int8_t* w,
                            int64_t ldw, const float* w_scale, const float* bias, int64_t N, void* y, int64_t ldy,
                            void* workspace, size_t workspace_bytes, void* stream);
W4A8_API int w4a8_int8_linear(const void* x, int64_t M, int64_t K, int64_t ldx, int32_t act, const int8_t* w, int64_t ldw,
                              const float* w_scale, const float* bias, int64_t N, void* y, int64_t ldy, void* workspace,
                              size_t workspace_bytes, void* stream);
/* Behind a norm: residual, residual_out, weight and eps as in w4a8_rms_norm. */
W4A8_API int w4a8_int8_linear_rms_norm(const void* x, int64_t M, int64_t K, int64_t ldx, const void* residual, int64_t ldr,
                                       void* residual_out, int64_t ldro, const void* weight, int32_t weight_dtype,
                                       float eps, const int8_t* w, int64_t ldw, const float* w_scale, const float* bias,
                                       int64_t N, void* y, int64_t ldy, void* workspace, size_t workspace_bytes,
                                       void* stream);

/* ---- paged 8-bit key / value cache ----
 * No counterpart in the reference (its serving stack keeps a bf16 cache).  One
 * layer's cache: int8 codes [pages, kv_heads, page_size, head_dim] and one fp32
 * scale per (page, kv head), for k and v each; value = code * scale.
 * page_size 16, 32, 64 or 128; head_dim 64 or 128; codes 16-byte aligned.
 *
 * The batch arguments of the calls below:
 *   page_table  int32 [batch, ld_table], table_cols columns in use: the page that
 *               holds tokens [c * page_size, (c + 1) * page_size) of a sequence
 *   kv_lens     int32 [batch]: tokens of each sequence in the cache, the call's
 *               own included; tokens past table_cols * page_size have no page
 *   cu          int32 [batch + 1]: the call's tokens of sequence s are rows
 *               [cu[s], cu[s + 1]), its LAST cu[s + 1] - cu[s] tokens
 * They are read on the device, so a captured graph follows their contents.  A
 * page id outside [0, pages) means "no page": its tokens are not written, not
 * attended to and read as zeros.  Distinct sequences written by one call must
 * not share a page that the call writes. */
typedef struct w4a8_kv_cache {
    void* k;
    void* v;
    void* k_scale;
    void* v_scale;
    int64_t pages;
    int32_t kv_heads, page_size, head_dim, reserved;
} w4a8_kv_cache;

/* Writes k, v (bf16 [tokens, ld], kv_heads * head_dim used) of the call's tokens.
 * A page's scale is max(its scale if it holds earlier tokens, max|new| / 127);
 * where it grows, earlier codes become rint(code * (old / new)); new codes are
 * rint(x / scale).  With cos_sin (f32 [table_rows, rot]: rot / 2 cosines, then
 * rot / 2 sines for each position; rot a multiple of 16, at most head_dim) the
 * first rot elements of every k head, and of every q head into q_out, are turned
 * by the token's position (the first and second half of them pairwise, or
 * neighbours with interleaved != 0); positions past the table use its last row.
 * q (bf16 [tokens, ldq], q_heads * head_dim used) may be NULL, q_out may be q.
 * Rows 16-byte aligned, leading dimensions multiples of 8. */
W4A8_API int w4a8_kv_write(const w4a8_kv_cache* cache, const int32_t* page_table, int64_t ld_table,
                           int64_t table_cols, const int32_t* kv_lens, const int32_t* cu_q, int64_t batch,
                           int64_t tokens, const void* k, int64_t ldk, const void* v, int64_t ldv, const void* q,
                           int64_t ldq, int32_t q_heads, void* q_out, int64_t ldqo, const float* cos_sin,
                           int64_t table_rows, int32_t rot, int32_t interleaved, void* stream);
/* The same with rotary positions that are not the tokens' places in their sequences, on up to
 * four axes (time, height, width of images and videos): pair i of a head turns by row
 * positions[a, t] of cos_sin, a = axis_of_pair[i].  positions int32 [axes, ld_positions] on the
 * device, read by the kernel (rows outside the table: its first or last one); axis_of_pair
 * [rot / 2] in HOST memory, read during the call, NULL for one axis.  cos_sin must be given. */
W4A8_API int w4a8_kv_write_axes(const w4a8_kv_cache* cache, const int32_t* page_table, int64_t ld_table,
                                int64_t table_cols, const int32_t* kv_lens, const int32_t* cu_q, int64_t batch,
                                int64_t tokens, const void* k, int64_t ldk, const void* v, int64_t ldv, const void* q,
                                int64_t ldq, int32_t q_heads, void* q_out, int64_t ldqo, const float* cos_sin,
                                int64_t table_rows, int32_t rot, int32_t interleaved, const int32_t* positions,
                                int64_t ld_positions, int32_t axes, const uint8_t* axis_of_pair, void* stream);
/* The rotation alone, without a cache: q and k (which may be NULL) bf16 [tokens, ld] of heads * head_dim into
 * q_out and k_out, each of which may be its input.  head_dim a multiple of 8, at most
 * W4A8_ROTARY_MAX_DIM; elements past rot are copied.  Rows 16-byte aligned, leading dimensions multiples of 8. */
#define W4A8_ROTARY_MAX_DIM 256
W4A8_API int w4a8_rotary(const void* q, int64_t ldq, int32_t q_heads, void* q_out, int64_t ldqo, const void* k, int64_t ldk,
                         int32_t k_heads, void* k_out, int64_t ldko, int64_t tokens, int32_t head_dim,
                         const float* cos_sin, int64_t table_rows, int32_t rot, int32_t interleaved,
                         const int32_t* positions, int64_t ld_positions, int32_t axes, const uint8_t* axis_of_pair,
                         void* stream);
/* Reads each sequence's last cu_out[s + 1] - cu_out[s] tokens back:
 * k, v bf16 [tokens, kv_heads, head_dim] dense. */
W4A8_API int w4a8_kv_read(const w4a8_kv_cache* cache, const int32_t* page_table, int64_t ld_table,
                          int64_t table_cols, const int32_t* kv_lens, const int32_t* cu_out, int64_t batch,
                          int64_t tokens, void* k, void* v, void* stream);

/* ---- pages kept on the device ----
 * Which pages a sequence holds and how long it is, as tensors that the calls below read and change on the
 * device, so that a captured step plans itself.  No counterpart in the reference.
 *   free_pages  int32 [pages]: a stack of page ids, its top at free_count[0] - 1
 *   table       int32 [sequences, columns]: the ceil(len / page_size) pages of each sequence in order
 *   lens        int32 [sequences]: tokens of each
 *   control     int32 [4], zeroed once: the status word, a counter that is 0 between calls, two of no use
 * sequences <= W4A8_PLAN_MAX_SEQUENCES, pages * page_size and columns * page_size < 2^31.  Calls on one state run
 * in stream order.
 *
 * A call that cannot be done as a whole changes nothing but the status word (its first non-zero
 * value stays until the caller clears it): W4A8_PLAN_ROW a row outside the state or twice in the call, _COUNT a
 * negative count, or more kept than held, _TOKENS more tokens than `tokens`, _PAGES too few free pages,
 * _COLUMNS a sequence past its columns, _STATE a state that contradicts itself. */
#define W4A8_PLAN_MAX_BATCH 2048
#define W4A8_PLAN_MAX_SEQUENCES 65536
#define W4A8_PLAN_ROW 1
#define W4A8_PLAN_COUNT 2
#define W4A8_PLAN_TOKENS 4
#define W4A8_PLAN_PAGES 8
#define W4A8_PLAN_COLUMNS 16
#define W4A8_PLAN_STATE 32
typedef struct w4a8_page_state {
    int32_t* free_pages;
    int32_t* free_count;
    int32_t* table;
    int32_t* lens;
    int32_t* control;
    int64_t pages, columns;
    int32_t sequences, page_size;
} w4a8_page_state;

/* Lengthens sequence rows[i] by counts[i] >= 0 tokens for i = 0 .. batch - 1, taking pages off the stack in this
 * order, and writes what the cache and attention calls take:
 *   page_table  int32 [batch, columns], -1 past a sequence's pages;  kv_lens [batch];  cu [batch + 1]
 *   slots       int32 [tokens] or NULL: page * page_size + place in the page, of each token of the step;
 *               -1 past the last one
 *   positions   int32 [axes, tokens] or NULL: rotary positions, 0 past the last token.  Without images the
 *               token's place in its sequence, on every axis.  With n_segs > 0 (axes = 3):
 *               segs int32 [n_segs, 4] holds (start, t, h, w) of grids whose first token is number `start` of its
 *               sequence, grids seg_cu[i] .. seg_cu[i + 1] (int32 [batch + 1]) being rows[i]'s in order; token r of a
 *               grid at text position o has positions o + r / (h w), o + r / w % h, o + r % w, and the
 *               text behind it goes on at o + max(t, h, w).  A grid with a side below 1 holds no tokens.
 * A refused step has page_table and slots -1, kv_lens, cu and positions 0. */
W4A8_API int w4a8_pages_plan(const w4a8_page_state* state, const int32_t* rows, const int32_t* counts, int64_t batch,
                             int64_t tokens, int32_t axes, const int32_t* seg_cu, const int32_t* segs, int64_t n_segs,
                             int32_t* page_table, int32_t* kv_lens, int32_t* cu, int32_t* slots, int32_t* positions,
                             void* stream);
/* Shortens sequence rows[i] to keep[i] tokens (NULL: 0) and gives its pages past them back, from the last page of the
 * last sequence to the first: the inverse of a plan over the same rows.  For sequences that ended and drafted
 * tokens that were not accepted. */
W4A8_API int w4a8_pages_shrink(const w4a8_page_state* state, const int32_t* rows, const int32_t* keep, int64_t batch,
                               void* stream);

/* ---- causal attention over the cache ----
 * out[t, h] = sum_j softmax_j(softmax_scale * q[t, h] . k_j) v_j over the cached
 * tokens j at or before query token t's position, k and v of kv head
 * h / (q_heads / kv_heads); a row that sees no token is zero.  q, out bf16
 * [tokens, ld] (q_heads * head_dim used; rows 16-byte aligned, ld a multiple of
 * 8); rows of q that cu gives to no sequence are left unwritten in out.
 * softmax_scale >= 0.  max_q_len is the longest cu[s + 1] - cu[s]: it chooses the
 * kernel and the workspace's size, and a call whose sequences are longer is slower,
 * not wrong.  batch <= W4A8_ATTENTION_MAX_BATCH, tokens * (q_heads / kv_heads) <=
 * 0x7FFF0000, cache->pages > 0.  Workspace as for the linear calls
 * (w4a8_attention_workspace_size bytes, 1024-byte aligned, zeroed before first use,
 * may be shared with them in stream order). */
#define W4A8_ATTENTION_MAX_BATCH 2048
W4A8_API size_t w4a8_attention_workspace_size(int64_t batch, int64_t tokens, int32_t q_heads, int32_t kv_heads,
                                              int32_t head_dim, int32_t max_q_len);
W4A8_API int w4a8_attention(const w4a8_kv_cache* cache, const int32_t* page_table, int64_t ld_table,
                            int64_t table_cols, const int32_t* kv_lens, const int32_t* cu_q, int64_t batch,
                            int64_t tokens, const void* q, int64_t ldq, int32_t q_heads, int32_t max_q_len,
                            float softmax_scale, void* out, int64_t ldo, void* workspace, size_t workspace_bytes,
                            void* stream);

/* ---- status ---- */
/* Synchronises `stream` and returns the device status word of `workspace`
 * (0 = no kernel reported a failure; otherwise 0x100 + the id of the wait
 * that ran out).  reset != 0 clears it. */
W4A8_API int w4a8_workspace_status(void* workspace, int32_t reset, void* stream);
W4A8_API const char* w4a8_status_string(int status);
W4A8_API int w4a8_last_cuda_error(void);
/* Library build: returns the sm architecture it was compiled for (100). */
W4A8_API int w4a8_build_arch(void);

/* ---- options (process-wide; no counterpart in the reference) ----
 * W4A8_OPT_FUSED_QUANT: a linear call with M <= 16, group size <= 256 and
 * 16-byte aligned activation rows quantises its activation inside the GEMM
 * (four quantiser warps per CTA, the bf16 rows brought in by 2-D tensor
 * copies) instead of running the standalone quantiser kernel first.  Same
 * bits.  Off by default: every CTA quantises the activation slice of each
 * weight tile it visits, and measured on B200 the fused call is slower at
 * every decode size (e.g. gate_up M = 16: 183 us against 34 us per call).
 * W4A8_OPT_AR_PUSH: w4a8_linear_prepared_allreduce stores every output tile
 * into every rank's receive slot (posted peer stores from the GEMM epilogue)
 * instead of its own slot only, the peers then reading it (the default).
 * Returns the previous flags. */
#define W4A8_OPT_FUSED_QUANT 1
#define W4A8_OPT_AR_PUSH 2
W4A8_API int w4a8_set_options(int32_t flags);

#ifdef __cplusplus
}
#endif

#endif /* W4A8_B200_H */
