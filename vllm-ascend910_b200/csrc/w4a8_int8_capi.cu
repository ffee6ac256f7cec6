// w4a8_int8_capi.cu -- C entry points of the linears in 8-bit integers (declared in
// include/w4a8_b200.h): argument checks, the workspace's parts, tensor maps, launches.
#include <algorithm>

#include "w4a8_b200.h"
#include "w4a8_kernels.h"

using namespace w4a8;

namespace {

constexpr int64_t kMaxRows = int64_t(1) << 24;

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// Status block, scales [M], codes [M, row] of a call.
struct Parts {
    size_t scale, codes, total;
    int64_t row;
};

Parts parts(int64_t M, int64_t K)
{
    Parts p{};
    p.row = round_up(K, 16);
    p.scale = 1024;
    p.codes = p.scale + static_cast<size_t>(round_up(M * 4, 1024));
    p.total = static_cast<size_t>(round_up(static_cast<int64_t>(p.codes) + M * p.row, 1024));
    return p;
}

int check_sizes(int64_t M, int64_t N, int64_t K)
{
    if (M < 0 || N <= 0 || K <= 0) return W4A8_ERR_INVALID;
    if (K > W4A8_INT8_MAX_K || M > kMaxRows || N > kMaxRows) return W4A8_ERR_UNSUPPORTED;
    return W4A8_OK;
}

int check_layer(const int8_t* w, int64_t ldw, const float* w_scale, const float* bias, int64_t K, const void* y, int64_t ldy,
                int64_t N)
{
    if (!w || !aligned(w, 16) || ldw < K || ldw % 16 != 0 || !w_scale || !aligned(w_scale, 4) || !aligned(bias, 4))
        return W4A8_ERR_INVALID;
    if (!y || ldy < N || !aligned(y, 2)) return W4A8_ERR_INVALID;
    return W4A8_OK;
}

// Rows of x for the quantiser; `q`, `scale`: where its outputs go.
int make_source(const void* x, int64_t M, int64_t K, int64_t ldx, int32_t act, TokenQuantParams* out)
{
    if (act != W4A8_ACT_NONE && act != W4A8_ACT_SWIGLU) return W4A8_ERR_UNSUPPORTED;
    const int64_t wide = act == W4A8_ACT_SWIGLU ? 2 * K : K;
    if (!x || ldx < wide || !aligned(x, 2)) return W4A8_ERR_INVALID;
    TokenQuantParams p{};
    p.x = static_cast<const uint16_t*>(x);
    p.ldx = ldx;
    p.M = static_cast<int>(M);
    p.K = static_cast<int>(K);
    p.vec_x = aligned(x, 16) && ldx % 8 == 0;
    *out = p;
    return W4A8_OK;
}

void put_codes(TokenQuantParams* p, int8_t* q, int64_t ldq, float* scale)
{
    p->q = q;
    p->ldq = ldq;
    p->scale = scale;
    p->vec_q = aligned(q, 8) && ldq % 8 == 0;
}

int run_gemm(const int8_t* q, int64_t ldq, const float* scale, int64_t M, int64_t K, const int8_t* w, int64_t ldw,
             const float* w_scale, const float* bias, int64_t N, void* y, int64_t ldy, void* workspace, int sms, cudaStream_t st,
             bool pdl)
{
    Int8GemmParams g{};
    const Int8Plan plan = int8_plan(M, N, K, sms);
    int rc = capi_bytes_map(&g.tm_w, w, K, N, ldw, plan.w_rows);
    if (rc == W4A8_OK) rc = capi_bytes_map(&g.tm_a, q, K, M, ldq, plan.a_rows);
    if (rc != W4A8_OK) return rc;
    g.a_scale = scale;
    g.w_scale = w_scale;
    g.bias = bias;
    g.y = static_cast<uint16_t*>(y);
    g.ldy = ldy;
    g.status = static_cast<int*>(workspace);
    g.M = static_cast<int>(M);
    g.N = static_cast<int>(N);
    g.K = static_cast<int>(K);
    const cudaError_t e = launch_int8_gemm(g, plan, sms, st, pdl);
    return e == cudaSuccess ? W4A8_OK : capi_fail_cuda(e);
}

// The quantiser into the workspace, then the product.
int run_linear(TokenQuantParams& t, int source, const int8_t* w, int64_t ldw, const float* w_scale, const float* bias, int64_t N,
               void* y, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream)
{
    int sms = 0, rc = capi_device_sms(&sms);
    if (rc != W4A8_OK) return rc;
    const Parts p = parts(t.M, t.K);
    if (!workspace || !aligned(workspace, 1024) || workspace_bytes < p.total) return W4A8_ERR_WORKSPACE;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    put_codes(&t, reinterpret_cast<int8_t*>(ws + p.codes), p.row, reinterpret_cast<float*>(ws + p.scale));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = launch_token_quant(t, source, st);
    if (e != cudaSuccess) return capi_fail_cuda(e);
    return run_gemm(t.q, p.row, t.scale, t.M, t.K, w, ldw, w_scale, bias, N, y, ldy, workspace, sms, st, true);
}

}  // namespace

extern "C" {

size_t w4a8_int8_workspace_size(int64_t M, int64_t K)
{
    if (M < 0 || K <= 0 || K > W4A8_INT8_MAX_K || M > kMaxRows) return 0;
    return parts(M, K).total;
}

int w4a8_int8_quant(const void* x, int64_t M, int64_t K, int64_t ldx, int32_t act, int8_t* q, int64_t ldq, float* scale,
                    void* stream)
{
    int rc = check_sizes(M, 1, K);
    if (rc != W4A8_OK || M == 0) return rc;
    TokenQuantParams t{};
    if ((rc = make_source(x, M, K, ldx, act, &t)) != W4A8_OK) return rc;
    if (!q || ldq < K || !scale || !aligned(scale, 4)) return W4A8_ERR_INVALID;
    int sms = 0;
    if ((rc = capi_device_sms(&sms)) != W4A8_OK) return rc;
    put_codes(&t, q, ldq, scale);
    const cudaError_t e = launch_token_quant(t, act == W4A8_ACT_SWIGLU ? kTokSwiglu : kTokPlain, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? W4A8_OK : capi_fail_cuda(e);
}

int w4a8_int8_gemm(const int8_t* q, int64_t ldq, const float* scale, int64_t M, int64_t K, const int8_t* w, int64_t ldw,
                   const float* w_scale, const float* bias, int64_t N, void* y, int64_t ldy, void* workspace,
                   size_t workspace_bytes, void* stream)
{
    int rc = check_sizes(M, N, K);
    if (rc != W4A8_OK || M == 0) return rc;
    if ((rc = check_layer(w, ldw, w_scale, bias, K, y, ldy, N)) != W4A8_OK) return rc;
    if (!q || !aligned(q, 16) || ldq < K || ldq % 16 != 0 || !scale || !aligned(scale, 4)) return W4A8_ERR_INVALID;
    int sms = 0;
    if ((rc = capi_device_sms(&sms)) != W4A8_OK) return rc;
    if (!workspace || !aligned(workspace, 1024) || workspace_bytes < 1024) return W4A8_ERR_WORKSPACE;
    return run_gemm(q, ldq, scale, M, K, w, ldw, w_scale, bias, N, y, ldy, workspace, sms, static_cast<cudaStream_t>(stream), false);
}

int w4a8_int8_linear(const void* x, int64_t M, int64_t K, int64_t ldx, int32_t act, const int8_t* w, int64_t ldw,
                     const float* w_scale, const float* bias, int64_t N, void* y, int64_t ldy, void* workspace,
                     size_t workspace_bytes, void* stream)
{
    int rc = check_sizes(M, N, K);
    if (rc != W4A8_OK || M == 0) return rc;
    TokenQuantParams t{};
    if ((rc = make_source(x, M, K, ldx, act, &t)) != W4A8_OK) return rc;
    if ((rc = check_layer(w, ldw, w_scale, bias, K, y, ldy, N)) != W4A8_OK) return rc;
    return run_linear(t, act == W4A8_ACT_SWIGLU ? kTokSwiglu : kTokPlain, w, ldw, w_scale, bias, N, y, ldy, workspace,
                      workspace_bytes, stream);
}

int w4a8_int8_linear_rms_norm(const void* x, int64_t M, int64_t K, int64_t ldx, const void* residual, int64_t ldr,
                              void* residual_out, int64_t ldro, const void* weight, int32_t weight_dtype, float eps,
                              const int8_t* w, int64_t ldw, const float* w_scale, const float* bias, int64_t N, void* y,
                              int64_t ldy, void* workspace, size_t workspace_bytes, void* stream)
{
    int rc = check_sizes(M, N, K);
    if (rc != W4A8_OK) return rc;
    if (K > W4A8_NORM_MAX_K) return W4A8_ERR_UNSUPPORTED;
    if (weight_dtype != W4A8_DTYPE_BF16 && weight_dtype != W4A8_DTYPE_F32) return W4A8_ERR_UNSUPPORTED;
    if (!(eps >= 0.0f)) return W4A8_ERR_INVALID;
    if (M == 0) return W4A8_OK;
    TokenQuantParams t{};
    if ((rc = make_source(x, M, K, ldx, W4A8_ACT_NONE, &t)) != W4A8_OK) return rc;
    if (!weight || !aligned(weight, weight_dtype == W4A8_DTYPE_F32 ? 4 : 2)) return W4A8_ERR_INVALID;
    if (residual && (ldr < K || !aligned(residual, 2))) return W4A8_ERR_INVALID;
    if (residual_out && (ldro < K || !aligned(residual_out, 2))) return W4A8_ERR_INVALID;
    if ((rc = check_layer(w, ldw, w_scale, bias, K, y, ldy, N)) != W4A8_OK) return rc;
    t.res = static_cast<const uint16_t*>(residual);
    t.res_out = static_cast<uint16_t*>(residual_out);
    t.ldr = ldr;
    t.ldro = ldro;
    t.vec_r = aligned(residual, 16) && ldr % 8 == 0;
    t.vec_ro = aligned(residual_out, 16) && ldro % 8 == 0;
    t.weight = weight;
    t.weight_f32 = weight_dtype == W4A8_DTYPE_F32;
    t.vec_w = aligned(weight, 16);
    t.eps = eps;
    return run_linear(t, kTokNorm, w, ldw, w_scale, bias, N, y, ldy, workspace, workspace_bytes, stream);
}

}  // extern "C"
