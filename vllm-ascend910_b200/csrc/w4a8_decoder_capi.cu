// w4a8_decoder_capi.cu -- C entry points of the operators around the linears:
// norm, quantised cache, attention (declared in include/w4a8_b200.h).  Argument
// checks and parameter blocks; the linear calls with a norm in front are in
// w4a8_capi.cu beside the other linear calls.
#include "w4a8_b200.h"
#include "w4a8_kernels.h"

using namespace w4a8;

namespace {

constexpr size_t kStatusBytes = 1024;      // status word block at the start of a workspace
constexpr int kCallsWord = 8;              // the count of started CTAs within it
constexpr int kTicketWord = 16;            // first ticket word within it (a byte counts up to 255 parts)
constexpr int64_t kMaxTokens = int64_t(1) << 30;

bool aligned(const void* ptr, uintptr_t a) { return (reinterpret_cast<uintptr_t>(ptr) & (a - 1)) == 0; }

// The cache and batch arguments that every entry point takes.
int make_view(const w4a8_kv_cache* c, const int32_t* table, int64_t ld_table, int64_t table_cols,
              const int32_t* kv_lens, const int32_t* cu, int64_t batch, int64_t tokens, CacheView* out)
{
    if (!c || batch < 0 || tokens < 0) return W4A8_ERR_INVALID;
    if (c->head_dim != 64 && c->head_dim != 128) return W4A8_ERR_UNSUPPORTED;
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return W4A8_ERR_UNSUPPORTED;
    if (c->kv_heads <= 0 || c->kv_heads > 4096 || c->pages <= 0 || c->pages > 0x7FFFFFFF) return W4A8_ERR_INVALID;
    if (tokens > kMaxTokens || batch > kMaxTokens || table_cols < 0 || ld_table < table_cols) return W4A8_ERR_INVALID;
    if (table_cols > 0x7FFFFFFF / c->page_size) return W4A8_ERR_INVALID;
    if (batch == 0 || tokens == 0) {
        *out = CacheView{};
        return W4A8_OK;
    }
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !table || !kv_lens || !cu) return W4A8_ERR_INVALID;
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4)) return W4A8_ERR_INVALID;
    if (!aligned(table, 4) || !aligned(kv_lens, 4) || !aligned(cu, 4)) return W4A8_ERR_INVALID;
    CacheView v{};
    v.k = static_cast<int8_t*>(c->k);
    v.v = static_cast<int8_t*>(c->v);
    v.k_scale = static_cast<float*>(c->k_scale);
    v.v_scale = static_cast<float*>(c->v_scale);
    v.table = table;
    v.kv_lens = kv_lens;
    v.cu = cu;
    v.ld_table = ld_table;
    v.pages = c->pages;
    v.tokens = tokens;
    v.table_cols = static_cast<int>(table_cols);
    v.batch = static_cast<int>(batch);
    v.kv_heads = c->kv_heads;
    v.page = c->page_size;
    v.page_log2 = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
    v.D = c->head_dim;
    *out = v;
    return W4A8_OK;
}

bool rows_ok(const void* p, int64_t ld, int64_t width) { return p && aligned(p, 16) && ld % 8 == 0 && ld >= width; }

}  // namespace

extern "C" {

int w4a8_kv_write(const w4a8_kv_cache* cache, const int32_t* page_table, int64_t ld_table, int64_t table_cols,
                  const int32_t* kv_lens, const int32_t* cu_q, int64_t batch, int64_t tokens, const void* k,
                  int64_t ldk, const void* v, int64_t ldv, const void* q, int64_t ldq, int32_t q_heads, void* q_out,
                  int64_t ldqo, const float* cos_sin, int64_t table_rows, int32_t rot, int32_t interleaved,
                  void* stream)
{
    KvWriteParams p{};
    int rc = make_view(cache, page_table, ld_table, table_cols, kv_lens, cu_q, batch, tokens, &p.c);
    if (rc != W4A8_OK) return rc;
    if (cos_sin && (rot <= 0 || rot > cache->head_dim || rot % 16 != 0)) return W4A8_ERR_UNSUPPORTED;
    if (cos_sin && (table_rows <= 0 || !aligned(cos_sin, 16))) return W4A8_ERR_INVALID;
    if (q && (q_heads <= 0 || q_heads > 65536)) return W4A8_ERR_INVALID;
    if (p.c.batch == 0) return W4A8_OK;
    const int64_t kvw = static_cast<int64_t>(cache->kv_heads) * cache->head_dim;
    if (!rows_ok(k, ldk, kvw) || !rows_ok(v, ldv, kvw)) return W4A8_ERR_INVALID;
    if (q) {
        const int64_t qw = static_cast<int64_t>(q_heads) * cache->head_dim;
        if (!rows_ok(q, ldq, qw) || !rows_ok(q_out, ldqo, qw)) return W4A8_ERR_INVALID;
    }
    int sms = 0;
    if ((rc = capi_device_sms(&sms)) != W4A8_OK) return rc;
    p.q = static_cast<const uint16_t*>(q);
    p.k = static_cast<const uint16_t*>(k);
    p.v = static_cast<const uint16_t*>(v);
    p.q_out = static_cast<uint16_t*>(q_out);
    p.cos_sin = cos_sin;
    p.ldq = ldq;
    p.ldk = ldk;
    p.ldv = ldv;
    p.ldqo = ldqo;
    p.table_rows = cos_sin ? table_rows : 1;
    p.q_heads = q_heads;
    p.rot = cos_sin ? rot : 0;
    p.interleaved = interleaved != 0;
    const cudaError_t e = launch_kv_write(p, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? W4A8_OK : capi_fail_cuda(e);
}

int w4a8_kv_read(const w4a8_kv_cache* cache, const int32_t* page_table, int64_t ld_table, int64_t table_cols,
                 const int32_t* kv_lens, const int32_t* cu_out, int64_t batch, int64_t tokens, void* k, void* v,
                 void* stream)
{
    KvReadParams p{};
    int rc = make_view(cache, page_table, ld_table, table_cols, kv_lens, cu_out, batch, tokens, &p.c);
    if (rc != W4A8_OK) return rc;
    if (p.c.batch == 0) return W4A8_OK;
    if (!k || !v || !aligned(k, 16) || !aligned(v, 16)) return W4A8_ERR_INVALID;
    int sms = 0;
    if ((rc = capi_device_sms(&sms)) != W4A8_OK) return rc;
    p.k = static_cast<uint16_t*>(k);
    p.v = static_cast<uint16_t*>(v);
    const cudaError_t e = launch_kv_read(p, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? W4A8_OK : capi_fail_cuda(e);
}

size_t w4a8_attention_workspace_size(int64_t batch, int64_t tokens, int32_t q_heads, int32_t kv_heads,
                                     int32_t head_dim, int32_t max_q_len)
{
    if (batch < 0 || tokens < 0 || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads != 0 || max_q_len < 0) return 0;
    if (head_dim != 64 && head_dim != 128) return 0;
    int sms = 0;
    if (capi_device_sms(&sms) != W4A8_OK) sms = 148;
    return kStatusBytes + attention_ws_bytes(static_cast<int>(batch), tokens, q_heads, kv_heads, head_dim, max_q_len, sms);
}

int w4a8_attention(const w4a8_kv_cache* cache, const int32_t* page_table, int64_t ld_table, int64_t table_cols,
                   const int32_t* kv_lens, const int32_t* cu_q, int64_t batch, int64_t tokens, const void* q,
                   int64_t ldq, int32_t q_heads, int32_t max_q_len, float softmax_scale, void* out, int64_t ldo,
                   void* workspace, size_t workspace_bytes, void* stream)
{
    AttentionParams p{};
    int rc = make_view(cache, page_table, ld_table, table_cols, kv_lens, cu_q, batch, tokens, &p.c);
    if (rc != W4A8_OK) return rc;
    if (q_heads <= 0 || q_heads > 65536 || q_heads % cache->kv_heads != 0) return W4A8_ERR_INVALID;
    if (max_q_len < 0 || !(softmax_scale >= 0.0f)) return W4A8_ERR_INVALID;
    if (batch > W4A8_ATTENTION_MAX_BATCH) return W4A8_ERR_UNSUPPORTED;
    if (tokens * (q_heads / cache->kv_heads) > 0x7FFF0000) return W4A8_ERR_UNSUPPORTED;   // packed rows are 32-bit
    if (p.c.batch == 0) return W4A8_OK;
    if (max_q_len == 0) return W4A8_ERR_INVALID;
    const int64_t qw = static_cast<int64_t>(q_heads) * cache->head_dim;
    if (!rows_ok(q, ldq, qw) || !rows_ok(out, ldo, qw)) return W4A8_ERR_INVALID;
    int sms = 0;
    if ((rc = capi_device_sms(&sms)) != W4A8_OK) return rc;
    const size_t need =
        kStatusBytes + attention_ws_bytes(p.c.batch, tokens, q_heads, cache->kv_heads, cache->head_dim, max_q_len, sms);
    if (!workspace || !aligned(workspace, 1024) || workspace_bytes < need) return W4A8_ERR_WORKSPACE;
    p.q = static_cast<const uint16_t*>(q);
    p.out = static_cast<uint16_t*>(out);
    p.ldq = ldq;
    p.ldo = ldo;
    p.q_heads = q_heads;
    p.group = q_heads / cache->kv_heads;
    p.group_magic = p.group == 1 ? 0 : ~static_cast<uint64_t>(0) / static_cast<uint64_t>(p.group) + 1;
    p.max_q = max_q_len;
    p.scale_log2 = softmax_scale * 1.4426950408889634f;
    p.status = static_cast<int*>(workspace);
    p.calls = static_cast<uint32_t*>(workspace) + kCallsWord;
    p.tickets = static_cast<uint32_t*>(workspace) + kTicketWord;
    if (sms > static_cast<int>(kStatusBytes / 4) - kTicketWord) return W4A8_ERR_DEVICE;
    p.ws = static_cast<uint8_t*>(workspace) + kStatusBytes;
    const cudaError_t e = launch_attention(p, sms, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? W4A8_OK : capi_fail_cuda(e);
}

}  // extern "C"
