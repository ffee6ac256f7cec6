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

// Positions of their own: int32 [axes, ld], and the axis of each of `pairs` pairs (host memory, read here).
int make_axes(const int32_t* positions, int64_t ld, int32_t axes, const uint8_t* axis_of_pair, int pairs, int64_t tokens,
              AxesView* out)
{
    if (!positions || !aligned(positions, 4) || axes < 1 || axes > kMaxAxes || pairs > 128) return W4A8_ERR_INVALID;
    if (axes > 1 && (!axis_of_pair || ld < tokens)) return W4A8_ERR_INVALID;
    AxesView v{};
    v.positions = positions;
    v.ld = ld;
    v.axes = axes;
    for (int i = 0; axis_of_pair && i < pairs; ++i) {
        if (axis_of_pair[i] >= axes) return W4A8_ERR_INVALID;
        v.map[i / 32] |= static_cast<uint64_t>(axis_of_pair[i]) << (2 * (i % 32));
    }
    *out = v;
    return W4A8_OK;
}

int make_pages(const w4a8_page_state* c, const int32_t* rows, int64_t batch, PagesParams* out)
{
    if (!c || batch < 0) return W4A8_ERR_INVALID;
    if (batch > W4A8_PLAN_MAX_BATCH || c->sequences > W4A8_PLAN_MAX_SEQUENCES) return W4A8_ERR_UNSUPPORTED;
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return W4A8_ERR_UNSUPPORTED;
    if (c->pages <= 0 || c->pages > 0x7FFFFFFF / c->page_size || c->sequences <= 0) return W4A8_ERR_INVALID;
    if (c->columns <= 0 || c->columns > 0x7FFFFFFF / c->page_size) return W4A8_ERR_INVALID;
    if (!c->free_pages || !c->free_count || !c->table || !c->lens || !c->control || (!rows && batch > 0)) return W4A8_ERR_INVALID;
    if (!aligned(c->free_pages, 4) || !aligned(c->free_count, 4) || !aligned(c->table, 4) || !aligned(c->lens, 4) ||
        !aligned(c->control, 4) || !aligned(rows, 4))
        return W4A8_ERR_INVALID;
    PagesParams p{};
    p.free = c->free_pages;
    p.free_count = c->free_count;
    p.table = c->table;
    p.lens = c->lens;
    p.status = c->control;
    p.ticket = reinterpret_cast<uint32_t*>(c->control) + 1;
    p.pages = static_cast<int>(c->pages);
    p.sequences = c->sequences;
    p.columns = static_cast<int>(c->columns);
    p.page_log2 = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
    p.rows = rows;
    p.batch = static_cast<int>(batch);
    *out = p;
    return W4A8_OK;
}

bool rows_ok(const void* p, int64_t ld, int64_t width) { return p && aligned(p, 16) && ld % 8 == 0 && ld >= width; }

int kv_write_impl(const w4a8_kv_cache* cache, const int32_t* page_table, int64_t ld_table, int64_t table_cols,
                  const int32_t* kv_lens, const int32_t* cu_q, int64_t batch, int64_t tokens, const void* k,
                  int64_t ldk, const void* v, int64_t ldv, const void* q, int64_t ldq, int32_t q_heads, void* q_out,
                  int64_t ldqo, const float* cos_sin, int64_t table_rows, int32_t rot, int32_t interleaved,
                  const int32_t* positions, int64_t ld_positions, int32_t axes, const uint8_t* axis_of_pair, bool own,
                  void* stream)
{
    KvWriteParams p{};
    int rc = make_view(cache, page_table, ld_table, table_cols, kv_lens, cu_q, batch, tokens, &p.c);
    if (rc != W4A8_OK) return rc;
    if (cos_sin && (rot <= 0 || rot > cache->head_dim || rot % 16 != 0)) return W4A8_ERR_UNSUPPORTED;
    if (cos_sin && (table_rows <= 0 || !aligned(cos_sin, 16))) return W4A8_ERR_INVALID;
    if (q && (q_heads <= 0 || q_heads > 65536)) return W4A8_ERR_INVALID;
    if (own && !cos_sin) return W4A8_ERR_INVALID;
    if (p.c.batch == 0) return W4A8_OK;
    if (own && (rc = make_axes(positions, ld_positions, axes, axis_of_pair, rot / 2, tokens, &p.axes)) != W4A8_OK) return rc;
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

}  // namespace

extern "C" {

int w4a8_kv_write(const w4a8_kv_cache* cache, const int32_t* page_table, int64_t ld_table, int64_t table_cols,
                  const int32_t* kv_lens, const int32_t* cu_q, int64_t batch, int64_t tokens, const void* k,
                  int64_t ldk, const void* v, int64_t ldv, const void* q, int64_t ldq, int32_t q_heads, void* q_out,
                  int64_t ldqo, const float* cos_sin, int64_t table_rows, int32_t rot, int32_t interleaved,
                  void* stream)
{
    return kv_write_impl(cache, page_table, ld_table, table_cols, kv_lens, cu_q, batch, tokens, k, ldk, v, ldv, q, ldq, q_heads,
                         q_out, ldqo, cos_sin, table_rows, rot, interleaved, nullptr, 0, 0, nullptr, false, stream);
}

int w4a8_kv_write_axes(const w4a8_kv_cache* cache, const int32_t* page_table, int64_t ld_table, int64_t table_cols,
                       const int32_t* kv_lens, const int32_t* cu_q, int64_t batch, int64_t tokens, const void* k,
                       int64_t ldk, const void* v, int64_t ldv, const void* q, int64_t ldq, int32_t q_heads, void* q_out,
                       int64_t ldqo, const float* cos_sin, int64_t table_rows, int32_t rot, int32_t interleaved,
                       const int32_t* positions, int64_t ld_positions, int32_t axes, const uint8_t* axis_of_pair,
                       void* stream)
{
    return kv_write_impl(cache, page_table, ld_table, table_cols, kv_lens, cu_q, batch, tokens, k, ldk, v, ldv, q, ldq, q_heads,
                         q_out, ldqo, cos_sin, table_rows, rot, interleaved, positions, ld_positions, axes, axis_of_pair, true,
                         stream);
}

int w4a8_rotary(const void* q, int64_t ldq, int32_t q_heads, void* q_out, int64_t ldqo, const void* k, int64_t ldk,
                int32_t k_heads, void* k_out, int64_t ldko, int64_t tokens, int32_t head_dim, const float* cos_sin,
                int64_t table_rows, int32_t rot, int32_t interleaved, const int32_t* positions, int64_t ld_positions,
                int32_t axes, const uint8_t* axis_of_pair, void* stream)
{
    if (tokens < 0 || tokens > kMaxTokens) return W4A8_ERR_INVALID;
    if (head_dim <= 0 || head_dim > W4A8_ROTARY_MAX_DIM || head_dim % 8 != 0) return W4A8_ERR_UNSUPPORTED;
    if (rot <= 0 || rot > head_dim || rot % 16 != 0) return W4A8_ERR_UNSUPPORTED;
    if (tokens == 0) return W4A8_OK;
    if (!cos_sin || !aligned(cos_sin, 16) || table_rows <= 0) return W4A8_ERR_INVALID;
    RotaryParams p{};
    const void* x[2] = {q, k};
    void* out[2] = {q_out, k_out};
    const int64_t ld[2] = {ldq, ldk}, ldo[2] = {ldqo, ldko};
    const int32_t heads[2] = {q_heads, k_heads};
    for (int i = 0; i < 2; ++i) {
        if (i == 1 && !k) break;
        if (heads[i] <= 0 || heads[i] > 65536) return W4A8_ERR_INVALID;
        const int64_t wide = static_cast<int64_t>(heads[i]) * head_dim;
        if (!rows_ok(x[i], ld[i], wide) || !rows_ok(out[i], ldo[i], wide)) return W4A8_ERR_INVALID;
        p.x[i] = static_cast<const uint16_t*>(x[i]);
        p.out[i] = static_cast<uint16_t*>(out[i]);
        p.ld[i] = ld[i];
        p.ldo[i] = ldo[i];
        p.heads[i] = heads[i];
    }
    int rc = make_axes(positions, ld_positions, axes, axis_of_pair, rot / 2, tokens, &p.axes);
    if (rc != W4A8_OK) return rc;
    int sms = 0;
    if ((rc = capi_device_sms(&sms)) != W4A8_OK) return rc;
    p.cos_sin = cos_sin;
    p.tokens = tokens;
    p.table_rows = table_rows;
    p.D = head_dim;
    p.rot = rot;
    p.interleaved = interleaved != 0;
    const cudaError_t e = launch_rotary(p, static_cast<cudaStream_t>(stream));
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

int w4a8_pages_plan(const w4a8_page_state* state, const int32_t* rows, const int32_t* counts, int64_t batch, int64_t tokens,
                    int32_t axes, const int32_t* seg_cu, const int32_t* segs, int64_t n_segs, int32_t* page_table,
                    int32_t* kv_lens, int32_t* cu, int32_t* slots, int32_t* positions, void* stream)
{
    PagesParams p{};
    int rc = make_pages(state, rows, batch, &p);
    if (rc != W4A8_OK) return rc;
    if (tokens < 0 || tokens > kMaxTokens || axes < 1 || axes > kMaxAxes) return W4A8_ERR_INVALID;
    if (!cu || !aligned(cu, 4)) return W4A8_ERR_INVALID;
    if (batch > 0 && (!counts || !aligned(counts, 4) || !page_table || !aligned(page_table, 4) || !kv_lens || !aligned(kv_lens, 4)))
        return W4A8_ERR_INVALID;
    if (!aligned(slots, 4) || !aligned(positions, 4) || n_segs < 0 || n_segs > 0x7FFFFFFF) return W4A8_ERR_INVALID;
    if (n_segs > 0 && (axes != 3 || !seg_cu || !segs || !aligned(seg_cu, 4) || !aligned(segs, 16))) return W4A8_ERR_INVALID;
    int sms = 0;
    if ((rc = capi_device_sms(&sms)) != W4A8_OK) return rc;
    p.counts = counts;
    p.tokens = tokens;
    p.axes = axes;
    p.n_segs = static_cast<int>(n_segs);
    p.seg_cu = n_segs > 0 ? seg_cu : nullptr;
    p.segs = n_segs > 0 ? segs : nullptr;
    p.page_table = page_table;
    p.kv_lens = kv_lens;
    p.cu = cu;
    p.slots = slots;
    p.positions = positions;
    const cudaError_t e = launch_pages_plan(p, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? W4A8_OK : capi_fail_cuda(e);
}

int w4a8_pages_shrink(const w4a8_page_state* state, const int32_t* rows, const int32_t* keep, int64_t batch, void* stream)
{
    PagesParams p{};
    int rc = make_pages(state, rows, batch, &p);
    if (rc != W4A8_OK) return rc;
    if (!aligned(keep, 4)) return W4A8_ERR_INVALID;
    if (batch == 0) return W4A8_OK;
    int sms = 0;
    if ((rc = capi_device_sms(&sms)) != W4A8_OK) return rc;
    p.counts = keep;
    const cudaError_t e = launch_pages_shrink(p, static_cast<cudaStream_t>(stream));
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
