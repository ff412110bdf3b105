// extern "C" surface of the paged key-value cache and the decode attention (declared in include/fp8lin.h).
#include "common.cuh"
#include "kernels.h"

using namespace fp8lin;

namespace {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Strides (in elements) of a [.., n, ..] dimension: whole 16-byte words, where there is more than one element to step over.
inline bool bad_stride(int64_t stride, int64_t n, int64_t words) { return n > 1 && (stride <= 0 || stride % words != 0); }

int view_of(const fp8lin_kv_cache* c, CacheView* v) {
    if (!c) return set_error(FP8LIN_ERR_NULL, "cache must not be NULL");
    if (c->dtype != FP8LIN_CACHE_BF16 && c->dtype != FP8LIN_CACHE_E4M3) return set_error(FP8LIN_ERR_ARG, "cache dtype must be FP8LIN_CACHE_BF16 or FP8LIN_CACHE_E4M3");
    if (c->num_blocks <= 0 || c->block_size <= 0 || c->num_kv_heads <= 0 || c->num_blocks > (1ll << 31) || c->num_kv_heads > 65535)
        return set_error(FP8LIN_ERR_SHAPE, "bad cache shape num_blocks=%lld block_size=%d num_kv_heads=%d", (long long)c->num_blocks, c->block_size, c->num_kv_heads);
    if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16 != 0)
        return set_error(FP8LIN_ERR_SHAPE, "head_dim=%d must be a multiple of 16 from 16 to 256", c->head_dim);
    const bool e4m3 = c->dtype == FP8LIN_CACHE_E4M3;
    if (!c->k || !c->v) return set_error(FP8LIN_ERR_NULL, "the cache's k and v must not be NULL");
    if (e4m3 && (!c->k_scale || !c->v_scale)) return set_error(FP8LIN_ERR_NULL, "an e4m3 cache needs k_scale and v_scale");
    if (!aligned16(c->k) || !aligned16(c->v)) return set_error(FP8LIN_ERR_ALIGN, "the cache's k and v must be 16-byte aligned");
    const int64_t words = e4m3 ? 16 : 8, elem = e4m3 ? 1 : 2;
    if (bad_stride(c->stride_block, c->num_blocks, words) || bad_stride(c->stride_token, c->block_size, words) || bad_stride(c->stride_head, c->num_kv_heads, words))
        return set_error(FP8LIN_ERR_ALIGN, "the cache's strides must be positive multiples of 16 bytes");
    if (e4m3 && ((c->num_blocks > 1 && c->scale_stride_block <= 0) || (c->block_size > 1 && c->scale_stride_token <= 0) || (c->num_kv_heads > 1 && c->scale_stride_head <= 0)))
        return set_error(FP8LIN_ERR_SHAPE, "the scales' strides must be positive");
    auto step = [](int64_t stride, int64_t n) { return n > 1 ? stride : 0; };
    *v = {static_cast<unsigned char*>(c->k), static_cast<unsigned char*>(c->v), e4m3 ? c->k_scale : nullptr, e4m3 ? c->v_scale : nullptr, c->num_blocks,
          elem * step(c->stride_block, c->num_blocks), elem * step(c->stride_token, c->block_size), elem * step(c->stride_head, c->num_kv_heads),
          step(c->scale_stride_block, c->num_blocks), step(c->scale_stride_token, c->block_size), step(c->scale_stride_head, c->num_kv_heads),
          c->block_size, c->num_kv_heads, c->head_dim, e4m3};
    return FP8LIN_OK;
}

int check_rows(const char* what, const void* k, int64_t kt, int64_t kh, const void* v, int64_t vt, int64_t vh, int64_t rows, int64_t heads) {
    if (!k || !v) return set_error(FP8LIN_ERR_NULL, "%s: k and v must not be NULL", what);
    if (!aligned16(k) || !aligned16(v) || bad_stride(kt, rows, 8) || bad_stride(vt, rows, 8) || bad_stride(kh, heads, 8) || bad_stride(vh, heads, 8))
        return set_error(FP8LIN_ERR_ALIGN, "%s: k and v must be 16-byte aligned with strides that are positive multiples of 8 elements", what);
    return FP8LIN_OK;
}

int check_tables(const int32_t* tables, int64_t ld, int64_t max_pages, int64_t batch) {
    if (batch < 0 || batch > (1ll << 24)) return set_error(FP8LIN_ERR_SHAPE, "bad batch %lld", (long long)batch);
    if (max_pages < 0 || max_pages > (1ll << 31) - 1 || (batch > 1 && ld < max_pages))
        return set_error(FP8LIN_ERR_SHAPE, "bad block tables: ld_tables=%lld max_pages=%lld", (long long)ld, (long long)max_pages);
    if (!tables && max_pages > 0 && batch > 0) return set_error(FP8LIN_ERR_NULL, "block_tables must not be NULL");
    return FP8LIN_OK;
}

int check_scratch(const void* workspace, size_t bytes, size_t need) {
    if (!workspace || bytes < need) return set_error(FP8LIN_ERR_WORKSPACE, "workspace too small: need %zu bytes", need);
    if ((reinterpret_cast<uintptr_t>(workspace) & 255) != 0) return set_error(FP8LIN_ERR_ALIGN, "workspace must be 256-byte aligned");
    if (!device_is_sm100()) return set_error(FP8LIN_ERR_ARCH, "fp8lin kernels are built for sm_100a only");
    return FP8LIN_OK;
}

}  // namespace

extern "C" {

int fp8lin_kv_cache_write(const fp8lin_kv_cache* cache, const void* k, int64_t k_stride_token, int64_t k_stride_head, const void* v,
                          int64_t v_stride_token, int64_t v_stride_head, const int32_t* slot_mapping, int64_t tokens, void* workspace,
                          size_t workspace_bytes, void* stream) {
    CacheView c;
    if (int rc = view_of(cache, &c)) return rc;
    if (tokens < 0 || tokens > (1ll << 30)) return set_error(FP8LIN_ERR_SHAPE, "bad number of tokens %lld", (long long)tokens);
    if (tokens == 0) return FP8LIN_OK;
    if (!slot_mapping) return set_error(FP8LIN_ERR_NULL, "slot_mapping must not be NULL");
    if (int rc = check_rows("fp8lin_kv_cache_write", k, k_stride_token, k_stride_head, v, v_stride_token, v_stride_head, tokens, c.kv_heads)) return rc;
    if (int rc = check_scratch(workspace, workspace_bytes, FP8LIN_WS_HEADER_BYTES)) return rc;
    const CacheRows x = {(__nv_bfloat16*)k, (__nv_bfloat16*)v, k_stride_token, k_stride_head, v_stride_token, v_stride_head, tokens};
    const cudaError_t e = launch_kv_cache_write(c, x, slot_mapping, ws_view(workspace, workspace_bytes).status, (cudaStream_t)stream);
    if (e != cudaSuccess) return set_error(FP8LIN_ERR_LAUNCH, "cache write launch: %s", cudaGetErrorString(e));
    return FP8LIN_OK;
}

int fp8lin_kv_cache_read(const fp8lin_kv_cache* cache, const int32_t* block_tables, int64_t ld_tables, int64_t max_pages, const int32_t* cu_seqlens,
                         int64_t batch, void* k, int64_t k_stride_token, int64_t k_stride_head, void* v, int64_t v_stride_token, int64_t v_stride_head,
                         int64_t rows, void* workspace, size_t workspace_bytes, void* stream) {
    CacheView c;
    if (int rc = view_of(cache, &c)) return rc;
    if (int rc = check_tables(block_tables, ld_tables, max_pages, batch)) return rc;
    if (rows < 0 || rows > (1ll << 30)) return set_error(FP8LIN_ERR_SHAPE, "bad number of rows %lld", (long long)rows);
    if (rows == 0 || batch == 0) return FP8LIN_OK;
    if (!cu_seqlens) return set_error(FP8LIN_ERR_NULL, "cu_seqlens must not be NULL");
    if (int rc = check_rows("fp8lin_kv_cache_read", k, k_stride_token, k_stride_head, v, v_stride_token, v_stride_head, rows, c.kv_heads)) return rc;
    if (int rc = check_scratch(workspace, workspace_bytes, FP8LIN_WS_HEADER_BYTES)) return rc;
    const CacheRows y = {(__nv_bfloat16*)k, (__nv_bfloat16*)v, k_stride_token, k_stride_head, v_stride_token, v_stride_head, rows};
    const cudaError_t e = launch_kv_cache_read(c, y, block_tables, ld_tables, max_pages, cu_seqlens, batch, ws_view(workspace, workspace_bytes).status,
                                               (cudaStream_t)stream);
    if (e != cudaSuccess) return set_error(FP8LIN_ERR_LAUNCH, "cache read launch: %s", cudaGetErrorString(e));
    return FP8LIN_OK;
}

size_t fp8lin_paged_attention_workspace_bytes(int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int dtype) {
    if (num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
    return FP8LIN_WS_HEADER_BYTES + paged_attention_scratch(num_heads, num_kv_heads, head_dim, dtype == FP8LIN_CACHE_E4M3);
}

int fp8lin_paged_attention(const fp8lin_kv_cache* cache, const void* q, int64_t q_stride_row, int64_t q_stride_head, const int32_t* block_tables,
                           int64_t ld_tables, int64_t max_pages, const int32_t* context_lens, int64_t batch, int64_t num_heads, float scale,
                           const float* out_scale, void* out, int64_t ld_out, void* workspace, size_t workspace_bytes, void* stream) {
    AttnArgs a = {};
    if (int rc = view_of(cache, &a.c)) return rc;
    if (int rc = check_tables(block_tables, ld_tables, max_pages, batch)) return rc;
    if (num_heads <= 0 || num_heads % a.c.kv_heads != 0 || num_heads > 65535)
        return set_error(FP8LIN_ERR_SHAPE, "num_heads=%lld must be a multiple of num_kv_heads=%d", (long long)num_heads, a.c.kv_heads);
    if (batch * num_heads > 0x7fffffff) return set_error(FP8LIN_ERR_SHAPE, "batch=%lld times num_heads=%lld is too large", (long long)batch, (long long)num_heads);
    if (batch == 0) return FP8LIN_OK;
    if (!q || !context_lens || !out) return set_error(FP8LIN_ERR_NULL, "q, context_lens and out must not be NULL");
    if (!aligned16(q) || bad_stride(q_stride_row, batch, 8) || bad_stride(q_stride_head, num_heads, 8))
        return set_error(FP8LIN_ERR_ALIGN, "q must be 16-byte aligned with strides that are positive multiples of 8 elements");
    if (!aligned16(out) || (batch > 1 && (ld_out < num_heads * a.c.dim || ld_out % (out_scale ? 16 : 8) != 0)))
        return set_error(FP8LIN_ERR_ALIGN, "out must be 16-byte aligned, its rows at least num_heads * head_dim elements and whole 16-byte words apart");
    const size_t need = fp8lin_paged_attention_workspace_bytes(num_heads, a.c.kv_heads, a.c.dim, cache->dtype);
    if (int rc = check_scratch(workspace, workspace_bytes, need)) return rc;
    const WsView ws = ws_view(workspace, workspace_bytes);
    a.q = (const __nv_bfloat16*)q;
    a.q_row = batch > 1 ? q_stride_row : 0;
    a.q_head = num_heads > 1 ? q_stride_head : 0;
    a.tables = block_tables;
    a.ld_tables = ld_tables;
    a.max_pages = max_pages;
    a.lens = context_lens;
    a.batch = (int)batch;
    a.heads = (int)num_heads;
    a.scale = scale;
    a.out_scale = out_scale;
    a.out = out;
    a.ld_out = ld_out;
    a.status = ws.status;
    a.counters = ws.counters;
    a.partial = reinterpret_cast<float*>(ws.body);
    const cudaError_t e = launch_paged_attention(a, (cudaStream_t)stream);
    if (e != cudaSuccess) return set_error(FP8LIN_ERR_LAUNCH, "paged attention launch: %s", cudaGetErrorString(e));
    return FP8LIN_OK;
}

}  // extern "C"
