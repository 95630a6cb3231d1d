// C entry points of ragged paged attention over 8-bit pools: argument checks and the choice of kernel.
#include "attn_q8.cuh"

namespace ns {
int launch_q8_simple(const Q8Params& p, int dtype, int pool_dtype, cudaStream_t st);
bool q8_decode_supported(const Q8Params& p, int dtype);
int launch_q8_decode(const Q8Params& p, int dtype, int pool_dtype, cudaStream_t st);
bool q8_prefill_supported(const Q8Params& p, int dtype);
int launch_q8_prefill(const Q8Params& p, int pool_dtype, int max_items, cudaStream_t st);
}

using namespace ns;

static int fill_params(Q8Params& p, const void* q, const void* k_pool, const void* v_pool, const float* k_scale, const float* v_scale,
                       const int32_t* block_tables, const int32_t* table_rows, const int32_t* seq_lens, const int32_t* cu_seqlens, void* out,
                       int32_t n_seqs, int64_t n_tokens, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int32_t block_size,
                       int32_t num_blocks, int32_t table_width, int64_t table_stride, int64_t q_stride, int64_t out_stride,
                       int64_t pool_block_stride, int64_t pool_pos_stride, int64_t pool_head_stride, int64_t scale_block_stride,
                       int64_t scale_head_stride, float scale, int dtype, int pool_dtype) {
    NS_REQUIRE(n_seqs >= 0 && n_tokens >= 0 && n_heads > 0 && n_kv_heads > 0 && head_dim > 0 && block_size > 0 && num_blocks >= 0 &&
                   table_width >= 0, NS_ERR_INVALID_ARG, "attn_q8: bad shape");
    NS_REQUIRE(n_heads % n_kv_heads == 0, NS_ERR_INVALID_ARG, "attn_q8: %d heads not divisible by %d kv heads", n_heads, n_kv_heads);
    NS_REQUIRE(dtype == NS_BF16 || dtype == NS_F32, NS_ERR_UNSUPPORTED, "attn_q8: dtype %d", dtype);
    NS_REQUIRE(pool_dtype == NS_INT8 || pool_dtype == NS_E4M3, NS_ERR_UNSUPPORTED, "attn_q8: pool dtype %d is not an 8-bit one", pool_dtype);
    NS_REQUIRE(cu_seqlens != nullptr || n_tokens == n_seqs, NS_ERR_INVALID_ARG, "attn_q8: without cu_seqlens every sequence has one token");
    NS_REQUIRE(n_tokens * n_heads < ((int64_t)1 << 33), NS_ERR_UNSUPPORTED, "attn_q8: %lld tokens", (long long)n_tokens);
    if (n_seqs > 0 && n_tokens > 0)
        NS_REQUIRE(q && k_pool && v_pool && k_scale && v_scale && block_tables && seq_lens && out, NS_ERR_INVALID_ARG, "attn_q8: null pointer");
    p = Q8Params{};
    p.q = q; p.k_pool = (const uint8_t*)k_pool; p.v_pool = (const uint8_t*)v_pool; p.k_scale = k_scale; p.v_scale = v_scale;
    p.block_tables = block_tables; p.table_rows = table_rows; p.seq_lens = seq_lens; p.cu_seqlens = cu_seqlens; p.out = out;
    p.n_tokens = n_tokens; p.table_stride = table_stride; p.q_stride = q_stride; p.out_stride = out_stride;
    p.blk_stride = pool_block_stride; p.pos_stride = pool_pos_stride; p.head_stride = pool_head_stride;
    p.sc_blk_stride = scale_block_stride; p.sc_head_stride = scale_head_stride;
    p.n_seqs = n_seqs; p.n_heads = n_heads; p.n_kv_heads = n_kv_heads; p.group = n_heads / n_kv_heads; p.head_dim = head_dim;
    p.block_size = block_size; p.num_blocks = num_blocks; p.table_width = table_width;
    p.block_shift = (block_size & (block_size - 1)) == 0 ? 31 - __builtin_clz((unsigned)block_size) : -1;
    p.scale = scale; p.scale_log2 = scale * 1.4426950408889634f;
    return NS_OK;
}

extern "C" int ns_ragged_paged_attn_q8_simple(const void* q, const void* k_pool, const void* v_pool, const float* k_scale, const float* v_scale,
                                              const int32_t* block_tables, const int32_t* table_rows, const int32_t* seq_lens,
                                              const int32_t* cu_seqlens, void* out, int32_t n_seqs, int64_t n_tokens, int32_t n_heads,
                                              int32_t n_kv_heads, int32_t head_dim, int32_t block_size, int32_t num_blocks,
                                              int32_t table_width, int64_t table_stride, int64_t q_stride, int64_t out_stride,
                                              int64_t pool_block_stride, int64_t pool_pos_stride, int64_t pool_head_stride,
                                              int64_t scale_block_stride, int64_t scale_head_stride, float scale, int dtype, int pool_dtype,
                                              void* stream) {
    Q8Params p;
    const int rc = fill_params(p, q, k_pool, v_pool, k_scale, v_scale, block_tables, table_rows, seq_lens, cu_seqlens, out, n_seqs, n_tokens,
                               n_heads, n_kv_heads, head_dim, block_size, num_blocks, table_width, table_stride, q_stride, out_stride,
                               pool_block_stride, pool_pos_stride, pool_head_stride, scale_block_stride, scale_head_stride, scale, dtype, pool_dtype);
    if (rc != NS_OK || n_seqs == 0 || n_tokens == 0) return rc;
    return launch_q8_simple(p, dtype, pool_dtype, (cudaStream_t)stream);
}

extern "C" int ns_ragged_paged_attn_q8(const void* q, const void* k_pool, const void* v_pool, const float* k_scale, const float* v_scale,
                                       const int32_t* block_tables, const int32_t* table_rows, const int32_t* seq_lens,
                                       const int32_t* cu_seqlens, void* out, int32_t n_seqs, int64_t n_tokens, int32_t n_heads,
                                       int32_t n_kv_heads, int32_t head_dim, int32_t block_size, int32_t num_blocks, int32_t table_width,
                                       int64_t table_stride, int64_t q_stride, int64_t out_stride, int64_t pool_block_stride,
                                       int64_t pool_pos_stride, int64_t pool_head_stride, int64_t scale_block_stride,
                                       int64_t scale_head_stride, float scale, int dtype, int pool_dtype, void* workspace,
                                       int64_t workspace_bytes, int32_t ws_max_seqs, int32_t ws_max_tokens, void* stream) {
    Q8Params p;
    int rc = fill_params(p, q, k_pool, v_pool, k_scale, v_scale, block_tables, table_rows, seq_lens, cu_seqlens, out, n_seqs, n_tokens,
                         n_heads, n_kv_heads, head_dim, block_size, num_blocks, table_width, table_stride, q_stride, out_stride,
                         pool_block_stride, pool_pos_stride, pool_head_stride, scale_block_stride, scale_head_stride, scale, dtype, pool_dtype);
    if (rc != NS_OK || n_seqs == 0 || n_tokens == 0) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if (!q8_decode_supported(p, dtype)) return launch_q8_simple(p, dtype, pool_dtype, st);
    NS_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0, NS_ERR_INVALID_ARG,
               "attn_q8: workspace is null or not 256-byte aligned");
    NS_REQUIRE(n_seqs <= ws_max_seqs && n_tokens <= ws_max_tokens, NS_ERR_WORKSPACE,
               "attn_q8: batch (%d seqs, %lld tokens) exceeds workspace capacity (%d, %d)", n_seqs, (long long)n_tokens, ws_max_seqs, ws_max_tokens);
    p.L = ws_layout(ws_max_seqs, ws_max_tokens, n_heads, head_dim);
    NS_REQUIRE(workspace_bytes >= p.L.total, NS_ERR_WORKSPACE, "attn_q8: workspace of %lld bytes < %lld needed", (long long)workspace_bytes,
               (long long)p.L.total);
    p.ws = (uint8_t*)workspace;
    p.sm_count = device_sm_count();
    NS_REQUIRE(p.sm_count > 0, NS_ERR_CUDA, "attn_q8: cannot query the SM count");
    const bool prefill = cu_seqlens != nullptr && n_tokens > 1, tc = prefill && q8_prefill_supported(p, dtype);
    p.overlap_prefill = tc ? 1 : 0;
    rc = launch_q8_decode(p, dtype, pool_dtype, st);
    if (rc != NS_OK || !prefill) return rc;
    rc = NS_ERR_UNSUPPORTED;
    if (tc) {
        // upper bound on prefill tiles from sizes the host knows (graph-safe)
        int64_t max_items = n_tokens / kPrefillTileTokens + n_seqs;
        const int64_t cap = (int64_t)ws_max_tokens / kPrefillTileTokens + ws_max_seqs + 1;
        rc = launch_q8_prefill(p, pool_dtype, (int)(max_items < cap ? max_items : cap), st);
    }
    if (rc != NS_ERR_UNSUPPORTED) return rc;
    p.only_prefill = 1;
    return launch_q8_simple(p, dtype, pool_dtype, st);
}
