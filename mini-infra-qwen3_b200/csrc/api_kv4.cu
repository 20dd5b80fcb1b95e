// C-ABI entry points of the 4-bit paged cache (include/mi_kv4.h) and of the block copies
// (mi_kv_copy_blocks): host-side argument checks, then launches on the caller's stream.
#include "../../include/mi_kv4.h"

#include "common.cuh"
#include "kernels.cuh"
#include "kv4_format.cuh"

namespace {

constexpr int64_t kMaxGrid = (int64_t(1) << 31) - 1;

int check_kv4_geometry(int64_t num_blocks, int block_size, int num_kv_heads, int head_dim, int dtype,
                       const void* k_pool, const void* v_pool) {
  if (int rc = check_pool_geometry(num_blocks, block_size, num_kv_heads, head_dim, dtype)) return rc;
  if (mi_kv4_page_bytes(block_size, head_dim) == 0)
    return fail(MI_ERR_INVALID, "a 4-bit cache needs head_dim a multiple of %d up to 256 (got %d)", MI_KV4_GROUP,
                head_dim);
  if (!aligned(k_pool, 4) || !aligned(v_pool, 4)) return fail(MI_ERR_INVALID, "4-bit pools must be 4-byte aligned");
  if (mi_kv4_page_bytes(block_size, head_dim) > kMaxGrid)
    return fail(MI_ERR_UNSUPPORTED, "pages of more than 2^31 - 1 bytes");
  if (num_blocks > kMaxGrid / block_size)
    return fail(MI_ERR_UNSUPPORTED, "a pool of more than 2^31 - 1 tokens (%lld blocks of %d)", (long long)num_blocks,
                block_size);
  return MI_OK;
}

// Whether eight consecutive source values are 16-byte loads.
bool kv4_vec(const void* k_src, const void* v_src, const mi::Kv4StoreArgs& a) {
  return pick_vec({k_src, v_src}, {a.k_sb[0], a.k_sb[1], a.k_sb[2], a.v_sb[0], a.v_sb[1], a.v_sb[2]}) == 16;
}

int fill_kv4_store(mi::Kv4StoreArgs& a, const void* k_src, const void* v_src, const int64_t* k_strides,
                   const int64_t* v_strides, void* k_pool, void* v_pool, int64_t num_blocks, int block_size,
                   int num_kv_heads, int head_dim, int dtype) {
  const int es = elem_size(dtype);
  if (!aligned(k_src, es) || !aligned(v_src, es)) return fail(MI_ERR_INVALID, "misaligned source");
  a.k_src = static_cast<const char*>(k_src);
  a.v_src = static_cast<const char*>(v_src);
  for (int i = 0; i < 3; ++i) {
    a.k_sb[i] = k_strides[i] * es;
    a.v_sb[i] = v_strides[i] * es;
  }
  a.k_pool = static_cast<char*>(k_pool);
  a.v_pool = static_cast<char*>(v_pool);
  a.num_blocks = num_blocks;
  a.page_bytes = mi_kv4_page_bytes(block_size, head_dim);
  a.block_size = block_size;
  a.heads = num_kv_heads;
  a.head_dim = head_dim;
  return MI_OK;
}

}  // namespace

extern "C" {

int64_t mi_kv4_page_bytes(int block_size, int head_dim) {
  if (block_size < 1 || head_dim < MI_KV4_GROUP || head_dim > 256 || head_dim % MI_KV4_GROUP) return 0;
  return mi::kv4_page_bytes(block_size, head_dim);
}

int mi_kv4_scatter(const void* k_src, const void* v_src, const int64_t* k_strides, const int64_t* v_strides,
                   int64_t src_rows, int64_t src_positions, const int64_t* token_rows,
                   const int64_t* token_positions, const int64_t* slot_mapping, int64_t num_tokens, void* k_pool,
                   void* v_pool, int64_t num_blocks, int block_size, int num_kv_heads, int head_dim, int dtype,
                   void* stream) {
  if (int rc = check_kv4_geometry(num_blocks, block_size, num_kv_heads, head_dim, dtype, k_pool, v_pool)) return rc;
  if (num_tokens < 0) return fail(MI_ERR_INVALID, "num_tokens < 0");
  if (num_tokens == 0) return MI_OK;
  if (num_tokens > kMaxGrid) return fail(MI_ERR_UNSUPPORTED, "%lld tokens exceed one launch", (long long)num_tokens);
  if (!k_src || !v_src || !k_strides || !v_strides || !slot_mapping || !k_pool || !v_pool)
    return fail(MI_ERR_INVALID, "mi_kv4_scatter: null pointer argument");
  mi::Kv4StoreArgs a{};
  if (int rc = fill_kv4_store(a, k_src, v_src, k_strides, v_strides, k_pool, v_pool, num_blocks, block_size,
                              num_kv_heads, head_dim, dtype))
    return rc;
  a.rows = token_rows;
  a.positions = token_positions;
  a.slots = slot_mapping;
  a.num_tokens = num_tokens;
  a.src_rows = src_rows;
  a.src_positions = src_positions;
  cudaError_t e = mi::launch_kv4_store(a, false, kv4_vec(k_src, v_src, a), dtype, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MI_OK : cuda_fail(e, "mi_kv4_scatter launch");
}

int mi_kv4_store_chunks(const void* k_src, const void* v_src, const int64_t* k_strides, const int64_t* v_strides,
                        int64_t batch, int64_t padded_len, const int64_t* chunk_lens, const int64_t* start_positions,
                        const int64_t* block_tables, int64_t table_stride, int64_t table_width, void* k_pool,
                        void* v_pool, int64_t num_blocks, int block_size, int num_kv_heads, int head_dim, int dtype,
                        void* stream) {
  if (int rc = check_kv4_geometry(num_blocks, block_size, num_kv_heads, head_dim, dtype, k_pool, v_pool)) return rc;
  if (batch < 0 || padded_len < 0 || table_width < 0) return fail(MI_ERR_INVALID, "negative size");
  if (batch == 0 || padded_len == 0) return MI_OK;
  if (!k_src || !v_src || !k_strides || !v_strides || !chunk_lens || !start_positions || !block_tables || !k_pool ||
      !v_pool)
    return fail(MI_ERR_INVALID, "mi_kv4_store_chunks: null pointer argument");
  if (padded_len > kMaxGrid / batch || table_width > kMaxGrid / block_size)
    return fail(MI_ERR_UNSUPPORTED, "%lld x %lld positions or %lld blocks a row exceed one launch", (long long)batch,
                (long long)padded_len, (long long)table_width);
  if (batch > 1 && table_stride < table_width)
    return fail(MI_ERR_INVALID, "block table rows of %lld entries at stride %lld", (long long)table_width,
                (long long)table_stride);
  mi::Kv4StoreArgs a{};
  if (int rc = fill_kv4_store(a, k_src, v_src, k_strides, v_strides, k_pool, v_pool, num_blocks, block_size,
                              num_kv_heads, head_dim, dtype))
    return rc;
  a.batch = batch;
  a.padded_len = padded_len;
  a.chunk_lens = chunk_lens;
  a.starts = start_positions;
  a.block_tables = block_tables;
  a.table_stride = table_stride;
  a.table_width = table_width;
  cudaError_t e = mi::launch_kv4_store(a, true, kv4_vec(k_src, v_src, a), dtype, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MI_OK : cuda_fail(e, "mi_kv4_store_chunks launch");
}

int mi_kv4_gather_blocks(const void* k_pool, const void* v_pool, const int64_t* block_ids, int64_t id_stride,
                         const int64_t* lengths, int fill_past, int64_t batch, int64_t blocks_per_row, void* k_out,
                         void* v_out, int64_t num_blocks, int block_size, int num_kv_heads, int head_dim, int dtype,
                         void* stream) {
  if (int rc = check_kv4_geometry(num_blocks, block_size, num_kv_heads, head_dim, dtype, k_pool, v_pool)) return rc;
  if (batch < 0 || blocks_per_row < 0) return fail(MI_ERR_INVALID, "negative size");
  if (batch == 0 || blocks_per_row == 0) return MI_OK;
  if (!k_pool || !v_pool || !block_ids || !k_out || !v_out)
    return fail(MI_ERR_INVALID, "mi_kv4_gather_blocks: null pointer argument");
  if (batch > 1 && id_stride < blocks_per_row)
    return fail(MI_ERR_INVALID, "block id rows of %lld entries at stride %lld", (long long)blocks_per_row,
                (long long)id_stride);
  if (!aligned(k_out, 16) || !aligned(v_out, 16)) return fail(MI_ERR_INVALID, "outputs must be 16-byte aligned");
  if (blocks_per_row > kMaxGrid / batch)
    return fail(MI_ERR_UNSUPPORTED, "%lld x %lld blocks exceed one launch", (long long)batch,
                (long long)blocks_per_row);
  if ((int64_t)block_size * num_kv_heads * head_dim > (int64_t(1) << 30))
    return fail(MI_ERR_UNSUPPORTED, "a block of more than 2^30 values");
  mi::Kv4GatherArgs a{};
  a.k_pool = static_cast<const char*>(k_pool);
  a.v_pool = static_cast<const char*>(v_pool);
  a.block_ids = block_ids;
  a.id_stride = id_stride;
  a.lengths = lengths;
  a.fill_past = fill_past;
  a.batch = batch;
  a.blocks_per_row = blocks_per_row;
  a.k_out = static_cast<char*>(k_out);
  a.v_out = static_cast<char*>(v_out);
  a.num_blocks = num_blocks;
  a.page_bytes = mi_kv4_page_bytes(block_size, head_dim);
  a.block_size = block_size;
  a.heads = num_kv_heads;
  a.head_dim = head_dim;
  cudaError_t e = mi::launch_kv4_gather(a, dtype, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MI_OK : cuda_fail(e, "mi_kv4_gather_blocks launch");
}

int mi_kv4_qk_norm_rope(const void* q, int64_t q_row_stride, const void* k, int64_t k_row_stride, const void* v,
                        int64_t v_row_stride, const void* q_weight, const void* k_weight, const void* cos,
                        const void* sin, int64_t cos_sin_row_stride, int64_t tokens, int hq, int hkv, int head_dim,
                        float eps, void* q_out, void* k_out, void* v_out, const int64_t* slot_mapping, void* k_pool,
                        void* v_pool, int64_t num_blocks, int block_size, int dtype, void* stream) {
  if (int rc = check_kv4_geometry(num_blocks, block_size, hkv, head_dim, dtype, k_pool, v_pool)) return rc;
  if (tokens > 0 && !slot_mapping) return fail(MI_ERR_INVALID, "mi_kv4_qk_norm_rope: null slot_mapping");
  return qk_norm_rope_impl(q, q_row_stride, k, k_row_stride, v, v_row_stride, q_weight, k_weight, cos, sin,
                           cos_sin_row_stride, tokens, hq, hkv, head_dim, eps, q_out, k_out, v_out, slot_mapping, k_pool,
                           v_pool, num_blocks * block_size, mi_kv4_page_bytes(block_size, head_dim), block_size, dtype,
                           stream);
}

size_t mi_kv4_paged_decode_workspace_size(int64_t batch, int num_q_heads, int num_kv_heads, int head_dim,
                                          int64_t max_blocks_per_seq, int block_size, int dtype) {
  if (batch <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || max_blocks_per_seq <= 0 ||
      mi_kv4_page_bytes(block_size, head_dim) == 0 || max_blocks_per_seq > kMaxGrid / block_size)
    return 0;
  return mi::plan_kv4_decode(batch, num_q_heads, num_kv_heads, head_dim, max_blocks_per_seq, block_size, dtype)
      .ws_bytes;
}

int mi_kv4_paged_decode(const void* q, const int64_t* q_strides, const void* k_new, const void* v_new,
                        const int64_t* new_strides, const int64_t* slot_mapping, void* k_pool, void* v_pool,
                        int64_t num_blocks, int block_size, int num_kv_heads, int head_dim,
                        const int64_t* block_tables, int64_t table_stride, int64_t max_blocks_per_seq,
                        const int64_t* context_lens, int64_t batch, int num_q_heads, float scale, void* out,
                        int64_t out_stride, void* workspace, size_t workspace_bytes, int dtype, void* stream) {
  if (int rc = check_kv4_geometry(num_blocks, block_size, num_kv_heads, head_dim, dtype, k_pool, v_pool)) return rc;
  if (batch < 0) return fail(MI_ERR_INVALID, "batch < 0");
  if (batch == 0) return MI_OK;
  if (batch > 65535) return fail(MI_ERR_UNSUPPORTED, "batch %lld exceeds 65535", (long long)batch);
  if (num_q_heads < 1 || num_q_heads % num_kv_heads != 0)
    return fail(MI_ERR_INVALID, "num_q_heads (%d) must be a positive multiple of num_kv_heads (%d)", num_q_heads,
                num_kv_heads);
  if (batch * num_q_heads > kMaxGrid)
    return fail(MI_ERR_UNSUPPORTED, "%lld x %d rows exceed one launch", (long long)batch, num_q_heads);
  if (!q || !q_strides || !k_pool || !v_pool || !block_tables || !context_lens || !out)
    return fail(MI_ERR_INVALID, "mi_kv4_paged_decode: null pointer argument");
  if (max_blocks_per_seq < 1 || (batch > 1 && table_stride < max_blocks_per_seq))
    return fail(MI_ERR_INVALID, "block table needs at least one column (max_blocks=%lld, stride=%lld)",
                (long long)max_blocks_per_seq, (long long)table_stride);
  if (max_blocks_per_seq > kMaxGrid / block_size)  // tokens of a row are counted in 32 bits
    return fail(MI_ERR_UNSUPPORTED, "block tables of %lld blocks of %d: more than 2^31 - 1 tokens a row",
                (long long)max_blocks_per_seq, block_size);
  const int es = elem_size(dtype);
  if (!aligned(q, es) || !aligned(out, es)) return fail(MI_ERR_INVALID, "mi_kv4_paged_decode: misaligned operands");
  mi::Kv4DecodePlan plan =
      mi::plan_kv4_decode(batch, num_q_heads, num_kv_heads, head_dim, max_blocks_per_seq, block_size, dtype);
  // the tensor-core kernel copies 16-byte aligned pages; head_dim >= 64 makes every page a multiple of 16
  if (plan.use_mma && !(aligned(k_pool, 16) && aligned(v_pool, 16))) plan = mi::Kv4DecodePlan{};
  if (plan.ws_bytes && (!workspace || workspace_bytes < plan.ws_bytes || !aligned(workspace, 256)))
    return fail(MI_ERR_INVALID, "workspace must be >= %zu bytes and 256-byte aligned (got %zu)", plan.ws_bytes,
                workspace_bytes);
  if (k_new || v_new || slot_mapping) {
    if (!k_new || !v_new || !slot_mapping || !new_strides)
      return fail(MI_ERR_INVALID, "k_new, v_new, new_strides and slot_mapping go together");
    const int64_t st[3] = {new_strides[0], new_strides[1], 0};
    if (int rc = mi_kv4_scatter(k_new, v_new, st, st, batch, 1, nullptr, nullptr, slot_mapping, batch, k_pool, v_pool,
                                num_blocks, block_size, num_kv_heads, head_dim, dtype, stream))
      return rc;
  }
  mi::Kv4DecodeArgs a{};
  a.q = static_cast<const char*>(q);
  a.q_sb = q_strides[0] * es;
  a.q_sh = q_strides[1] * es;
  a.k_pool = static_cast<const char*>(k_pool);
  a.v_pool = static_cast<const char*>(v_pool);
  a.page_bytes = mi_kv4_page_bytes(block_size, head_dim);
  a.block_tables = block_tables;
  a.table_stride = table_stride;
  a.max_blocks = max_blocks_per_seq;
  a.context_lens = context_lens;
  a.batch = batch;
  a.num_blocks = num_blocks;
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  a.groups = num_q_heads / num_kv_heads;
  a.head_dim = head_dim;
  a.block_size = block_size;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = static_cast<char*>(out);
  a.out_sb = out_stride * es;
  a.ctas = plan.ctas;
  a.whole = plan.whole;
  a.min_steps = plan.min_steps;
  a.part_rows = plan.part_rows;
  if (plan.ws_bytes) {
    char* ws = static_cast<char*>(workspace);
    a.ws_o = reinterpret_cast<float*>(ws);
    a.ws_ml = reinterpret_cast<float*>(ws + plan.o_bytes);
    a.cuts = reinterpret_cast<mi::Kv4Cut*>(ws + plan.o_bytes + plan.ml_bytes);
  }
  cudaError_t e = mi::launch_kv4_decode(a, plan, dtype, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MI_OK : cuda_fail(e, "mi_kv4_paged_decode launch");
}

int mi_kv_copy_blocks(void* const* pools, int num_pools, const int64_t* pairs, int64_t num_pairs,
                      int64_t num_blocks, int64_t block_bytes, void* stream) {
  if (num_pools < 0 || num_pairs < 0) return fail(MI_ERR_INVALID, "negative size");
  if (num_blocks < 1 || block_bytes < 1)
    return fail(MI_ERR_INVALID, "pool geometry must be positive (blocks=%lld, bytes=%lld)", (long long)num_blocks,
                (long long)block_bytes);
  if (num_pools == 0 || num_pairs == 0) return MI_OK;
  if (!pools || !pairs) return fail(MI_ERR_INVALID, "mi_kv_copy_blocks: null pointer argument");
  if (num_pairs > kMaxGrid) return fail(MI_ERR_UNSUPPORTED, "%lld pairs exceed one launch", (long long)num_pairs);
  for (int first = 0; first < num_pools; first += mi::kMaxCopyPools) {
    mi::PageCopyArgs a{};
    a.num_pools = num_pools - first < mi::kMaxCopyPools ? num_pools - first : mi::kMaxCopyPools;
    a.pairs = pairs;
    a.num_pairs = num_pairs;
    a.num_blocks = num_blocks;
    a.block_bytes = block_bytes;
    int vec = pick_vec({}, {block_bytes});
    for (int i = 0; i < a.num_pools; ++i) {
      if (!pools[first + i]) return fail(MI_ERR_INVALID, "mi_kv_copy_blocks: pool %d is null", first + i);
      a.pools[i] = static_cast<char*>(pools[first + i]);
      vec = std::min(vec, pick_vec({pools[first + i]}, {}));
    }
    cudaError_t e = mi::launch_page_copy(a, vec, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(e, "mi_kv_copy_blocks launch");
  }
  return MI_OK;
}

}  // extern "C"
