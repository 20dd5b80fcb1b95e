/*
 * mi_kv4.h — C ABI of the 4-bit paged KV cache (libmi_paged.so, sm_100a).
 *
 * A cache whose pages hold 4-bit codes: 5 bits a value with the parameters, 3.2 times the tokens of
 * a 16-bit pool in the same memory and 3.2 times fewer bytes per decode step.  The conventions are
 * those of mi_paged.h: plain device pointers, element strides, int64 metadata, asynchronous on the
 * given stream, no allocation, MI_ERR_* codes, device-side checks in the status word.
 *
 * Format.  The head_dim values of one token and KV head are cut into groups of MI_KV4_GROUP = 32.
 * A group x stands for m + s * c with bfloat16 minimum m and step s and codes c in 0..15:
 *     m = bf16(min x),  s = bf16((max x - m) / 15),  c = clamp(round((x - m) / s), 0, 15)
 * in fp32 arithmetic, rounding to nearest even; c = 0 where s = 0; a zero m is +0.  A group with an infinity or a
 * NaN (or whose m or s overflows bfloat16) is stored as m = NaN, s = 0: it reads back as NaN.
 *   pool   uint8 [num_blocks, num_kv_heads, mi_kv4_page_bytes(block_size, head_dim)], contiguous
 *   page   codes [head_dim/32, block_size, 16 bytes]: byte i of a group holds value 2i in its low and
 *          value 2i + 1 in its high four bits; then parameters [block_size, head_dim/32] of (s, m),
 *          two bfloat16 each
 * head_dim is a multiple of 32, at most 256; any block_size.  An all-zero page reads as zeros; block 0
 * is the null block, as in mi_paged.h.  `dtype` is the type of the dense operands (q, K/V, outputs).
 */
#ifndef MI_KV4_H
#define MI_KV4_H

#include "mi_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MI_KV4_GROUP 32

/* Bytes of one page (one block of one KV head): block_size * head_dim * 5 / 8; 0 for a geometry the
 * format does not have. */
int64_t mi_kv4_page_bytes(int block_size, int head_dim);

/*
 * mi_kv4_scatter — mi_kv_scatter into 4-bit pools: token i, the source's (token_rows[i], :,
 * token_positions[i], :), is quantised into slot slot_mapping[i] of both pools.  Source strides,
 * NULL index arrays, bounds and flags as in mi_kv_scatter.  Slots must be distinct.
 */
int mi_kv4_scatter(const void* k_src, const void* v_src, const int64_t* k_strides, const int64_t* v_strides,
                   int64_t src_rows, int64_t src_positions, const int64_t* token_rows,
                   const int64_t* token_positions, const int64_t* slot_mapping, int64_t num_tokens, void* k_pool,
                   void* v_pool, int64_t num_blocks, int block_size, int num_kv_heads, int head_dim, int dtype,
                   void* stream);

/*
 * mi_kv4_store_chunks — mi_kv_store_chunks into 4-bit pools: row b's last chunk_lens[b] positions are
 * quantised at logical positions start_positions[b] + j, slots from the block tables.  table_width
 * columns of a row are valid to read.
 */
int mi_kv4_store_chunks(const void* k_src, const void* v_src, const int64_t* k_strides, const int64_t* v_strides,
                        int64_t batch, int64_t padded_len, const int64_t* chunk_lens, const int64_t* start_positions,
                        const int64_t* block_tables, int64_t table_stride, int64_t table_width, void* k_pool,
                        void* v_pool, int64_t num_blocks, int block_size, int num_kv_heads, int head_dim, int dtype,
                        void* stream);

/*
 * mi_kv4_gather_blocks — blocks of both pools as dense ones: out[b, j] = values of block
 * block_ids[b * id_stride + j], rounded to dtype (fp16 by way of fp32); k_out/v_out contiguous
 * [batch, blocks_per_row, block_size, num_kv_heads, head_dim], the layout of a dense pool of
 * batch * blocks_per_row blocks.  With lengths (NULL: all), row b's tokens at and past lengths[b] are
 * written as zeros, whatever the pages hold there, and the ids of blocks wholly past it are not read;
 * with fill_past == 0 those blocks are not written either (the attention reads none of them).  A block
 * id out of range reads as zeros and sets MI_STATUS_BAD_BLOCK.
 */
int mi_kv4_gather_blocks(const void* k_pool, const void* v_pool, const int64_t* block_ids, int64_t id_stride,
                         const int64_t* lengths, int fill_past, int64_t batch, int64_t blocks_per_row, void* k_out,
                         void* v_out, int64_t num_blocks, int block_size, int num_kv_heads, int head_dim, int dtype,
                         void* stream);

/*
 * mi_kv4_qk_norm_rope — mi_qk_norm_rope (mi_layers.h) whose decode append goes to 4-bit pools: roped K and V,
 * rounded to dtype, are quantised into the pages at slot_mapping, the bytes that mi_kv4_scatter of k_out and
 * v_out would leave there.  head_dim in {32, 64, 128, 256}.
 */
int mi_kv4_qk_norm_rope(const void* q, int64_t q_row_stride, const void* k, int64_t k_row_stride, const void* v,
                        int64_t v_row_stride, const void* q_weight, const void* k_weight, const void* cos,
                        const void* sin, int64_t cos_sin_row_stride, int64_t tokens, int hq, int hkv, int head_dim,
                        float eps, void* q_out, void* k_out, void* v_out, const int64_t* slot_mapping, void* k_pool,
                        void* v_pool, int64_t num_blocks, int block_size, int dtype, void* stream);

/*
 * mi_kv4_paged_decode — mi_paged_decode over 4-bit pools: one query token per sequence attends to
 * positions [0, context_lens[b]) of its block table; arguments as there.  With k_new, v_new,
 * new_strides and slot_mapping the new tokens are quantised into the pools first.  A row with
 * context length 0 gets zeros.  A table row covers at most 2^31 - 1 tokens (MI_ERR_UNSUPPORTED).  What
 * the pages hold past a context length is never used.  A block id
 * out of range reads the null block and sets MI_STATUS_BAD_BLOCK.  Softmax, sums and accumulators
 * are fp32.
 */
size_t mi_kv4_paged_decode_workspace_size(int64_t batch, int num_q_heads, int num_kv_heads, int head_dim,
                                          int64_t max_blocks_per_seq, int block_size, int dtype);
int mi_kv4_paged_decode(const void* q, const int64_t* q_strides, const void* k_new, const void* v_new,
                        const int64_t* new_strides, const int64_t* slot_mapping, void* k_pool, void* v_pool,
                        int64_t num_blocks, int block_size, int num_kv_heads, int head_dim,
                        const int64_t* block_tables, int64_t table_stride, int64_t max_blocks_per_seq,
                        const int64_t* context_lens, int64_t batch, int num_q_heads, float scale, void* out,
                        int64_t out_stride, void* workspace, size_t workspace_bytes, int dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MI_KV4_H */
