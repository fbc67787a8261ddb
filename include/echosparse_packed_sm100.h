/* C ABI of libechosparse_sm100.so (B200, sm_100a) for attention over packed sequences and over a paged cache of keys and values.
 *
 * Conventions (all entry points):
 *   - plain device pointers and sizes; the caller allocates every buffer; `stream` is a cudaStream_t; nothing synchronises;
 *   - return 0 on success, a negative code on a rejected call or a failed launch; es_last_error() gives the text;
 *   - D = 64 or 128, dtype 0 = bf16, 1 = fp16; heads is a multiple of kv_heads, query head h reads key head h / (heads / kv_heads);
 *   - strides are in elements, multiples of 8; the last dimension is contiguous; pointers are 16-byte aligned (workspaces, and the outputs
 *     of the packed operators, 32-byte; lse and int32 arrays 4-byte);
 *   - scale, the factor of the logits, is from 2^-126 to 2^126;
 *   - lse is the natural-log LSE in fp32, -inf for rows without a key, whose output is 0;
 *   - every wait inside the kernels is bounded; outputs of a tile whose wait gave up are NaN, and so is what later calls of the
 *     device return until es_device_status (echosparse_sm100.h) has read and cleared the word.
 *
 * Packed sequences: the tokens of all sequences lie behind one another, [tokens, heads, D]; cu [batch + 1] int32 (not decreasing)
 * gives the first token of each sequence and the end of the last. Values outside 0 .. tokens are clamped. Rows of no sequence get output
 * 0, LSE -inf and gradient 0.
 */
#ifndef ECHOSPARSE_PACKED_SM100_H
#define ECHOSPARSE_PACKED_SM100_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Attention of every sequence of a packed batch to its own keys. q [total_q, heads, D], k, v [total_k, kv_heads, D] with a token and a
 * head stride each; o [total_q, heads, D] contiguous, lse [heads, total_q]; o_rest (like o, or NULL) receives what rounding o left, for
 * the backward. Sequence b has queries cu_q[b] .. cu_q[b + 1] and keys cu_k[b] ..
 * cu_k[b + 1]; with causal, query i of nq sees key j of nk where j <= i + nk - nq. workspace: es_packed_fwd_workspace_bytes bytes,
 * may be NULL where that is 0. */
long long es_packed_fwd_workspace_bytes(int32_t batch, int32_t total_q, int32_t total_k, int32_t heads, int32_t kv_heads, int32_t D);
int es_packed_attn_fwd(const void* q, const void* k, const void* v, void* o, void* o_rest, float* lse, const int32_t* cu_q,
                       const int32_t* cu_k, int32_t batch, int32_t total_q, int32_t total_k, int32_t heads, int32_t kv_heads, int32_t D, int64_t q_token,
                       int64_t q_head, int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head, float scale, int32_t causal,
                       int32_t dtype, void* workspace, void* stream);

/* The backward of es_packed_attn_fwd: dq [total_q, heads, D] and dk, dv [total_k, kv_heads, D] contiguous, dk and dv summed over the query heads
 * of the key's group. o and o_rest (or NULL) are the forward's, dout has a token and a head stride. dq, or dk and dv, may be NULL. One owner per row and no
 * atomics: the same inputs give the same bits. workspace: es_packed_bwd_workspace_bytes bytes. */
long long es_packed_bwd_workspace_bytes(int32_t batch, int32_t total_q, int32_t total_k, int32_t heads, int32_t kv_heads, int32_t D);
int es_packed_attn_bwd(const void* q, const void* k, const void* v, const void* o, const void* o_rest, const void* dout, const float* lse,
                       void* dq, void* dk, void* dv, const int32_t* cu_q, const int32_t* cu_k, int32_t batch, int32_t total_q, int32_t total_k,
                       int32_t heads, int32_t kv_heads, int32_t D, int64_t q_token, int64_t q_head, int64_t k_token, int64_t k_head,
                       int64_t v_token, int64_t v_head, int64_t do_token, int64_t do_head, float scale, int32_t causal, int32_t dtype,
                       void* workspace, void* stream);

/* Attention of the newest `tokens` queries of each request to a shared prefix and to the request's own tokens, both in pages of a cache
 * k_cache, v_cache [pages, page_size, kv_heads, D] (page, token and head strides). q, o [batch, tokens, heads, D] contiguous, lse
 * [batch, heads, tokens]. prefix_pages [n_prefix_pages]: the pages of the prefix, of which the first prefix_len tokens count; table
 * [batch, table_width]: the pages of each request's own tokens, of which lengths[b] count, the queries' own keys the last of them: query i
 * sees the whole prefix and own tokens 0 .. lengths[b] - tokens + i. Keys in pages outside 0 .. pages - 1 are not attended to.
 * page_size 16, 32, 64, 128 or 256; at most 2^23 requests. workspace: es_prefix_workspace_bytes bytes, may be NULL where that is 0. */
long long es_prefix_workspace_bytes(int32_t batch, int32_t tokens, int32_t heads, int32_t kv_heads, int32_t D, int32_t prefix_len,
                                    int32_t table_width, int32_t page_size);
int es_prefix_attn(const void* q, const void* k_cache, const void* v_cache, void* o, float* lse, const int32_t* prefix_pages,
                   int32_t n_prefix_pages, int32_t prefix_len, const int32_t* table, int32_t table_width, const int32_t* lengths,
                   int32_t batch, int32_t tokens, int32_t heads, int32_t kv_heads, int32_t D, int32_t pages, int32_t page_size,
                   int64_t k_page, int64_t k_token, int64_t k_head, int64_t v_page, int64_t v_token, int64_t v_head, float scale,
                   int32_t dtype, void* workspace, void* stream);

/* Pages and slots of the next tokens of a batch of requests. lengths [batch]: tokens that request b holds (in the first
 * ceil(lengths[b] / page_size) pages of its row of table [batch, table_width]); new_tokens [batch]: tokens it gets. The pages that are missing
 * are taken from free_pages [n_free] in order, request by request, and written into the rows. Written: slots, positions [total]: slot (page *
 * page_size + offset) and position in its request of every new token, the tokens of request b at cu_new[b] .. cu_new[b + 1], slot and position
 * -1 behind the last; cu_new [batch + 1]; lengths_out [batch]; taken [2] = pages taken, pages that were needed but not there. Tokens for which
 * the free list or the row has no page get slot -1 and do not count in lengths_out, and the row's entry is -1. */
int es_extend_tables(const int32_t* lengths, const int32_t* new_tokens, int32_t* table, const int32_t* free_pages, int32_t n_free,
                     int32_t batch, int32_t table_width, int32_t page_size, int32_t total, int32_t* slots, int32_t* positions,
                     int32_t* cu_new, int32_t* lengths_out, int32_t* taken, void* stream);

/* k_cache[slot], v_cache[slot] = k[t], v[t] with slot = slots[t], for every token t whose slot lies in the cache (0 .. pages * page_size - 1);
 * the others are skipped. Of two tokens with the same slot either may be stored. k, v [total, kv_heads, D] with strides. */
int es_store_kv(const void* k, const void* v, void* k_cache, void* v_cache, const int32_t* slots, int32_t total, int32_t kv_heads,
                int32_t D, int32_t pages, int32_t page_size, int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head,
                int64_t kc_page, int64_t kc_token, int64_t kc_head, int64_t vc_page, int64_t vc_token, int64_t vc_head, void* stream);

#ifdef __cplusplus
}
#endif
#endif
