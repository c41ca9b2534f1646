/*
 * ecq_kv4.h -- a paged KV cache held in 4 bits: the block tables and slot maps
 * of a serving step built on the device, K and V rows stored and read back,
 * and attention over the cache (no counterpart in the reference, which has no
 * model runtime; its weight form `symbol * scale + zero` per group,
 * src/quantizer.py:33-35, is the cache's value form).
 *
 * Every launch takes a cudaStream_t (as void*), allocates nothing, never
 * synchronises the host and returns 0 or a negative ECQ_ERR_*. Bad values that
 * only the device sees (page numbers, slots, lengths) are skipped and OR a
 * ECQ_STATUS_* bit into *status (int32, device memory; may be NULL).
 *
 * Pool. uint8 [n_pages][kv_heads][page bytes], 16-byte aligned; page_size is
 * 16, 32, 64, 128 or 256 tokens, head_dim D 64 or 128, group_size g 32, 64 or
 * 128 (at most D). A page of one head is page_size / 16 blocks of 16 tokens:
 *   K codes   [16][D / 2 bytes]
 *   V codes   [16][D / 2 bytes]
 *   K params  [16][D / g] pairs (scale, zero) of fp16
 *   V params  [16][D / g] pairs (scale, zero) of fp16
 * that is 16 D + 128 D / g bytes. The value of a channel is code * scale + zero.
 * Nibbles go low first. Nibble n of a K row is channel 32 w + 8 t + i, where n
 * counts (t, w, i) over [4][D / 32][8]; nibble n of a V row is channel 8 s + r,
 * where n counts (r, s) over [8][D / 8]: the order in which the attention
 * kernel's lanes take them. A token's slot is page * page_size + its place in
 * the page (int32, so n_pages * page_size < 2^31).
 *
 * Stored values: x is clamped to +-65504; zero = fp16(min of the group), scale
 * = fp16((max - min) / 15), code = (x - zero) / scale rounded to nearest even
 * and clamped to 0..15 (0 where scale is 0). A NaN makes its group's scale and
 * zero NaN. The scale may be rounded up, so that code 15 stands for a little more
 * than the group's maximum, 65584 at most: read back in fp16 a value of 65520 or
 * more is infinite.
 */
#ifndef ECQ_KV4_H
#define ECQ_KV4_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ECQ_KV4_F16 0
#define ECQ_KV4_BF16 1
#define ECQ_STATUS_NO_PAGES 8u /* the free stack (or its room) does not suffice */
#define ECQ_KV4_MAX_BATCH 8192

/* Bytes of one page of one head; negative for sizes without a kernel. */
int64_t ecq_kv4_page_bytes(int32_t head_dim, int32_t page_size, int32_t group_size);

/* One serving step's bookkeeping: request b of `batch` (at most
 * ECQ_KV4_MAX_BATCH) grows from seq_lens[b] tokens by new_lens[b] (>= 0).
 *   seq_lens_out[b] = seq_lens[b] + new_lens[b]
 *   block_table[b][j] (row stride table_stride, max_pages columns) gets a page
 *     for every j the longer request needs and the shorter one did not; pages
 *     are popped off the end of free_pages[0 .. *free_count) in the order of
 *     requests and columns. Other entries stay.
 *   q_starts[batch + 1] = exclusive sums of new_lens
 *   slots[i], positions[i] for token i < q_starts[batch]: its slot in the pool
 *     and its position in its request; -1 for q_starts[batch] <= i < max_tokens
 *   *free_count_out = what is left on the stack
 * seq_lens_out may be seq_lens and free_count_out free_count; no other pair may
 * overlap (refused, for these two). All or nothing: where a length is negative or too long for its table
 * row, the new tokens are more than max_tokens, a page that would be popped or
 * that a request goes on in is negative or has slots of 2^31 and more
 * (ECQ_STATUS_BADARG) or the pages do not suffice (ECQ_STATUS_NO_PAGES),
 * lengths, count and table stay as they were, q_starts is all 0 and slots and
 * positions all -1. */
int32_t ecq_kv4_extend(const void *seq_lens, const void *new_lens, void *seq_lens_out, void *block_table,
                       int64_t table_stride, int32_t max_pages, int32_t batch, int32_t page_size,
                       const void *free_pages, int32_t free_capacity, const void *free_count, void *free_count_out,
                       void *q_starts, void *slots, void *positions, int32_t max_tokens, void *status, void *stream);

/* Gives the pages of the requests with done[b] != 0 (uint8) back: pushed on
 * free_pages in the order of requests and columns, their lengths set to 0. The
 * table's entries stay (a length of 0 makes them unused). All or nothing as
 * above, bad pages among those to be pushed included; ECQ_STATUS_NO_PAGES where
 * the stack (free_capacity) has no room. What lies behind the stack's end may be
 * overwritten in any case. */
int32_t ecq_kv4_release(const void *done, const void *seq_lens, void *seq_lens_out, const void *block_table,
                        int64_t table_stride, int32_t max_pages, int32_t batch, int32_t page_size, void *free_pages,
                        int32_t free_capacity, const void *free_count, void *free_count_out, void *status,
                        void *stream);

/* Stores rows k[t][h], v[t][h] (head_dim contiguous elements of dtype; strides
 * in elements, multiples of 8; 16-byte aligned) at slots[t], t < tokens. A
 * negative slot stores nothing; one beyond the pool sets ECQ_STATUS_BADARG.
 * Slots of one call must differ: of two rows for one slot either's parts may
 * stay. */
int32_t ecq_kv4_append(const void *k, int64_t k_token_stride, int64_t k_head_stride, const void *v,
                       int64_t v_token_stride, int64_t v_head_stride, int32_t dtype, void *pages, int64_t n_pages,
                       int32_t kv_heads, int32_t head_dim, int32_t page_size, int32_t group_size, const void *slots,
                       int32_t tokens, void *status, void *stream);

/* Reads rows back: k, v [tokens][kv_heads][head_dim] = code * scale + zero,
 * rounded once to dtype; zeros for a negative or bad slot. */
int32_t ecq_kv4_gather(void *k, void *v, int32_t dtype, const void *pages, int64_t n_pages, int32_t kv_heads,
                       int32_t head_dim, int32_t page_size, int32_t group_size, const void *slots, int32_t tokens,
                       void *status, void *stream);

/* Attention of new tokens over the cache that already holds them. Request b
 * has queries q_starts[b] .. q_starts[b + 1] - 1 (at most max_q; q_starts NULL:
 * query b is request b's one), the last of its seq_lens[b] tokens: query i of n
 * sees keys 0 .. seq_lens[b] - n + i. Query head h reads cache head
 * h / (heads / kv_heads). out = softmax(q . k * scale) v, zeros where a query
 * sees no key; rows of out at or behind q_starts[batch] are not written. q and
 * out: [total_q][heads][head_dim] of dtype, strides in elements, head_dim
 * contiguous, q 16-byte aligned with strides that are multiples of 8, out
 * 8-byte aligned with multiples of 4. heads / kv_heads is at most 64. A page
 * number outside the pool, or a length below 0 or beyond the table's row, sets
 * ECQ_STATUS_BADARG and its keys are left out. The same status says that a
 * request had more than max_q queries and some of its rows were not written.
 * For requests with many rows K and V are rounded to fp16, and values past its
 * end (65520 to 65584 as ecq_kv4_append stores them) count as +-65504.
 * workspace:
 * ecq_kv4_attention_workspace_bytes, its content does not matter; calls that
 * may overlap need one each. */
int64_t ecq_kv4_attention_workspace_bytes(int32_t batch, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                          int32_t max_q, int32_t max_pages, int32_t page_size);
int32_t ecq_kv4_attention(const void *q, int64_t q_token_stride, int64_t q_head_stride, void *out,
                          int64_t out_token_stride, int64_t out_head_stride, int32_t dtype, const void *pages,
                          int64_t n_pages, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t page_size,
                          int32_t group_size, const void *block_table, int64_t table_stride, int32_t max_pages,
                          const void *seq_lens, const void *q_starts, int32_t batch, int32_t total_q, int32_t max_q,
                          float scale, void *workspace, int64_t workspace_bytes, void *status, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* ECQ_KV4_H */
