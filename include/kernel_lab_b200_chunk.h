/*
 * kernel_lab_b200_chunk.h -- C ABI of the chunked step over a paged KV cache: chunks of new tokens
 * appended to the cache, attention of those tokens over it, and the cache's pages themselves (copied,
 * given to growing and forked sequences, compacted). Same library, conventions and status codes as
 * kernel_lab_b200.h: device pointers as `void*`, the stream as `void*`, 0 or a `cudaError_t` as the
 * result, nothing thrown, work enqueued on the stream without a host synchronisation or an allocation.
 *
 * A chunk: sequence b's new tokens are the rows indptr[b] to indptr[b + 1] - 1 of a tensor of `tokens`
 * rows (indptr: [batch + 1] int32, ascending, within [0, tokens]). Rows of no sequence are neither read nor
 * written.
 */
#ifndef KERNEL_LAB_B200_CHUNK_H_
#define KERNEL_LAB_B200_CHUNK_H_

#include <stddef.h>
#include <stdint.h>

#include "kernel_lab_b200.h"
#include "kernel_lab_b200_block8.h"

#ifdef __cplusplus
extern "C" {
#endif

/* code_type of a cache that holds q's own dtype (beside KL_CODE_E4M3 and KL_CODE_INT8). */
enum { KL_CODE_NONE = -1 };

/* Status bit beside those of kernel_lab_b200.h: kl_paged_reserve had too few free pages. */
enum { KL_STATUS_NO_PAGES = 32 };

/*
 * kl_paged_kv_append for chunks: row indptr[b] + i of k_new / v_new ([tokens][num_kv_heads * head_dim], rows
 * new_row_stride elements apart) goes to token position positions[b] + i of sequence b. A negative
 * positions[b] skips the sequence; a position past max_pages_per_seq * page_size or a page id outside
 * [0, num_pages) skips the row and ORs KL_STATUS_BAD_PAGE into *status (if non-null). Caches are contiguous
 * [num_pages, page_size, num_kv_heads, head_dim] of `dtype`. Sequences must not write the same slot in one call.
 */
int kl_paged_kv_append_chunks(int dtype, void* k_cache, void* v_cache, const void* k_new, const void* v_new,
                              const int32_t* block_table, const int32_t* positions, const int32_t* indptr, int batch,
                              int64_t tokens, int num_kv_heads, int head_dim, int page_size,
                              int64_t block_table_stride, int max_pages_per_seq, int64_t num_pages,
                              int64_t new_row_stride, uint32_t* status, void* stream);

/* The same into an e4m3 cache with a scale for each KV head: e4m3(x / scale[h]), as kl_paged_kv_append_fp8.
 * head_dim is even. */
int kl_paged_kv_append_chunks_fp8(int dtype, void* k_cache, void* v_cache, const void* k_new, const void* v_new,
                                  const float* k_scale, const float* v_scale, const int32_t* block_table,
                                  const int32_t* positions, const int32_t* indptr, int batch, int64_t tokens,
                                  int num_kv_heads, int head_dim, int page_size, int64_t block_table_stride,
                                  int max_pages_per_seq, int64_t num_pages, int64_t new_row_stride, uint32_t* status,
                                  void* stream);

/*
 * Attention of chunks of new tokens over a paged cache. Sequence b holds seq_lens[b] tokens, the n =
 * indptr[b + 1] - indptr[b] new ones last (already appended). For new token i and query head h with KV head g,
 *   out[indptr[b] + i, h] = sum_j p_j V_j,  p = softmax over j of scale * q[indptr[b] + i, h] . K_j,
 * over the tokens j < seq_lens[b], with `causal` non-zero only those up to its own position:
 * j <= seq_lens[b] - n + i. A token that has none to attend to (seq_lens[b] < n - i) gets zeros. What is
 * masked does not count, whatever it holds (infinities and NaN included).
 *
 *   q     [tokens, num_q_heads, head_dim] of `dtype`, rows q_row_stride elements apart, a row contiguous
 *   out   [tokens, num_q_heads, head_dim], contiguous; rows of no sequence are left as they were
 *   caches  logically [num_pages, page_size, num_kv_heads, head_dim]: page, token and head are page_stride,
 *         token_stride and head_stride elements apart, head_dim is contiguous; both have the same strides
 *   code_type KL_CODE_NONE: elements of `dtype`, no scales (k_scale and v_scale NULL). KL_CODE_E4M3 or
 *         KL_CODE_INT8: element = code * scale[page * scale_page_stride + h], fp32; scale_page_stride 0 is a
 *         scale for each KV head, num_kv_heads one for each page and KV head; q is fp16 or bf16
 * Lengths beyond max_pages_per_seq * page_size are clamped (KL_STATUS_LEN_CLAMPED); pages whose id is outside
 * [0, num_pages) are skipped (KL_STATUS_BAD_PAGE). head_dim is at most 256, num_pages at least 1, batch at most
 * 65535, tokens and max_pages_per_seq * page_size at most 2^31 - 257.
 *
 * Arithmetic: products accumulate in fp32, the softmax is in fp32 (exponentials off by up to 1.1e-4 of themselves for bf16
 * over 16-bit caches, 4e-6 otherwise). fp16 and bf16: a probability, over 8-bit caches one times its value scale (codes enter
 * the products exactly), is rounded to q's dtype: bf16 to 2^-8 of itself, fp16 to 2^-11 where it is at least 2^-21 of
 * its row's largest, by up to 2^-32 of that below.
 *
 * Scratch from kl_paged_chunk_attention_workspace_size, under kl_paged_decode's rules (`sync` zero before its
 * first use, left zero but for the status word; calls that overlap on the GPU need separate buffers); partials start at a
 * multiple of 32 bytes, sync at one of 4. After KL_STATUS_WAIT_TIMEOUT the output is invalid and `sync` has to be zeroed
 * again. fp16 and bf16 with head_dim a multiple of 8 (of 16 over 8-bit caches), groups of up to 128 query heads, pages of a
 * multiple of 8 tokens, a positive scale and 16-byte aligned rows run on the tensor cores; everything else runs on the
 * CUDA cores.
 */
int kl_paged_chunk_attention_workspace_size(int dtype, int code_type, int64_t tokens, int batch, int num_q_heads,
                                            int num_kv_heads, int head_dim, size_t* partial_bytes,
                                            size_t* sync_bytes);

int kl_paged_chunk_attention(int dtype, int code_type, void* out, const void* q, const void* k_cache,
                             const void* v_cache, const float* k_scale, const float* v_scale,
                             const int32_t* block_table, const int32_t* seq_lens, const int32_t* indptr, int batch,
                             int64_t tokens, int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                             int64_t q_row_stride, int64_t page_stride, int64_t token_stride, int64_t head_stride,
                             int64_t scale_page_stride, int64_t block_table_stride, int max_pages_per_seq,
                             int64_t num_pages, int causal, float scale, void* partials, size_t partial_bytes,
                             void* sync, size_t sync_bytes, void* stream);

/*
 * Pools: tensors whose first dimension is the page. Tensor t's page p is the bytes[t] bytes at
 * base[t] + p * stride[t]; all of them have num_pages pages. The arrays are host arrays, read during the call.
 */
typedef struct {
  int count;
  void* const* base;
  const int64_t* stride;
  const int64_t* bytes;
} kl_page_pools_t;

/*
 * Copies page src[i] to page dst[i] in every tensor, i < pairs (src, dst: device int32). A negative src or dst
 * skips the pair; ids of num_pages and more skip it too and OR KL_STATUS_BAD_PAGE into *status (if non-null).
 * No page may be the destination of two pairs, or of one and the source of another: what such a page holds
 * afterwards is unspecified.
 */
int kl_paged_copy_pages(const kl_page_pools_t* pools, const int32_t* src, const int32_t* dst, int64_t pairs,
                        int64_t num_pages, uint32_t* status, void* stream);

/*
 * Pages for the tokens to come, and forks. Row r of the new table stands for sequence parents[r] of the old one
 * (parents NULL: r itself, rows == batch; negative: an empty row), whose first ceil(len / page_size) entries it
 * takes over: rows with one parent share its pages. Sequences that no row stands for are dropped. A page is in
 * use if one of those entries names it, and free otherwise, so that no counts are kept and dropping or
 * shortening a sequence frees its pages; every holder of pages has to be a row.
 * Each row then gets, in the order of the rows, the free pages with the lowest ids:
 *   a copy of its last page, if that is partly filled, the row is to write (new_tokens[r] > 0) and another
 *   entry names it too (of several rows that are to write to it and are its only holders, the lowest keeps
 *   it): the page's contents are copied in every tensor;
 *   then pages for the tokens len .. len + new_tokens[r] - 1 that its last page has no room for.
 * A row whose new tokens do not fit in the table's width, or for whose needs and those of the rows before it
 * the free pages do not suffice, gets none (KL_STATUS_NO_PAGES); a row that needs none is always served.
 *   out_table  [rows, width] int32, contiguous: entries past a row's pages are 0, which is a page like any other:
 *              nothing may be appended for a row that was not served or is empty
 *   out_lens   [rows] int32: seq_lens[parents[r]] (new tokens not counted)
 *   served     [rows] bytes: 1, or 0 for a row that got none of what it needs
 * No output overlaps an input or another output, but that out_lens may be seq_lens where parents is NULL.
 * Lengths beyond width * page_size are clamped (KL_STATUS_LEN_CLAMPED). Entries outside [0, num_pages) are taken over
 * but stand for no page (KL_STATUS_BAD_PAGE). Parents past the batch make empty rows as negative ones do; they are not
 * reported. An empty row has length 0, needs nothing and is served. Negative new_tokens count as 0. rows at most 2^24.
 * Scratch from kl_paged_reserve_workspace_size, under kl_paged_decode's rules (`sync` zero before its first use, left zero
 * but for the status word; calls that overlap on the GPU need separate buffers); both start at a multiple of 16 bytes. A
 * call launches several kernels that hand data on through the scratch: nothing else that uses these buffers may be put on
 * the stream, by another host thread for instance, until it has returned.
 */
int kl_paged_reserve_workspace_size(int64_t num_pages, int rows, size_t* scratch_bytes, size_t* sync_bytes);

int kl_paged_reserve(const kl_page_pools_t* pools, int32_t* out_table, int32_t* out_lens, uint8_t* served,
                     const int32_t* block_table, const int32_t* seq_lens, const int32_t* new_tokens,
                     const int32_t* parents, int batch, int rows, int width, int page_size,
                     int64_t block_table_stride, int64_t num_pages, void* scratch, size_t scratch_bytes,
                     void* sync, size_t sync_bytes, void* stream);

/*
 * Moves the pages in use (those that the first ceil(seq_lens[b] / page_size) entries of the rows name; *used
 * of them) to the ids 0 .. *used - 1: the ones with ids of *used and more, in ascending order, to the free ids
 * below, in ascending order, in every tensor. out_table ([batch, width] int32, contiguous) receives the entries
 * under the pages' new ids, 0 past a row's pages. Entries outside [0, num_pages) are taken over (KL_STATUS_BAD_PAGE),
 * lengths clamped as above. Neither output overlaps an input or the other. Scratch as above.
 */
int kl_paged_compact_workspace_size(int64_t num_pages, size_t* scratch_bytes, size_t* sync_bytes);

int kl_paged_compact(const kl_page_pools_t* pools, int32_t* out_table, int32_t* used, const int32_t* block_table,
                     const int32_t* seq_lens, int batch, int width, int page_size, int64_t block_table_stride,
                     int64_t num_pages, void* scratch, size_t scratch_bytes, void* sync, size_t sync_bytes,
                     void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KERNEL_LAB_B200_CHUNK_H_ */
