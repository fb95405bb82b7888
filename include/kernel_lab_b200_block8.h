/*
 * kernel_lab_b200_block8.h -- C ABI of the 8-bit serving step: RMSNorm with an e4m3 output, and a
 * paged KV cache held in 8 bits with one scale for each page and KV head (append, decode attention,
 * selection of pages). Same library, conventions and status codes as kernel_lab_b200.h: device
 * pointers as `void*`, the stream as `void*`, 0 or a `cudaError_t` as the result, nothing thrown,
 * work enqueued on the stream without a host synchronisation or an allocation.
 *
 * The block-scaled cache:
 *   k_cache, v_cache   codes, one byte an element, logically [num_pages, page_size, num_kv_heads,
 *                      head_dim]: page, token and head are page_stride, token_stride and
 *                      head_stride bytes apart (any order of the three), head_dim is contiguous;
 *                      both tensors have the same strides
 *   code_type          KL_CODE_E4M3 or KL_CODE_INT8
 *   k_scale, v_scale   [num_pages, num_kv_heads] fp32, contiguous: element = code * scale
 *   k_bounds           [num_pages, num_kv_heads, 2, head_dim] int8, contiguous: per channel the
 *                      least (0) and largest (1) key code of the page's tokens, rounded outward to
 *                      whole units of 1 (int8) or 4 (e4m3) codes, so that
 *                      bounds * unit * k_scale encloses the page's keys
 */
#ifndef KERNEL_LAB_B200_BLOCK8_H_
#define KERNEL_LAB_B200_BLOCK8_H_

#include <stddef.h>
#include <stdint.h>

#include "kernel_lab_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

enum {
  KL_CODE_E4M3 = 0,
  KL_CODE_INT8 = 1
};

/*
 * RMSNorm over rows of length `hidden` with an e4m3 output. With `residual` (and residual_out, which
 * may be the same pointer): residual_out <- dtype(x + residual), bit-exact, and r = residual_out;
 * without (both NULL): r = x. Then, in fp32, y = r * rsqrt(mean(r^2) + eps) * weight, and for each
 * group of group_size columns (0: the whole row; the last group may be short)
 *   a = max |y|, scale = a / 448, code = e4m3(y * 448 / a) (nearest-even, saturating; NaN stays NaN),
 * or scale = 0 and codes of 0 where a or max |r * weight| is below 2^-100. The codes are formed from
 * r * weight, whose magnitude has to stay below 2^126.
 *   codes   [rows, hidden] bytes            scales   [rows, ceil(hidden / group_size)] fp32
 * x rows are x_row_stride elements apart; the other tensors are contiguous. rows == 0 is a no-op.
 */
int kl_rms_norm_fp8(int dtype, void* codes, float* scales, void* residual_out, const void* x, const void* residual,
                    const void* weight, int rows, int hidden, int64_t x_row_stride, int group_size, float eps,
                    void* stream);

/*
 * Append new tokens to a block-scaled cache. Sequence b's new tokens are rows indptr[b] to
 * indptr[b + 1] - 1 of k_new / v_new ([tokens][num_kv_heads * head_dim] of `dtype`, rows
 * new_row_stride elements apart) and take the token positions positions[b], positions[b] + 1, ...;
 * with indptr NULL each sequence has one (tokens == batch). A negative position skips the sequence.
 * Position p goes to page block_table[b, p / page_size], slot p % page_size.
 *
 * For each touched page, KV head and tensor, with a = the largest finite magnitude of its new elements:
 *   need  = int8: max(fl(a * fl(1 / 127)), 2^-126); e4m3: the least power of two 2^k, k >= -126, with
 *           a <= 448 * 2^k (so that a later growth rescales codes exactly); 0 if a is 0
 *   scale = max(need, the page's present scale if slots before the first new one are in use, else 0)
 *   new codes  = Q(x * (1 / scale)); if the scale grew, the codes in the slots before the first new
 *   one become Q(code * (old / scale)). Q rounds to nearest even and saturates at 448 or 127; NaN
 *   stays NaN in e4m3 and becomes 0 in int8. A scale below 2^-126 gives codes 0.
 * Slots after the last new one are left alone. k_bounds (may be NULL) is rewritten for every touched
 * page from its slots up to the last new one, NaN counting as 0.
 *
 * Sequences must not append to the same page in one call. A position past max_pages_per_seq *
 * page_size or a page id outside [0, num_pages) skips that page's tokens and ORs KL_STATUS_BAD_PAGE
 * into *status (if non-null); rows outside every [indptr[b], indptr[b + 1]) are skipped. head_dim is at
 * most 1024.
 */
int kl_paged_kv_append_block8(int dtype, int code_type, void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                              void* k_bounds, const void* k_new, const void* v_new, const int32_t* block_table,
                              const int32_t* positions, const int32_t* indptr, int batch, int64_t tokens,
                              int num_kv_heads, int head_dim, int page_size, int64_t page_stride,
                              int64_t token_stride, int64_t head_stride, int64_t block_table_stride,
                              int max_pages_per_seq, int64_t num_pages, int64_t new_row_stride, uint32_t* status,
                              void* stream);

/*
 * Single-token decode attention over a block-scaled cache: with K = code * k_scale[page, h] and
 * V = code * v_scale[page, h],  out[b, h] = softmax(scale * q[b, h] . K_b^T) V_b.
 * selected NULL: over the first seq_lens[b] tokens. Otherwise `selected` is [batch, num_kv_heads,
 * num_selected] int32, contiguous: for KV head h of sequence b only the tokens of the pages in columns
 * selected[b, h, :] of its block-table row are attended to (each column at most once; entries outside
 * [0, ceil(seq_lens[b] / page_size)) select nothing), the last page up to seq_lens[b]. An entry that selects nothing
 * still takes the time of a page without reading one.
 * A row with nothing to attend to gives zeros. Lengths beyond max_pages_per_seq * page_size are
 * clamped (KL_STATUS_LEN_CLAMPED); page ids outside [0, num_pages) are skipped (KL_STATUS_BAD_PAGE).
 *
 * q and out are fp16 or bf16 ([batch, num_q_heads, head_dim], 16-byte aligned); head_dim is a
 * multiple of 16 up to 256; page_size is 8 or a multiple of 16; the caches and their strides are
 * 16-byte aligned, the strides below 2^31; at most 128 query heads a KV head (64 for head_dim above 128). Others return
 * cudaErrorInvalidValue. The products run in fp16 (codes exactly; an fp16 q as it is; a bf16 q scaled by a
 * power of two, exact for elements down to 2^-31 of their head's largest, others off by at most 2^-39 of it)
 * and accumulate in fp32. A token's probability times its value scale is rounded to fp16: it is off by at
 * most 2^-11 of itself or 2^-25 of the query head's largest such product, whatever the scales of the other pages.
 *
 * Scratch: kl_paged_decode_block8_workspace_size with the same arguments (num_selected 0 without a
 * selection), under kl_paged_decode's rules (`sync` zero before its first use, left zero).
 */
int kl_paged_decode_block8_workspace_size(int batch, int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                                          int max_pages_per_seq, int num_selected, size_t* partial_bytes,
                                          size_t* sync_bytes);

int kl_paged_decode_block8(int dtype, int code_type, void* out, const void* q, const void* k_cache,
                           const void* v_cache, const float* k_scale, const float* v_scale,
                           const int32_t* block_table, const int32_t* seq_lens, const int32_t* selected, int batch,
                           int num_q_heads, int num_kv_heads, int head_dim, int page_size, int64_t page_stride,
                           int64_t token_stride, int64_t head_stride, int64_t block_table_stride,
                           int max_pages_per_seq, int64_t num_pages, int num_selected, float scale, void* partials,
                           size_t partial_bytes, void* sync, size_t sync_bytes, void* stream);

/*
 * Pages that a decode step should read, per sequence and KV head, by an upper bound of q . k over each
 * page's keys: with a query head's q rounded to int8 (sq = fl(max|q| * fl(1 / 127)), qi = round(q * fl(1 / sq))),
 *   I(page) = sum_d max(qi[d] * lo[d], qi[d] * hi[d])                       (k_bounds; whole numbers)
 *   score(page) = max over the KV head's query heads of fl(I * sq), times fl(unit * k_scale[page, h])
 * The first sink_pages and the last recent_pages pages always come first; then the largest scores;
 * ties go to the lower column. selected [batch, num_kv_heads, num_selected] int32 receives the
 * min(num_selected, pages in use) block-table columns in ascending order, then -1. I is exact, so the
 * choice depends on no order of summation. Infinities count as the largest code, NaN as 0.
 * num_selected >= sink_pages + recent_pages; head_dim a multiple of 16 up to 256; q fp32, fp16 or bf16; num_pages
 * at least 1.
 * Scratch from kl_paged_block_select_workspace_size, under kl_paged_decode's rules.
 */
int kl_paged_block_select_workspace_size(int batch, int num_kv_heads, int max_pages_per_seq, size_t* scratch_bytes,
                                         size_t* sync_bytes);

int kl_paged_block_select(int dtype, int code_type, int32_t* selected, const void* q, const void* k_bounds,
                          const float* k_scale, const int32_t* block_table, const int32_t* seq_lens, int batch,
                          int num_q_heads, int num_kv_heads, int head_dim, int page_size, int64_t block_table_stride,
                          int max_pages_per_seq, int64_t num_pages, int num_selected, int sink_pages,
                          int recent_pages, void* scratch, size_t scratch_bytes, void* sync, size_t sync_bytes,
                          void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KERNEL_LAB_B200_BLOCK8_H_ */
