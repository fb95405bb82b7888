// What the chunk-attention kernels share: the call's arguments and a sequence's rows and keys.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"
#include "kernel_lab_b200.h"
#include "kernel_lab_b200_chunk.h"

namespace klb {
namespace chunk_attention {

struct Args {
  void* out;
  const void* q;
  const void* k;
  const void* v;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_table;
  const int32_t* seq_lens;
  const int32_t* indptr;
  int64_t tokens;
  int64_t q_stride, page_stride, token_stride, head_stride;  // elements
  int64_t scale_stride;                                      // of a page's scales
  int64_t bt_stride, num_pages;
  int batch, hq, hkv, group, dim, page_size, max_pages, causal;
  float scale_log2;  // scale * log2(e)
  uint32_t* status;
  // Tensor-core kernel:
  int tile_tokens;     // tokens of a 128-row tile
  int block_tokens;    // of a block of one or two tiles
  int box_rows;        // token rows of a TMA box, a power of two: 1 << box_shift
  int box_shift;
  // A 16-bit tile in shared memory: groups of 8 tokens group_bytes apart, a row's 128-byte halves half_bytes apart. With
  // `merged` a TMA box has both halves: its coordinates are head * head_halves in halves and
  // page * page_groups + head * head_groups + token / 8 in groups, total_groups (and more) giving zeros.
  uint32_t group_bytes, half_bytes;
  int merged, head_halves, head_groups, page_groups, total_groups;
  float* partials;     // pieces of split row blocks
  uint32_t* counters;  // arrivals at a split block's rows
};

// Sequence b of the call: its rows first .. first + n - 1, its length.
struct Seq {
  int64_t first;
  int n, len;
};

__device__ __forceinline__ Seq read_seq(const Args& a, int b, bool report) {
  const int64_t lo = min(max(static_cast<int64_t>(__ldcg(a.indptr + b)), int64_t(0)), a.tokens);
  const int64_t hi = min(max(static_cast<int64_t>(__ldcg(a.indptr + b + 1)), int64_t(0)), a.tokens);
  Seq s{lo, static_cast<int>(max(hi - lo, int64_t(0))), max(0, __ldcg(a.seq_lens + b))};
  const int room = a.max_pages * a.page_size;
  if (s.len > room) {
    s.len = room;
    if (report) atomicOr(a.status, kStatusLenClamped);
  }
  return s;
}

// Keys that token i of the sequence sees.
__device__ __forceinline__ int keys_of(const Args& a, const Seq& s, int i) {
  return a.causal ? max(0, s.len - s.n + i + 1) : s.len;
}

// ----------------------------------------------------------------- tensor-core path (chunk_attention_tc.cu)

// Whether the call's types, sizes, strides and alignment allow it.
bool tc_fits(const Args& a, int dtype, int code_type);
size_t tc_partial_bytes(int head_dim, int sms);
size_t tc_sync_bytes(int sms);
cudaError_t launch_tc(Args a, int dtype, int code_type, int sms, cudaStream_t st);

}  // namespace chunk_attention
}  // namespace klb
