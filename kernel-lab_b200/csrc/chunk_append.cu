// Append of chunks of new tokens to a paged cache (16- and 32-bit, and e4m3 with a scale for each KV head):
// row indptr[b] + i of k_new / v_new goes to token position positions[b] + i of sequence b.
//
// HBM-bound: every row is read once and written once. A warp takes a row of both tensors, all of its 16-byte
// units in flight at once, and finds the row's sequence by itself: 32 entries of indptr a step, so that 1024
// sequences take two dependent loads. 35,000 rows of 2 x 1024 bf16 elements: 49 us, 6,030 GB/s, 0.92 of the measured copy; to
// e4m3 50 us, 4,430 GB/s.
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "common.cuh"
#include "kernel_lab_b200.h"
#include "kernel_lab_b200_chunk.h"

namespace klb {
namespace chunk_append {

constexpr int kThreads = 256;

struct Args {
  void* k_cache;
  void* v_cache;
  const void* k_new;
  const void* v_new;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_table;
  const int32_t* positions;
  const int32_t* indptr;
  int64_t tokens;
  int64_t bt_stride;
  int64_t new_stride;
  int64_t num_pages;
  int batch;
  int max_pages;
  int page_size;
  int row_elems;
  int head_dim;
  uint32_t* status;
};

// The last b with indptr[b] <= row (-1: none), by the whole warp.
__device__ __forceinline__ int find_sequence(const int32_t* indptr, int batch, int64_t row, int lane) {
  int lo = 0, n = batch + 1;  // the answer is lo - 1 + the count of entries among [lo, lo + n) that are <= row
  while (n > 32) {
    const int step = (n + 31) / 32;
    const int i = lo + lane * step;
    const bool le = lane * step < n && __ldcg(indptr + i) <= row;
    const int c = __popc(__ballot_sync(0xffffffffu, le));
    if (c == 0) return lo - 1;
    const int first = (c - 1) * step;  // this probe is <= row, the next one is not
    lo += first + 1;
    n = min(step - 1, n - first - 1);
  }
  const bool le = lane < n && __ldcg(indptr + lo + lane) <= row;
  return lo - 1 + __popc(__ballot_sync(0xffffffffu, le));
}

// Where a row goes: its row index in the pool, -1 if nowhere.
__device__ __forceinline__ int64_t destination(const Args& a, int64_t row, int lane) {
  const int b = find_sequence(a.indptr, a.batch, row, lane);
  if (b < 0 || b >= a.batch) return -1;
  const int64_t i = row - __ldcg(a.indptr + b);
  const int start = __ldcg(a.positions + b);
  if (start < 0 || i < 0) return -1;
  const int64_t pos = start + i, col = pos / a.page_size;
  int64_t page = -1;
  if (col < a.max_pages) page = __ldcg(a.block_table + b * a.bt_stride + col);
  if (page < 0 || page >= a.num_pages) {
    if (lane == 0 && a.status) atomicOr(a.status, kStatusBadPage);
    return -1;
  }
  return page * a.page_size + (pos - col * a.page_size);
}

// Rows as they are, in units U (16 bytes where everything is aligned to that, else an element).
template <typename U>
__global__ void __launch_bounds__(kThreads) append_rows(const Args a, int units, int64_t src_units) {
  wait_prior_grid();
  allow_next_grid();
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (row >= a.tokens) return;
  const int64_t to = destination(a, row, lane);
  if (to < 0) return;
  const U* ks = static_cast<const U*>(a.k_new) + row * src_units;
  const U* vs = static_cast<const U*>(a.v_new) + row * src_units;
  U* kd = static_cast<U*>(a.k_cache) + to * units;
  U* vd = static_cast<U*>(a.v_cache) + to * units;
  constexpr int K = 4;  // units of each tensor in flight a lane
  for (int base = 0; base < units; base += 32 * K) {
    U k[K], v[K];
#pragma unroll
    for (int u = 0; u < K; ++u) {
      const int i = base + u * 32 + lane;
      if (i < units) {
        k[u] = __ldcg(ks + i);
        v[u] = __ldcg(vs + i);
      }
    }
#pragma unroll
    for (int u = 0; u < K; ++u) {
      const int i = base + u * 32 + lane;
      if (i < units) {
        kd[i] = k[u];
        vd[i] = v[u];
      }
    }
  }
}

// A scale, its reciprocal, and how a quotient may be formed with it: by the reciprocal alone where the scale is a power
// of two (the product is the quotient then), by the reciprocal but for quotients next to a border, or by division.
struct Scale {
  float s, inv;
  uint32_t near;  // a quotient whose last 19 bits are within 8 of zero is divided again; 0: none
  bool divide;
  __device__ explicit Scale(float x) : s(x), inv(1.0f / x) {
    divide = !(fabsf(x) >= 0x1p-100f && fabsf(x) <= 0x1p100f);
    near = (__float_as_uint(x) & 0x007fffffu) ? 16u : 0u;
  }
};

// e4m3(x / s), N elements, nearest-even, saturating; NaN stays NaN. x * (1 / s) is off by at most two units in the last of
// 24 places. A border between two codes has at most five significant bits, so the codes are those of the quotient unless the
// last 19 bits of the product are all but zero: one element in 32,768 of those that are not round numbers. A division
// takes about 15 instructions, which bound the kernel (35,000 rows of 2 x 1024 elements: 70.0 us, by products 50 us).
template <typename E, int N>
__device__ __forceinline__ void quantise(const Vec<E, N>& x, const Scale& s, uint8_t* to) {
  float q[N];
  bool again = s.divide;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    q[u] = Storage<E>::load(x.v[u]) * s.inv;
    again |= ((__float_as_uint(q[u]) + 8u) & 0x7ffffu) < s.near;
  }
  if (again) {
#pragma unroll
    for (int u = 0; u < N; ++u) q[u] = Storage<E>::load(x.v[u]) / s.s;
  }
  Vec<__nv_fp8x2_storage_t, N / 2> y;
#pragma unroll
  for (int u = 0; u < N; u += 2) y.v[u / 2] = __nv_cvt_float2_to_fp8x2(make_float2(q[u], q[u + 1]), __NV_SATFINITE, __NV_E4M3);
  *reinterpret_cast<Vec<__nv_fp8x2_storage_t, N / 2>*>(to) = y;
}

// N elements of both tensors a lane and step.
template <typename E, int N>
__global__ void __launch_bounds__(kThreads) append_rows_e4m3(const Args a) {
  wait_prior_grid();
  allow_next_grid();
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (row >= a.tokens) return;
  const int64_t to = destination(a, row, lane);
  if (to < 0) return;
  const E* const ks = static_cast<const E*>(a.k_new) + row * a.new_stride;
  const E* const vs = static_cast<const E*>(a.v_new) + row * a.new_stride;
  uint8_t* const kd = static_cast<uint8_t*>(a.k_cache) + to * a.row_elems;
  uint8_t* const vd = static_cast<uint8_t*>(a.v_cache) + to * a.row_elems;
#pragma unroll 2
  for (int i = lane * N; i < a.row_elems; i += 32 * N) {  // N divides head_dim
    Vec<E, N> k, v;
    if (N > 2) {
      k = *reinterpret_cast<const Vec<E, N>*>(ks + i);
      v = *reinterpret_cast<const Vec<E, N>*>(vs + i);
    } else {  // rows at any element
      k.v[0] = ks[i], k.v[1] = ks[i + 1];
      v.v[0] = vs[i], v.v[1] = vs[i + 1];
    }
    const int h = i / a.head_dim;
    quantise<E, N>(k, Scale(__ldg(a.k_scale + h)), kd + i);
    quantise<E, N>(v, Scale(__ldg(a.v_scale + h)), vd + i);
  }
}

bool pdl() {
  static const bool on = env_switch_on("KL_APPEND_PDL");
  return on;
}

template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), const Args& a, cudaStream_t st, const A&... more) {
  const int64_t blocks = (a.tokens + kThreads / 32 - 1) / (kThreads / 32);
  return launch_kernel(pdl(), kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, a, more...);
}

bool all_aligned(std::initializer_list<const void*> ps, uintptr_t n) {
  for (const void* p : ps) {
    if (reinterpret_cast<uintptr_t>(p) % n) return false;
  }
  return true;
}

template <typename E>
cudaError_t launch_e4m3(const Args& a, cudaStream_t st) {
  constexpr int N = 16 / sizeof(E);
  const bool vec = a.head_dim % N == 0 && a.new_stride % N == 0 && all_aligned({a.k_new, a.v_new}, 16) &&
                   all_aligned({a.k_cache, a.v_cache}, N);
  if (vec) return launch(append_rows_e4m3<E, N>, a, st);
  return all_aligned({a.k_cache, a.v_cache}, 2) ? launch(append_rows_e4m3<E, 2>, a, st) : cudaErrorInvalidValue;
}

// What both forms refuse; 0 where the call is fine.
int refused(const Args& a, int dtype) {
  if (a.batch < 0 || a.tokens < 0 || a.tokens > INT32_MAX || a.head_dim <= 0 || a.row_elems <= 0 || a.page_size <= 0 ||
      a.max_pages < 0 || a.bt_stride < a.max_pages || a.num_pages < 0 || a.new_stride < a.row_elems || !a.k_cache ||
      !a.v_cache || !a.k_new || !a.v_new || (!a.block_table && a.max_pages > 0) || !a.positions || !a.indptr) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  const bool known = dtype == KL_FLOAT32 || dtype == KL_FLOAT16 || dtype == KL_BFLOAT16;
  return known ? 0 : static_cast<int>(cudaErrorInvalidValue);
}

Args make(void* k_cache, void* v_cache, const void* k_new, const void* v_new, const float* k_scale,
          const float* v_scale, const int32_t* block_table, const int32_t* positions, const int32_t* indptr, int batch,
          int64_t tokens, int num_kv_heads, int head_dim, int page_size, int64_t block_table_stride,
          int max_pages_per_seq, int64_t num_pages, int64_t new_row_stride, uint32_t* status) {
  const int64_t row = num_kv_heads > 0 && head_dim > 0 ? static_cast<int64_t>(num_kv_heads) * head_dim : 0;
  return Args{k_cache, v_cache, k_new, v_new, k_scale, v_scale, block_table, positions, indptr, tokens,
              block_table_stride, new_row_stride, num_pages, batch, max_pages_per_seq, page_size,
              row <= (1 << 24) ? static_cast<int>(row) : 0, head_dim, status};
}

}  // namespace chunk_append
}  // namespace klb

extern "C" int kl_paged_kv_append_chunks(int dtype, void* k_cache, void* v_cache, const void* k_new, const void* v_new,
                                         const int32_t* block_table, const int32_t* positions, const int32_t* indptr,
                                         int batch, int64_t tokens, int num_kv_heads, int head_dim, int page_size,
                                         int64_t block_table_stride, int max_pages_per_seq, int64_t num_pages,
                                         int64_t new_row_stride, uint32_t* status, void* stream) {
  using namespace klb::chunk_append;
  if (batch == 0 || tokens == 0) return 0;
  const Args a = make(k_cache, v_cache, k_new, v_new, nullptr, nullptr, block_table, positions, indptr, batch, tokens,
                      num_kv_heads, head_dim, page_size, block_table_stride, max_pages_per_seq, num_pages,
                      new_row_stride, status);
  if (const int rc = refused(a, dtype)) return rc;
  const auto st = static_cast<cudaStream_t>(stream);
  const int e = dtype == KL_FLOAT32 ? 4 : 2;
  const bool vec = a.row_elems * static_cast<int64_t>(e) % 16 == 0 && new_row_stride * e % 16 == 0 &&
                   all_aligned({k_cache, v_cache, k_new, v_new}, 16);
  cudaError_t rc;
  if (vec) {
    rc = launch(append_rows<uint4>, a, st, a.row_elems / (16 / e), new_row_stride / (16 / e));
  } else if (e == 4) {
    rc = launch(append_rows<float>, a, st, a.row_elems, new_row_stride);
  } else {
    rc = launch(append_rows<uint16_t>, a, st, a.row_elems, new_row_stride);
  }
  return static_cast<int>(rc);
}

extern "C" int kl_paged_kv_append_chunks_fp8(int dtype, void* k_cache, void* v_cache, const void* k_new,
                                             const void* v_new, const float* k_scale, const float* v_scale,
                                             const int32_t* block_table, const int32_t* positions,
                                             const int32_t* indptr, int batch, int64_t tokens, int num_kv_heads,
                                             int head_dim, int page_size, int64_t block_table_stride,
                                             int max_pages_per_seq, int64_t num_pages, int64_t new_row_stride,
                                             uint32_t* status, void* stream) {
  using namespace klb::chunk_append;
  if (batch == 0 || tokens == 0) return 0;
  const Args a = make(k_cache, v_cache, k_new, v_new, k_scale, v_scale, block_table, positions, indptr, batch, tokens,
                      num_kv_heads, head_dim, page_size, block_table_stride, max_pages_per_seq, num_pages,
                      new_row_stride, status);
  if (const int rc = refused(a, dtype)) return rc;
  if (!k_scale || !v_scale || head_dim % 2) return static_cast<int>(cudaErrorInvalidValue);
  const auto st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case KL_FLOAT32: return static_cast<int>(launch_e4m3<float>(a, st));
    case KL_FLOAT16: return static_cast<int>(launch_e4m3<__half>(a, st));
    default: return static_cast<int>(launch_e4m3<__nv_bfloat16>(a, st));
  }
}
