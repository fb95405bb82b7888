// Attention of chunks of new tokens over a paged cache: sequence b's n new tokens are its last n, and token i
// sees the keys up to its own position (causal) or all of them.
//
//   out[i, h] = sum_j p_ij V_j,   p_ij = exp(s_ij - max_j s_ij) / sum_j exp(s_ij - max_j s_ij),   s_ij = scale q_i.K_j
//
// The rows of one product are the (token, query head) pairs of a KV head: its query heads share keys and values.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <type_traits>

#include "chunk_attention.cuh"

namespace klb {
namespace chunk_attention {

// ----------------------------------------------------------------- CUDA-core kernel
//
// Any dtype, cache, group, head_dim up to 256, page size and stride. A CTA takes kRows rows of one KV head and
// walks their keys kKeys at a time: K and V widened to fp32 in shared memory (rows padded with zeros to whole float4s), a thread
// per four scores, eight threads a row for the softmax and for the row's output. Bound by shared-memory loads (a float4 of
// q and four of K for 16 multiply-adds) and, with few rows, by one CTA's walk over a whole context, which is not split: fp32,
// 8 x 4 draft tokens over up to 1024 of 32/8 heads of 128 320 us, 4 tokens over 32,768 9.6 ms.

constexpr int kRows = 16, kKeys = 32, kThreads = 128, kMaxDim = 256;

template <typename C>
struct Code {  // an element of a cache, as fp32
  static __device__ __forceinline__ float load(C v) { return Storage<C>::load(v); }
};
template <>
struct Code<__nv_fp8_e4m3> {
  static __device__ __forceinline__ float load(__nv_fp8_e4m3 v) { return static_cast<float>(v); }
};
template <>
struct Code<int8_t> {
  static __device__ __forceinline__ float load(int8_t v) { return static_cast<float>(v); }
};

// Floats between rows of K (and of q and V without the last four): whole float4s, K's rows in turn on other banks.
__host__ __device__ __forceinline__ int padded(int dim) { return (dim + 3) / 4 * 4; }
size_t generic_smem(int dim) {
  const size_t d = padded(dim);
  return sizeof(float) * (kRows * d + kKeys * (2 * d + 4) + kRows * kKeys);
}

template <typename T, typename C>
__global__ void __launch_bounds__(kThreads) generic_kernel(const __grid_constant__ Args a) {
  extern __shared__ float smem[];
  __shared__ int s_found[2];
  __shared__ int s_scan[kThreads / 32];
  __shared__ int64_t s_page[kKeys];  // a key's page, -1: not to be attended to
  __shared__ int s_slot[kKeys];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, dim = a.dim;
  const int wide = padded(dim), k_row = wide + 4;
  float* sq = smem;                  // [kRows][wide]
  float* sk = sq + kRows * wide;     // [kKeys][wide + 4]
  float* sv = sk + kKeys * k_row;    // [kKeys][wide]
  float* sp = sv + kKeys * wide;     // [kRows][kKeys]; -1: masked
  wait_prior_grid();
  allow_next_grid();

  // Row block blockIdx.x of KV head blockIdx.y: whose it is.
  const int target = blockIdx.x, kvh = blockIdx.y;
  if (tid == 0) s_found[0] = -1;
  long long run = 0;
  for (int base = 0; base < a.batch; base += kThreads) {
    const int b = base + tid;
    int mine = 0;
    if (b < a.batch) {
      const Seq s = read_seq(a, b, false);
      mine = static_cast<int>((static_cast<int64_t>(s.n) * a.group + kRows - 1) / kRows);
    }
    int inc = mine;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, m);
      if (lane >= m) inc += y;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    long long before = run;
    for (int w = 0; w < warp; ++w) before += s_scan[w];
    for (int w = 0; w < kThreads / 32; ++w) run += s_scan[w];
    const long long first = before + inc - mine;
    if (target >= first && target < first + mine) {
      s_found[0] = b;
      s_found[1] = static_cast<int>(target - first);
    }
    if (run > target) break;
  }
  __syncthreads();
  const int b = s_found[0];
  if (b < 0) return;
  const Seq s = read_seq(a, b, tid == 0);
  const int64_t row0 = static_cast<int64_t>(s_found[1]) * kRows, rows = static_cast<int64_t>(s.n) * a.group;

  for (int i = warp; i < kRows; i += kThreads / 32) {
    const int64_t r = row0 + i;
    const bool there = r < rows;
    const int64_t token = s.first + (there ? r / a.group : 0);
    const T* const from = static_cast<const T*>(a.q) + token * a.q_stride + (kvh * a.group + (there ? r % a.group : 0)) * static_cast<int64_t>(dim);
    for (int d = lane; d < wide; d += 32) sq[i * wide + d] = there && d < dim ? Storage<T>::load(from[d]) : 0.0f;
  }
  const int r = tid >> 3, part = tid & 7;  // this thread's row, and its eighth of the row
  const int64_t my_row = row0 + r;
  const int limit = my_row < rows ? keys_of(a, s, static_cast<int>(my_row / a.group)) : 0;
  const int last_limit = keys_of(a, s, static_cast<int>((min(rows, row0 + kRows) - 1) / a.group));
  constexpr int kParts = kMaxDim / 32;  // float4s of the row's output a thread: columns 4 * part + 32 * i
  float4 acc[kParts];
#pragma unroll
  for (int i = 0; i < kParts; ++i) acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float m = -INFINITY, l = 0.0f;

  for (int k0 = 0; k0 < last_limit; k0 += kKeys) {
    __syncthreads();
    if (tid < kKeys) {
      const int j = k0 + tid;
      int64_t page = -1;
      if (j < s.len) {
        page = __ldcg(a.block_table + b * a.bt_stride + j / a.page_size);
        if (page < 0 || page >= a.num_pages) {
          page = -1;
          atomicOr(a.status, kStatusBadPage);
        }
      }
      s_page[tid] = page;
      s_slot[tid] = j % a.page_size;
    }
    __syncthreads();
    // A warp's four keys, 64 columns of each in flight.
    constexpr int kMine = kKeys / (kThreads / 32);
    float ks[kMine], vs[kMine];
    int64_t at[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int j = warp + i * (kThreads / 32);
      const int64_t page = s_page[j];
      at[i] = page < 0 ? -1 : page * a.page_stride + s_slot[j] * a.token_stride + kvh * a.head_stride;
      ks[i] = vs[i] = 1.0f;
      if (!std::is_same<C, T>::value && page >= 0) {
        ks[i] = __ldcg(a.k_scale + page * a.scale_stride + kvh);
        vs[i] = __ldcg(a.v_scale + page * a.scale_stride + kvh);
      }
    }
    for (int d0 = lane; d0 < wide; d0 += 64) {
      float x[kMine][2], y[kMine][2];
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int d = d0 + 32 * u;
          const bool there = at[i] >= 0 && d < dim;
          x[i][u] = there ? Code<C>::load(static_cast<const C*>(a.k)[at[i] + d]) : 0.0f;
          y[i][u] = there ? Code<C>::load(static_cast<const C*>(a.v)[at[i] + d]) : 0.0f;
        }
      }
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int j = warp + i * (kThreads / 32);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int d = d0 + 32 * u;
          if (d >= wide) break;
          sk[j * k_row + d] = std::is_same<C, T>::value || at[i] < 0 ? x[i][u] : x[i][u] * ks[i];
          sv[j * wide + d] = std::is_same<C, T>::value || at[i] < 0 ? y[i][u] : y[i][u] * vs[i];
        }
      }
    }
    __syncthreads();
    float x[kKeys / 8];
#pragma unroll
    for (int i = 0; i < kKeys / 8; ++i) x[i] = 0.0f;
#pragma unroll 4
    for (int d = 0; d < wide; d += 4) {
      const float4 qd = *reinterpret_cast<const float4*>(sq + r * wide + d);
#pragma unroll
      for (int i = 0; i < kKeys / 8; ++i) {
        const float4 kd = *reinterpret_cast<const float4*>(sk + (part + 8 * i) * k_row + d);
        x[i] = fmaf(qd.x, kd.x, fmaf(qd.y, kd.y, fmaf(qd.z, kd.z, fmaf(qd.w, kd.w, x[i]))));
      }
    }
    float mc = -INFINITY;
    bool seen[kKeys / 8];
#pragma unroll
    for (int i = 0; i < kKeys / 8; ++i) {
      const int j = part + 8 * i;
      seen[i] = k0 + j < limit && s_page[j] >= 0;
      x[i] *= a.scale_log2;
      if (seen[i]) mc = fmaxf(mc, x[i]);
    }
#pragma unroll
    for (int w = 4; w > 0; w >>= 1) mc = fmaxf(mc, __shfl_xor_sync(0xffffffffu, mc, w));
    const float mn = fmaxf(m, mc), shift = mn == -INFINITY ? 0.0f : mn;
    const float alpha = exp2f(m - shift);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kKeys / 8; ++i) {
      const float p = exp2f(x[i] - shift);
      if (seen[i]) sum += p;
      sp[r * kKeys + part + 8 * i] = seen[i] ? p : -1.0f;
    }
#pragma unroll
    for (int w = 4; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    m = mn;
    l = l * alpha + sum;
    __syncwarp();  // a row's eight threads are in one warp
#pragma unroll
    for (int i = 0; i < kParts; ++i) acc[i] = make_float4(acc[i].x * alpha, acc[i].y * alpha, acc[i].z * alpha, acc[i].w * alpha);
#pragma unroll 4
    for (int j = 0; j < kKeys; ++j) {
      const float p = sp[r * kKeys + j];
      if (p < 0.0f) continue;  // masked, whatever V holds
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        if (32 * i >= wide) break;
        const int d = 4 * part + 32 * i;
        if (d < wide) {
          const float4 v = *reinterpret_cast<const float4*>(sv + j * wide + d);
          acc[i] = make_float4(fmaf(p, v.x, acc[i].x), fmaf(p, v.y, acc[i].y), fmaf(p, v.z, acc[i].z), fmaf(p, v.w, acc[i].w));
        }
      }
    }
  }
  if (my_row >= rows) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T* out = static_cast<T*>(a.out) + ((s.first + my_row / a.group) * a.hq + kvh * a.group + my_row % a.group) * dim;
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    const float o[4] = {acc[i].x, acc[i].y, acc[i].z, acc[i].w};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int d = 4 * part + 32 * i + u;
      if (d < dim) out[d] = Storage<T>::store(o[u] * inv);
    }
  }
}

template <typename T, typename C>
cudaError_t launch_generic(const Args& a, cudaStream_t st) {
  const size_t smem = generic_smem(a.dim);
  cudaError_t e = cudaFuncSetAttribute(generic_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  // At most this many blocks of rows: each sequence's last one may be short.
  const int64_t blocks = a.tokens * a.group / kRows + std::min<int64_t>(a.batch, a.tokens);
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(a.hkv));
  return launch_kernel(true, generic_kernel<T, C>, grid, dim3(kThreads), smem, st, a);
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    (void)cudaGetLastError();
    return 148;
  }
  return n;
}

}  // namespace chunk_attention
}  // namespace klb

extern "C" int kl_paged_chunk_attention_workspace_size(int dtype, int code_type, int64_t tokens, int batch,
                                                       int num_q_heads, int num_kv_heads, int head_dim,
                                                       size_t* partial_bytes, size_t* sync_bytes) {
  if (!partial_bytes || !sync_bytes) return static_cast<int>(cudaErrorInvalidValue);
  const int sms = klb::chunk_attention::sm_count();
  *partial_bytes = dtype == KL_FLOAT32 ? 0 : klb::chunk_attention::tc_partial_bytes(head_dim, sms);
  *sync_bytes = klb::chunk_attention::tc_sync_bytes(sms);
  return 0;
}

extern "C" int kl_paged_chunk_attention(int dtype, int code_type, void* out, const void* q, const void* k_cache,
                                        const void* v_cache, const float* k_scale, const float* v_scale,
                                        const int32_t* block_table, const int32_t* seq_lens, const int32_t* indptr,
                                        int batch, int64_t tokens, int num_q_heads, int num_kv_heads, int head_dim,
                                        int page_size, int64_t q_row_stride, int64_t page_stride, int64_t token_stride,
                                        int64_t head_stride, int64_t scale_page_stride, int64_t block_table_stride,
                                        int max_pages_per_seq, int64_t num_pages, int causal, float scale,
                                        void* partials, size_t partial_bytes, void* sync, size_t sync_bytes,
                                        void* stream) {
  using namespace klb::chunk_attention;
  const int invalid = static_cast<int>(cudaErrorInvalidValue);
  if (batch < 0 || tokens < 0) return invalid;
  if (batch == 0 || tokens == 0) return 0;
  if (dtype != KL_FLOAT32 && dtype != KL_FLOAT16 && dtype != KL_BFLOAT16) return invalid;
  const bool coded = code_type != KL_CODE_NONE;
  if (coded && code_type != KL_CODE_E4M3 && code_type != KL_CODE_INT8) return invalid;
  if (coded && (dtype == KL_FLOAT32 || !k_scale || !v_scale || scale_page_stride < 0)) return invalid;
  if (batch > 65535 || tokens > INT_MAX - 256 || num_kv_heads <= 0 || num_kv_heads > 65535 || num_q_heads <= 0 || num_q_heads % num_kv_heads != 0 ||
      head_dim <= 0 || head_dim > kMaxDim || page_size <= 0 || max_pages_per_seq < 0 || block_table_stride < max_pages_per_seq ||
      num_pages < 1 || static_cast<int64_t>(max_pages_per_seq) * page_size > INT_MAX - 256 ||
      q_row_stride < static_cast<int64_t>(num_q_heads) * head_dim || page_stride < 0 || token_stride < 0 || head_stride < 0) {
    return invalid;
  }
  if (!out || !q || !k_cache || !v_cache || (!block_table && max_pages_per_seq > 0) || !seq_lens || !indptr || !sync || sync_bytes < 256) return invalid;
  if (reinterpret_cast<uintptr_t>(sync) % 4) return invalid;
  Args a{};
  a.out = out;
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.block_table = block_table;
  a.seq_lens = seq_lens;
  a.indptr = indptr;
  a.tokens = tokens;
  a.q_stride = q_row_stride;
  a.page_stride = page_stride;
  a.token_stride = token_stride;
  a.head_stride = head_stride;
  a.scale_stride = scale_page_stride;
  a.bt_stride = block_table_stride;
  a.num_pages = num_pages;
  a.batch = batch;
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.dim = head_dim;
  a.page_size = page_size;
  a.max_pages = max_pages_per_seq;
  a.causal = causal != 0;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.status = static_cast<uint32_t*>(sync);
  const auto st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  const int sms = sm_count();
  if (partials && partial_bytes >= tc_partial_bytes(head_dim, sms) && sync_bytes >= tc_sync_bytes(sms) &&
      tc_fits(a, dtype, code_type)) {
    if (reinterpret_cast<uintptr_t>(partials) % 32) return invalid;  // pieces are stored 32 bytes at a time
    a.partials = static_cast<float*>(partials);
    a.counters = static_cast<uint32_t*>(sync) + 64;
    return static_cast<int>(launch_tc(a, dtype, code_type, sms, st));
  }
  if (!coded) {
    e = dtype == KL_FLOAT32   ? launch_generic<float, float>(a, st)
        : dtype == KL_FLOAT16 ? launch_generic<__half, __half>(a, st)
                              : launch_generic<__nv_bfloat16, __nv_bfloat16>(a, st);
  } else if (dtype == KL_FLOAT16) {
    e = code_type == KL_CODE_E4M3 ? launch_generic<__half, __nv_fp8_e4m3>(a, st) : launch_generic<__half, int8_t>(a, st);
  } else {
    e = code_type == KL_CODE_E4M3 ? launch_generic<__nv_bfloat16, __nv_fp8_e4m3>(a, st)
                                  : launch_generic<__nv_bfloat16, int8_t>(a, st);
  }
  return static_cast<int>(e);
}
