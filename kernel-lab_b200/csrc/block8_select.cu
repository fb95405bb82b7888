// Selection of the pages a decode step should read (block-sparse decode), for sm_100a.
//
// For a sequence, KV head and page: with q rounded to int8 per query head (qi, scale sq) and the
// page's key bounds lo <= hi (int8),
//   I = sum_d max(qi_d lo_d, qi_d hi_d) = sum_d max(qi_d, 0) hi_d + min(qi_d, 0) lo_d
//   score = fl(max over the group's query heads of fl(I * sq)) * fl(unit * k_scale)
// I is a whole number below 2^24 (at most 2 * 127 * 127 * 256 / 2), formed by four-way integer dot
// products, so the score is the same in whatever order it is summed, and so is the choice: the
// num_selected largest, ties to the lower page, the first and last pages first of all.
//
// Bound by reading the bounds: 2 * head_dim bytes a page and head, a sixteenth of the page's codes at
// 16 tokens a page. A block takes a slice of one (sequence, KV head)'s pages: 16 bytes of lo and of hi
// a lane, head_dim / 16 lanes (rounded up to a power of two) side by side on a page, four pages in
// flight a lane; the group's q sits in shared memory and is read once for the four pages. The four
// sums are reduced over the lanes by halving (each step exchanges half of the sums), then the score
// goes to scratch as an order-preserving integer. The block that completes the row's count selects:
// a radix selection over the keys in shared memory (a digit of 8 bits a pass, from the first bit in
// which they differ, ending when a digit's keys are all wanted), then a compaction in page order.
// Blocks wait for no other.
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>

#include "block8.cuh"
#include "kernel_lab_b200_block8.h"

namespace klb {
namespace {

constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelPages = 4;          // pages in flight a lane
constexpr int kSelPasses = 2;         // passes of a block where the call has many
constexpr int kSelKeys = 8192;        // keys a block holds in shared memory; longer rows stay in L2

struct SelectArgs {
  int32_t* selected;
  const void* q;
  const int8_t* bounds;
  const float* k_scale;
  const int32_t* block_table;
  const int32_t* seq_lens;
  uint32_t* keys;   // [batch * num_kv_heads][max_pages]
  uint32_t* sync;   // [0] status, [1 + row] arrival counters
  int64_t bt_stride, num_pages;
  int num_kv_heads, group, head_dim, page_size, max_pages;
  int num_selected, sink, recent;
  int slice;        // pages a block scores
  float unit;       // codes a bound's unit stands for
};

// An order-preserving whole number above 0 for any score (zeros of either sign alike).
__device__ __forceinline__ uint32_t key_of(float s) {
  const uint32_t b = __float_as_uint(s + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ int pages_in_use(const SelectArgs& a, int b) {
  const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page_size;
  const int64_t len = min(static_cast<int64_t>(a.seq_lens[b]), cap);
  return len > 0 ? static_cast<int>((len - 1) / a.page_size + 1) : 0;
}

// q of the group's query heads as int8: the positive parts, then the negative parts, `row` words each.
template <typename E>
__device__ __forceinline__ void quantise_q(const SelectArgs& a, int64_t first_head, int row, uint32_t* words,
                                           float* sq) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int n = warp; n < a.group; n += kSelWarps) {
    const E* q = static_cast<const E*>(a.q) + (first_head + n) * a.head_dim;
    float v[8];
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int d = (k * 32 + lane) * 4 + j;
        v[k * 4 + j] = d < a.head_dim ? Storage<E>::load(q[d]) : 0.0f;
        const float f = fabsf(v[k * 4 + j]);
        if (f <= FLT_MAX) top = fmaxf(top, f);
      }
    }
    const float scale = warp_allreduce_max(top) * kPer127;
    const float inv = reciprocal_scale(scale);
    if (lane == 0) sq[n] = scale;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t up = 0, down = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int qi = max(-127, min(127, __float2int_rn(v[k * 4 + j] * inv)));  // NaN: 0
        up |= static_cast<uint32_t>(max(qi, 0) & 0xff) << (8 * j);
        down |= static_cast<uint32_t>(min(qi, 0) & 0xff) << (8 * j);
      }
      const int w = k * 32 + lane;
      if (w < row) {
        words[n * 2 * row + w] = up;
        words[n * 2 * row + row + w] = down;
      }
    }
  }
}

// Sum over the block of two counts and the exclusive sums before this warp.
struct WarpCounts {
  int gt_before, eq_before, gt, eq;
};
__device__ __forceinline__ WarpCounts count_before(int gt, int eq, int2* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) part[warp] = make_int2(gt, eq);
  __syncthreads();
  WarpCounts c{0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) {
    if (w < warp) c.gt_before += part[w].x, c.eq_before += part[w].y;
    c.gt += part[w].x;
    c.eq += part[w].y;
  }
  return c;
}

// LANES: lanes side by side on a page (head_dim / 16 rounded up to a power of two).
template <typename E, int LANES>
__global__ void __launch_bounds__(kSelThreads, 4) block_select_kernel(const SelectArgs a) {
  constexpr int kRow = LANES * 4;           // words of one head's q part
  constexpr int kAtOnce = kSelThreads / LANES;
  extern __shared__ __align__(16) uint32_t s_dyn[];  // q words and scales; then the keys
  __shared__ uint32_t s_hist[kSelThreads];  // a digit of 8 bits
  __shared__ uint32_t s_red[2][kSelWarps];
  __shared__ int2 s_part[kSelWarps];
  __shared__ int s_last, s_digit, s_rest;

  wait_prior_grid();
  allow_next_grid();
  const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = pages_in_use(a, b);
  const int lo = blockIdx.x * a.slice;
  const int64_t row = static_cast<int64_t>(b) * a.num_kv_heads + h;
  int32_t* out = a.selected + row * a.num_selected;
  if (n <= a.num_selected) {  // every page
    if (blockIdx.x == 0) {
      for (int i = tid; i < a.num_selected; i += kSelThreads) out[i] = i < n ? i : -1;
    }
    return;
  }
  if (lo >= n) return;
  uint32_t* const keys = a.keys + row * a.max_pages;

  // ---- scores of pages [lo, hi): page ids first, then their bounds, q's rounding under those loads
  uint32_t* const q_words = s_dyn;
  float* const sq = reinterpret_cast<float*>(s_dyn + a.group * 2 * kRow);
  const int hi = min(n, lo + a.slice);
  const int sub = tid % LANES, col = tid / LANES;
  const bool wide = sub * 16 < a.head_dim;
  const int32_t* const table = a.block_table + b * a.bt_stride;
  int page[kSelPages];
#pragma unroll
  for (int k = 0; k < kSelPages; ++k) {
    const int p = lo + k * kAtOnce + col;
    page[k] = p < hi ? table[p] : -1;
  }
  for (int p0 = lo; p0 < hi; p0 += kAtOnce * kSelPages) {
    uint4 bl[kSelPages], bh[kSelPages];
    float scale[kSelPages];
    uint32_t bad = 0;  // pages outside the pool
#pragma unroll
    for (int k = 0; k < kSelPages; ++k) {
      const bool ok = page[k] >= 0 && page[k] < a.num_pages;
      bad |= ok ? 0u : 1u << k;
      const int64_t at = static_cast<int64_t>(ok ? page[k] : 0) * a.num_kv_heads + h;
      bl[k] = bh[k] = make_uint4(0, 0, 0, 0);
      scale[k] = 0.0f;
      if (ok) {
        const int8_t* from = a.bounds + at * 2 * a.head_dim + sub * 16;
        if (wide) {
          bl[k] = __ldg(reinterpret_cast<const uint4*>(from));
          bh[k] = __ldg(reinterpret_cast<const uint4*>(from + a.head_dim));
        }
        scale[k] = __ldg(a.k_scale + at) * a.unit;
      }
    }
#pragma unroll
    for (int k = 0; k < kSelPages; ++k) {  // the next pass's pages
      const int p = p0 + (kSelPages + k) * kAtOnce + col;
      page[k] = p < hi ? table[p] : -1;
    }
    if (p0 == lo) {
      quantise_q<E>(a, row * a.group, kRow, q_words, sq);
      __syncthreads();
    }
    float best = -INFINITY;  // of the page this lane ends up with
#pragma unroll 2
    for (int m = 0; m < a.group; ++m) {
      const uint4 up = *reinterpret_cast<const uint4*>(q_words + m * 2 * kRow + sub * 4);
      const uint4 down = *reinterpret_cast<const uint4*>(q_words + m * 2 * kRow + kRow + sub * 4);
      int s[kSelPages];
#pragma unroll
      for (int k = 0; k < kSelPages; ++k) {
        int v = __dp4a(static_cast<int>(up.x), static_cast<int>(bh[k].x), 0);
        v = __dp4a(static_cast<int>(up.y), static_cast<int>(bh[k].y), v);
        v = __dp4a(static_cast<int>(up.z), static_cast<int>(bh[k].z), v);
        v = __dp4a(static_cast<int>(up.w), static_cast<int>(bh[k].w), v);
        v = __dp4a(static_cast<int>(down.x), static_cast<int>(bl[k].x), v);
        v = __dp4a(static_cast<int>(down.y), static_cast<int>(bl[k].y), v);
        v = __dp4a(static_cast<int>(down.z), static_cast<int>(bl[k].z), v);
        s[k] = __dp4a(static_cast<int>(down.w), static_cast<int>(bl[k].w), v);
      }
      // Halving: lanes with bit LANES / 2 keep pages 2, 3, the others 0, 1; then bit LANES / 4.
      const bool up1 = (sub & (LANES / 2)) != 0, up2 = (sub & (LANES / 4)) != 0;
      const int k0 = up1 ? s[2] : s[0], k1 = up1 ? s[3] : s[1];
      const int g0 = up1 ? s[0] : s[2], g1 = up1 ? s[1] : s[3];
      const int a0 = k0 + __shfl_xor_sync(0xffffffffu, g0, LANES / 2);
      const int a1 = k1 + __shfl_xor_sync(0xffffffffu, g1, LANES / 2);
      int sum = (up2 ? a1 : a0) + __shfl_xor_sync(0xffffffffu, up2 ? a0 : a1, LANES / 4);
#pragma unroll
      for (int x = LANES / 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      best = fmaxf(best, static_cast<float>(sum) * sq[m]);
    }
    // The lanes with sub % (LANES / 4) == 0 write the page of their two high bits.
    const int k = sub / (LANES / 4);
    const int p = p0 + k * kAtOnce + col;
    if (sub % (LANES / 4) == 0 && p < hi) {
      const float f = k == 0 ? scale[0] : k == 1 ? scale[1] : k == 2 ? scale[2] : scale[3];
      const bool ok = (bad >> k & 1u) == 0;
      if (!ok) atomicOr(a.sync, kStatusBadPage);
      keys[p] = ok ? key_of(best * f) : key_of(-INFINITY);
    }
  }

  // ---- the block that completes the row selects
  const int slices = (n - 1) / a.slice + 1;
  __syncthreads();
  if (tid == 0) {
    bool last = true;
    if (slices > 1) {
      uint32_t* counter = a.sync + 1 + row;
      last = atom_add_acq_rel_gpu(counter, 1) == static_cast<uint32_t>(slices - 1);
      if (last) *counter = 0;
    }
    s_last = last;
  }
  __syncthreads();
  if (!s_last) return;

  // Pages [first, end) compete for `want` places; the sinks and the recent ones are in.
  const int first = min(a.sink, n), end = max(first, n - a.recent);
  int want = a.num_selected - (n - (end - first));
  const int count = end - first;
  const uint32_t* row_keys = keys + first;
  if (count <= kSelKeys) {
    for (int i = tid; i < count; i += kSelThreads) s_dyn[i] = __ldcg(keys + first + i);
    row_keys = s_dyn;
    __syncthreads();
  }
  const auto key_at = [&](int i) { return row_keys == s_dyn ? s_dyn[i] : __ldcg(keys + first + i); };

  // The bits in which the keys differ: from the highest of (and ^ or) down.
  uint32_t all_and = 0xffffffffu, all_or = 0;
  for (int i = tid; i < count; i += kSelThreads) {
    const uint32_t k = key_at(i);
    all_and &= k;
    all_or |= k;
  }
  all_and = __reduce_and_sync(0xffffffffu, all_and);
  all_or = __reduce_or_sync(0xffffffffu, all_or);
  if (lane == 0) s_red[0][warp] = all_and, s_red[1][warp] = all_or;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) all_and &= s_red[0][w], all_or |= s_red[1][w];
  const uint32_t differ = all_and ^ all_or;
  int low = differ ? 32 - __clz(differ) : 0;  // bits from `low` up are decided
  // The threshold's decided bits. Keys above it are in; of the keys equal to it in those bits the first
  // `want` are.
  uint32_t prefix = low < 32 ? all_or >> low << low : 0u;
  if (want == 0) {
    prefix = 0xffffffffu;
    low = 0;
  }
  const int wanted = want;
  while (low > 0) {
    const int shift = max(0, low - 8);
    s_hist[tid] = 0;
    __syncthreads();
    const uint32_t decided = low < 32 ? 0xffffffffu << low : 0u;
    for (int i = tid; i < count; i += kSelThreads) {
      const uint32_t k = key_at(i);
      if ((k & decided) == prefix) atomicAdd(&s_hist[(k >> shift) & (0xffu >> (8 - (low - shift)))], 1u);
    }
    __syncthreads();
    if (warp == 0) {  // lane l: digits 255 - 8l down; the digit at which the count reaches `want`
      uint32_t c[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        c[j] = s_hist[255 - (lane * 8 + j)];
        sum += c[j];
      }
      uint32_t inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      uint32_t above = inc - sum;
      const uint32_t target = static_cast<uint32_t>(want);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (above < target && above + c[j] >= target) {
          s_digit = 255 - (lane * 8 + j);
          s_rest = static_cast<int>(target - above);
          s_last = above + c[j] == target;  // every key of this digit is wanted
        }
        above += c[j];
      }
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(s_digit) << shift;
    want = s_rest;
    low = shift;
    if (s_last) break;
  }
  const uint32_t mask = 0xffffffffu << low;  // low < 32: the first digit decides eight bits

  // Compaction in page order: each warp takes a run of keys, counts, then writes.
  const int run = ((count + kSelWarps - 1) / kSelWarps + 31) & ~31;
  const int r0 = min(count, warp * run), r1 = min(count, r0 + run);
  int gt = 0, eq = 0;
  for (int i = r0; i < r1; i += 32) {
    const bool in = i + lane < r1;
    const uint32_t k = in ? key_at(i + lane) & mask : 0u;
    gt += __popc(__ballot_sync(0xffffffffu, in && k > prefix));
    eq += __popc(__ballot_sync(0xffffffffu, in && k == prefix));
  }
  const WarpCounts c = count_before(gt, eq, s_part);
  int gt_at = c.gt_before, eq_at = c.eq_before;
  for (int i = tid; i < first; i += kSelThreads) out[i] = i;
  for (int i = tid; i < n - end; i += kSelThreads) out[first + wanted + i] = end + i;
  for (int i = r0; i < r1; i += 32) {
    const bool in = i + lane < r1;
    const uint32_t k = in ? key_at(i + lane) & mask : 0u;
    const uint32_t mg = __ballot_sync(0xffffffffu, in && k > prefix);
    const uint32_t me = __ballot_sync(0xffffffffu, in && k == prefix);
    const uint32_t below = (1u << lane) - 1u;
    const int g = gt_at + __popc(mg & below), e = eq_at + __popc(me & below);
    const bool tie = (me >> lane) & 1u;
    if (((mg >> lane) & 1u) || (tie && e < want)) out[first + g + min(e, want)] = first + i + lane;
    gt_at += __popc(mg);
    eq_at += __popc(me);
  }
}

struct SelectPlan {
  int lanes, slice, slices;
  size_t scratch_bytes, sync_bytes;
};

bool select_pdl() {
  static const bool on = env_switch_on("KL_DECODE_PDL");
  return on;
}

template <typename E, int LANES>
cudaError_t launch_select(const SelectArgs& a, dim3 grid, cudaStream_t st) {
  const size_t q_bytes = static_cast<size_t>(a.group) * (2 * LANES * 4 + 1) * sizeof(uint32_t);
  const size_t key_bytes = static_cast<size_t>(std::min(a.max_pages, kSelKeys)) * sizeof(uint32_t);
  const size_t smem = std::max(q_bytes, key_bytes);
  const auto kernel = block_select_kernel<E, LANES>;
  if (smem > 46 * 1024) {  // 48 KB less the static part
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_shared_memory(kernel, 128 * 1024, done);
    if (e != cudaSuccess) return e;
  }
  return launch_kernel(select_pdl(), kernel, grid, dim3(kSelThreads), smem, st, a);
}

template <typename E>
cudaError_t launch_lanes(const SelectArgs& a, dim3 grid, cudaStream_t st) {
  const int units = a.head_dim / 16;
  if (units <= 4) return launch_select<E, 4>(a, grid, st);
  if (units <= 8) return launch_select<E, 8>(a, grid, st);
  return launch_select<E, 16>(a, grid, st);
}

}  // namespace
}  // namespace klb

extern "C" int kl_paged_block_select_workspace_size(int batch, int num_kv_heads, int max_pages_per_seq,
                                                    size_t* scratch_bytes, size_t* sync_bytes) {
  if (!scratch_bytes || !sync_bytes || batch < 0 || num_kv_heads <= 0 || max_pages_per_seq < 0) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  *scratch_bytes = static_cast<size_t>(batch) * num_kv_heads * max_pages_per_seq * sizeof(uint32_t);
  *sync_bytes = (1 + static_cast<size_t>(batch) * num_kv_heads) * sizeof(uint32_t);
  return 0;
}

extern "C" int kl_paged_block_select(int dtype, int code_type, int32_t* selected, const void* q, const void* k_bounds,
                                     const float* k_scale, const int32_t* block_table, const int32_t* seq_lens,
                                     int batch, int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                                     int64_t block_table_stride, int max_pages_per_seq, int64_t num_pages,
                                     int num_selected, int sink_pages, int recent_pages, void* scratch,
                                     size_t scratch_bytes, void* sync, size_t sync_bytes, void* stream) {
  using namespace klb;
  constexpr int kInvalid = static_cast<int>(cudaErrorInvalidValue);
  if (batch == 0) return 0;
  if (batch < 0 || batch > 65535 || num_kv_heads <= 0 || num_kv_heads > 65535 || num_q_heads <= 0 ||
      num_q_heads % num_kv_heads != 0 || num_q_heads / num_kv_heads > 128 || head_dim <= 0 || head_dim % 16 != 0 ||
      head_dim > 256 || page_size <= 0 || max_pages_per_seq < 0 || block_table_stride < max_pages_per_seq ||
      num_pages < 0 || num_pages > INT32_MAX || num_selected <= 0 || sink_pages < 0 || recent_pages < 0 ||
      static_cast<int64_t>(sink_pages) + recent_pages > num_selected || !selected || !q || !k_bounds || !k_scale ||
      !block_table || !seq_lens || !sync || (reinterpret_cast<uintptr_t>(k_bounds) & 15u) != 0) {
    return kInvalid;
  }
  if (code_type != KL_CODE_E4M3 && code_type != KL_CODE_INT8) return kInvalid;
  size_t need = 0, need_sync = 0;
  kl_paged_block_select_workspace_size(batch, num_kv_heads, max_pages_per_seq, &need, &need_sync);
  if (scratch_bytes < need || sync_bytes < need_sync || (need > 0 && !scratch)) return kInvalid;
  SelectArgs a{};
  a.selected = selected;
  a.q = q;
  a.bounds = static_cast<const int8_t*>(k_bounds);
  a.k_scale = k_scale;
  a.block_table = block_table;
  a.seq_lens = seq_lens;
  a.keys = static_cast<uint32_t*>(scratch);
  a.sync = static_cast<uint32_t*>(sync);
  a.bt_stride = block_table_stride;
  a.num_pages = num_pages;
  a.num_kv_heads = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.head_dim = head_dim;
  a.page_size = page_size;
  a.max_pages = max_pages_per_seq;
  a.num_selected = num_selected;
  a.sink = sink_pages;
  a.recent = recent_pages;
  a.unit = static_cast<float>(code_type == KL_CODE_E4M3 ? E4m3Code::kBoundUnit : Int8Code::kBoundUnit);
  // A block scores kSelPasses passes (its threads' four pages each): the second pass's loads hide behind
  // the first, and short rows leave no block idle for long.
  const int units = head_dim / 16;
  const int lanes = units <= 4 ? 4 : units <= 8 ? 8 : 16;
  const int pass = kSelThreads / lanes * kSelPages;
  const int64_t passes = std::max<int64_t>(1, (static_cast<int64_t>(max_pages_per_seq) + pass - 1) / pass);
  const int64_t rows = static_cast<int64_t>(batch) * num_kv_heads;
  const int64_t per = rows * passes <= 4 * static_cast<int64_t>(sm_count()) ? 1 : kSelPasses;
  a.slice = static_cast<int>(std::min<int64_t>(per * pass, INT32_MAX));
  const dim3 grid(static_cast<unsigned>((passes + per - 1) / per), static_cast<unsigned>(num_kv_heads),
                  static_cast<unsigned>(batch));
  const auto st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case KL_FLOAT32: return static_cast<int>(launch_lanes<float>(a, grid, st));
    case KL_FLOAT16: return static_cast<int>(launch_lanes<__half>(a, grid, st));
    case KL_BFLOAT16: return static_cast<int>(launch_lanes<__nv_bfloat16>(a, grid, st));
    default: return kInvalid;
  }
}
