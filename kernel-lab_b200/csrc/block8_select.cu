// Selection of the pages a decode step should read (block-sparse decode), for sm_100a.
//
// For a sequence, KV head and page: with q rounded to int8 per query head (qi, scale sq) and the
// page's key bounds lo <= hi (int8),
//   I = sum_d max(qi_d lo_d, qi_d hi_d) = sum_d max(qi_d, 0) hi_d + min(qi_d, 0) lo_d
//   score = fl(max over the group's query heads of fl(I * sq)) * fl(unit * k_scale)
// I is a whole number below 2^24 (at most 127 * 127 * 256), formed by int8 matrix instructions with
// 32-bit accumulation, so the score is the same in whatever order it is summed, and so is the choice: the
// num_selected largest, ties to the lower page, the first and last pages first of all.
//
// Bound by reading the bounds: 2 * head_dim bytes a page and head, a sixteenth of the page's codes at
// 16 tokens a page. A block takes a slice of one (sequence, KV head)'s pages, a warp 16 of them at a
// time as the rows of mma.m16n8k32 (8 query heads as columns): the contraction runs over the channels in
// the order in which a lane's 16-byte reads deliver them, so bounds go from global memory straight
// into the products, eight reads in flight a lane. (By four-way dot products the same took 55
// instructions for each head and 16 pages.) The score
// goes to scratch as an order-preserving integer. The block that completes the row's count selects:
// a radix selection over the keys in its registers (a digit of 8 bits a pass, from the first bit in
// which they differ, ending when a digit's keys are all wanted), then a compaction in page order.
// Blocks wait for no other. Measured (32/8 heads of 128): 64 ragged sequences of up to 16384 tokens in
// pages of 16 26.4 us for 73 MB, 1 x 32768 tokens 8.0 us; the reads alone take 14.4 us of the first (256 bytes at
// random places), the rounding of q and the selection most of the rest.
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>

#include "block8.cuh"
#include "kernel_lab_b200_block8.h"

namespace klb {
// A namespace with a name: an unnamed one's symbols carry a hash of the file's text, and with them the
// compiler's register allocation would change with a comment.
namespace block8_select {

constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelTile = 16;          // pages of a warp's products
constexpr int kSelPass = kSelWarps * kSelTile;
constexpr int kSelPasses = 4;         // passes of kSelPass pages a block takes where the call has many
constexpr int kSelFew = 8, kSelMany = 16;  // keys a thread holds: rows of up to 2048 pages, chunks of 4096

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
  int q_aligned;    // q's rows start on 16 bytes
  float unit;       // codes a bound's unit stands for
};

// An order-preserving whole number above 0 for any score (zeros of either sign alike).
__device__ __forceinline__ uint32_t key_of(float s) {
  const uint32_t b = __float_as_uint(s + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ int pages_in_use(const SelectArgs& a, int b) {
  const int len = a.seq_lens[b];
  return len > 0 ? min(static_cast<int>(static_cast<uint32_t>(len - 1) / static_cast<uint32_t>(a.page_size)) + 1, a.max_pages) : 0;
}

// This lane's 8 elements of a query head: channels 4 * lane .. + 3 and 128 more.
template <typename E>
__device__ __forceinline__ void load_q(const SelectArgs& a, int64_t head, float (&v)[8]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int d = k * 128 + lane * 4;
    const E* q = static_cast<const E*>(a.q) + head * a.head_dim + d;
    Vec<E, 4> e;
#pragma unroll
    for (int j = 0; j < 4; ++j) e.v[j] = Storage<E>::store(0.0f);
    if (d < a.head_dim) {  // head_dim is a multiple of 16
      if (a.q_aligned) {
        e = *reinterpret_cast<const Vec<E, 4>*>(q);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) e.v[j] = q[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[k * 4 + j] = Storage<E>::load(e.v[j]);
  }
}

// A query head as int8: the positive parts, then the negative parts, `row` words each. By one warp.
__device__ __forceinline__ void quantise_q(const float (&v)[8], int row, uint32_t* words, float* sq) {
  const int lane = threadIdx.x & 31;
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (fabsf(v[i]) <= FLT_MAX) top = fmaxf(top, fabsf(v[i]));
  }
  const float scale = warp_allreduce_max(top) * kPer127;
  const float inv = reciprocal_scale(scale);
  if (lane == 0) *sq = scale;
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
      words[w] = up;
      words[row + w] = down;
    }
  }
}

// D += A (16 x 32, row) * B (32 x 8, col), int8, 32-bit accumulation.
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct SelectShared {
  uint32_t hist[2][kSelThreads];  // a digit of 8 bits, two passes in turn
  uint32_t red[2][kSelWarps];
  int2 before[kSelMany * kSelWarps];  // keys above / at the threshold before each 32 of a chunk
  int2 total;
  int digit, rest, exact;
};

// All threads: writes to `out` the indices of the `want` largest of keys[0, count) in ascending order,
// `first` added, ties to the lower index. A thread holds PER keys, index j * 256 + its own; rows longer
// than that are read again from L2 for each pass.
template <int PER>
__device__ __forceinline__ void select_largest(const uint32_t* keys, int count, int want, int first, int32_t* out,
                                               SelectShared& sh) {
  constexpr int kChunk = PER * kSelThreads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t k[PER];
  const auto read = [&](int c0) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = c0 + j * kSelThreads + tid;
      k[j] = i < count ? __ldcg(keys + i) : 0u;
    }
  };
  // f(key) over the chunk's keys of this thread; a chunk that is the only one stays in registers.
  const bool once = count <= kChunk;
  read(0);
  const auto for_keys = [&](auto&& f) {
    for (int c0 = 0; c0 < count; c0 += kChunk) {
      if (!once) read(c0);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (c0 + j * kSelThreads + tid < count) f(k[j]);
      }
    }
  };

  // The bits in which the keys differ: from the highest of (and ^ or) down.
  uint32_t all_and = 0xffffffffu, all_or = 0;
  for_keys([&](uint32_t key) { all_and &= key, all_or |= key; });
  all_and = __reduce_and_sync(0xffffffffu, all_and);
  all_or = __reduce_or_sync(0xffffffffu, all_or);
  if (lane == 0) sh.red[0][warp] = all_and, sh.red[1][warp] = all_or;
  sh.hist[0][tid] = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) all_and &= sh.red[0][w], all_or |= sh.red[1][w];
  const uint32_t differ = all_and ^ all_or;
  int low = differ ? 32 - __clz(differ) : 0;  // bits from `low` up are decided
  // The threshold's decided bits. Keys above it are in; of the keys equal to it in those bits the first
  // `rest` are.
  uint32_t prefix = low < 32 ? all_or >> low << low : 0u;
  int rest = want;
  for (int pass = 0; low > 0; ++pass) {
    uint32_t* const hist = sh.hist[pass & 1];
    const int shift = max(0, low - 8);
    const uint32_t decided = low < 32 ? 0xffffffffu << low : 0u, digits = 0xffu >> (8 - (low - shift));
    for_keys([&](uint32_t key) {
      if ((key & decided) == prefix) atomicAdd(&hist[(key >> shift) & digits], 1u);
    });
    __syncthreads();
    sh.hist[(pass + 1) & 1][tid] = 0;
    if (warp == 0) {  // lane l: digits 255 - 8l down; the digit at which the count reaches `rest`
      const uint4 hi = *reinterpret_cast<const uint4*>(&hist[252 - lane * 8]);
      const uint4 lo = *reinterpret_cast<const uint4*>(&hist[248 - lane * 8]);
      const uint32_t c[8] = {hi.w, hi.z, hi.y, hi.x, lo.w, lo.z, lo.y, lo.x};
      const uint32_t sum = c[0] + c[1] + c[2] + c[3] + c[4] + c[5] + c[6] + c[7];
      uint32_t inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      uint32_t above = inc - sum;
      const uint32_t target = static_cast<uint32_t>(rest);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (above < target && above + c[j] >= target) {
          sh.digit = 255 - (lane * 8 + j);
          sh.rest = static_cast<int>(target - above);
          sh.exact = above + c[j] == target;  // every key of this digit is wanted
        }
        above += c[j];
      }
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(sh.digit) << shift;
    rest = sh.rest;
    low = shift;
    if (sh.exact) break;
  }
  const uint32_t mask = 0xffffffffu << low;  // low < 32: the first digit decides eight bits

  // Compaction: counts of each 32 keys, their sums before each, then the indices.
  int gt_at = 0, eq_at = 0;
  for (int c0 = 0; c0 < count; c0 += kChunk) {
    if (!once) read(c0);
    const auto votes = [&](int j, uint32_t& gt, uint32_t& eq) {
      const bool in = c0 + j * kSelThreads + tid < count;
      const uint32_t key = k[j] & mask;
      gt = __ballot_sync(0xffffffffu, in && key > prefix);
      eq = __ballot_sync(0xffffffffu, in && key == prefix);
    };
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      uint32_t gt, eq;
      votes(j, gt, eq);
      if (lane == 0) sh.before[j * kSelWarps + warp] = make_int2(__popc(gt), __popc(eq));
    }
    __syncthreads();
    if (warp == 0) {
      constexpr int kEach = PER * kSelWarps / 32;
      int2 c[kEach];
      int g = 0, e = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        c[i] = sh.before[lane * kEach + i];
        g += c[i].x;
        e += c[i].y;
      }
      int gi = g, ei = e;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, gi, o), y = __shfl_up_sync(0xffffffffu, ei, o);
        if (lane >= o) gi += x, ei += y;
      }
      if (lane == 31) sh.total = make_int2(gi, ei);
      g = gi - g;
      e = ei - e;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        sh.before[lane * kEach + i] = make_int2(g, e);
        g += c[i].x;
        e += c[i].y;
      }
    }
    __syncthreads();
    const uint32_t below = (1u << lane) - 1u;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      uint32_t gt, eq;
      votes(j, gt, eq);
      const int2 b = sh.before[j * kSelWarps + warp];
      const int g = gt_at + b.x + __popc(gt & below), e = eq_at + b.y + __popc(eq & below);
      const bool tie = (eq >> lane) & 1u;
      if (((gt >> lane) & 1u) || (tie && e < rest)) out[g + min(e, rest)] = first + c0 + j * kSelThreads + tid;
    }
    gt_at += sh.total.x;
    eq_at += sh.total.y;
    __syncthreads();
  }
}

// CHUNKS: 16-byte pieces of a bound a lane reads (head_dim / 64, rounded up to a power of two). Up to 128 channels
// four blocks an SM: 64 registers, 24 to 40 bytes spilled.
template <typename E, int CHUNKS>
__global__ void __launch_bounds__(kSelThreads, CHUNKS == 4 ? 2 : 4) block_select_kernel(const SelectArgs a) {
  constexpr int kRow = CHUNKS * 16;         // words of one head's q part
  extern __shared__ __align__(16) uint32_t s_dyn[];  // q words of whole groups of 8 heads, then scales
  __shared__ __align__(16) SelectShared s_sel;
  __shared__ int s_last;

  wait_prior_grid();
  allow_next_grid();
  const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  // What needs no length is asked for together with it: this warp's first query head and the first
  // pass's pages (entries past the length lie in the table and are not used).
  const int32_t* const table = a.block_table + b * a.bt_stride;
  const int lo = blockIdx.x * a.slice;
  const int64_t row = static_cast<int64_t>(b) * a.num_kv_heads + h;
  int page[2];  // of rows g and g + 8
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int p = lo + warp * kSelTile + g + 8 * k;
    page[k] = p < a.max_pages ? table[p] : -1;
  }
  float q_first[8];
  if (warp < a.group) load_q<E>(a, row * a.group + warp, q_first);
  const int n = pages_in_use(a, b);
  int32_t* out = a.selected + row * a.num_selected;
  if (n <= a.num_selected) {  // every page
    if (blockIdx.x == 0) {
      for (int i = tid; i < a.num_selected; i += kSelThreads) out[i] = i < n ? i : -1;
    }
    return;
  }
  if (lo >= n) return;
  uint32_t* const keys = a.keys + row * a.max_pages;

  // ---- scores of pages [lo, hi)
  const int octets = (a.group + 7) / 8;
  uint32_t* const q_words = s_dyn;
  float* const sq = reinterpret_cast<float*>(s_dyn + octets * 8 * 2 * kRow);
  const int hi = min(n, lo + a.slice);
  const int8_t* const bounds = a.bounds + h * 2 * a.head_dim + c * 16;  // of page 0
  const int64_t page_bytes = static_cast<int64_t>(a.num_kv_heads) * 2 * a.head_dim;
  for (int m = warp; m < octets * 8; m += kSelWarps) {  // heads past the group: zeros
    if (m != warp && m < a.group) load_q<E>(a, row * a.group + m, q_first);
    if (m >= a.group) {
#pragma unroll
      for (int i = 0; i < 8; ++i) q_first[i] = 0.0f;
    }
    quantise_q(q_first, kRow, q_words + m * 2 * kRow, sq + m);
  }
  __syncthreads();
  for (int p0 = lo; p0 < hi; p0 += kSelPass) {
    uint4 bh[2][CHUNKS], bl[2][CHUNKS];
    bool ok[2];
    float scale[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {  // a page outside the pool, or past the end: page 0's, unused
      ok[k] = page[k] >= 0 && page[k] < a.num_pages;
      const int at = ok[k] ? page[k] : 0;
      const int8_t* from = bounds + at * page_bytes;
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j) {
        bh[k][j] = bl[k][j] = make_uint4(0, 0, 0, 0);
        if ((j * 4 + c) * 16 < a.head_dim) {
          bl[k][j] = __ldg(reinterpret_cast<const uint4*>(from + j * 64));
          bh[k][j] = __ldg(reinterpret_cast<const uint4*>(from + j * 64 + a.head_dim));
        }
      }
      scale[k] = __ldg(a.k_scale + static_cast<int64_t>(at) * a.num_kv_heads + h);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {  // the next pass's pages
      const int p = p0 + kSelPass + warp * kSelTile + g + 8 * k;
      page[k] = p < hi ? table[p] : -1;
    }
    float best[2] = {-INFINITY, -INFINITY};
    for (int m = 0; m < a.group; m += 8) {
      const uint32_t* const q = q_words + (m + g) * 2 * kRow + c * 4;
      int d[4] = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j) {
        const uint4 up = *reinterpret_cast<const uint4*>(q + j * 16);
        const uint4 down = *reinterpret_cast<const uint4*>(q + kRow + j * 16);
        mma_s8(d, bh[0][j].x, bh[1][j].x, bh[0][j].y, bh[1][j].y, up.x, up.y);
        mma_s8(d, bh[0][j].z, bh[1][j].z, bh[0][j].w, bh[1][j].w, up.z, up.w);
        mma_s8(d, bl[0][j].x, bl[1][j].x, bl[0][j].y, bl[1][j].y, down.x, down.y);
        mma_s8(d, bl[0][j].z, bl[1][j].z, bl[0][j].w, bl[1][j].w, down.z, down.w);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {  // heads m + 2c and m + 2c + 1
        const int head = m + 2 * c + e;
        const float s = sq[head];
        if (head < a.group) {
          best[0] = fmaxf(best[0], static_cast<float>(d[e]) * s);
          best[1] = fmaxf(best[1], static_cast<float>(d[2 + e]) * s);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      best[k] = fmaxf(best[k], __shfl_xor_sync(0xffffffffu, best[k], 1));
      best[k] = fmaxf(best[k], __shfl_xor_sync(0xffffffffu, best[k], 2));
      const int p = p0 + warp * kSelTile + g + 8 * k;
      if (c == k && p < hi) {
        if (!ok[k]) atomicOr(a.sync, kStatusBadPage);
        keys[p] = ok[k] ? key_of(best[k] * (scale[k] * a.unit)) : key_of(-INFINITY);
      }
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
  const int count = end - first, want = a.num_selected - (n - count);
  for (int i = tid; i < first; i += kSelThreads) out[i] = i;
  for (int i = tid; i < n - end; i += kSelThreads) out[first + want + i] = end + i;
  if (want == 0) return;
  if (count <= kSelFew * kSelThreads) {
    select_largest<kSelFew>(keys + first, count, want, first, out + first, s_sel);
  } else {
    select_largest<kSelMany>(keys + first, count, want, first, out + first, s_sel);
  }
}

bool select_pdl() {
  static const bool on = env_switch_on("KL_DECODE_PDL");
  return on;
}

template <typename E, int CHUNKS>
cudaError_t launch_select(const SelectArgs& a, dim3 grid, cudaStream_t st) {
  const size_t heads = static_cast<size_t>((a.group + 7) / 8) * 8;
  const size_t smem = heads * (2 * CHUNKS * 16 + 1) * sizeof(uint32_t);
  const auto kernel = block_select_kernel<E, CHUNKS>;
  if (smem > 40 * 1024) {  // 48 KB less the static part
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_shared_memory(kernel, 128 * 1024, done);
    if (e != cudaSuccess) return e;
  }
  return launch_kernel(select_pdl(), kernel, grid, dim3(kSelThreads), smem, st, a);
}

template <typename E>
cudaError_t launch_chunks(const SelectArgs& a, dim3 grid, cudaStream_t st) {
  if (a.head_dim <= 64) return launch_select<E, 1>(a, grid, st);
  if (a.head_dim <= 128) return launch_select<E, 2>(a, grid, st);
  return launch_select<E, 4>(a, grid, st);
}

}  // namespace block8_select
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
  using namespace klb::block8_select;
  constexpr int kInvalid = static_cast<int>(cudaErrorInvalidValue);
  if (batch == 0) return 0;
  if (batch < 0 || batch > 65535 || num_kv_heads <= 0 || num_kv_heads > 65535 || num_q_heads <= 0 ||
      num_q_heads % num_kv_heads != 0 || num_q_heads / num_kv_heads > 128 || head_dim <= 0 || head_dim % 16 != 0 ||
      head_dim > 256 || page_size <= 0 || max_pages_per_seq < 0 || block_table_stride < max_pages_per_seq ||
      num_pages <= 0 || num_pages > INT32_MAX || num_selected <= 0 || sink_pages < 0 || recent_pages < 0 ||
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
  a.q_aligned = (reinterpret_cast<uintptr_t>(q) & 15u) == 0;
  a.unit = static_cast<float>(code_type == KL_CODE_E4M3 ? E4m3Code::kBoundUnit : Int8Code::kBoundUnit);
  // A block scores kSelPasses passes where the call has many: q is rounded once for them (64 ragged
  // sequences of up to 16384 tokens with the decode of their selected pages: 1 pass a block 90.8 us, 2 86.4, 4 87.3).
  const int64_t passes = std::max<int64_t>(1, (static_cast<int64_t>(max_pages_per_seq) + kSelPass - 1) / kSelPass);
  const int64_t rows = static_cast<int64_t>(batch) * num_kv_heads;
  const int64_t per = rows * passes <= 4 * static_cast<int64_t>(sm_count()) ? 1 : kSelPasses;
  a.slice = static_cast<int>(std::min<int64_t>(per * kSelPass, INT32_MAX));
  const dim3 grid(static_cast<unsigned>((passes + per - 1) / per), static_cast<unsigned>(num_kv_heads),
                  static_cast<unsigned>(batch));
  const auto st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case KL_FLOAT32: return static_cast<int>(launch_chunks<float>(a, grid, st));
    case KL_FLOAT16: return static_cast<int>(launch_chunks<__half>(a, grid, st));
    case KL_BFLOAT16: return static_cast<int>(launch_chunks<__nv_bfloat16>(a, grid, st));
    default: return kInvalid;
  }
}
