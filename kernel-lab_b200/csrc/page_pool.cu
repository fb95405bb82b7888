// The pages of a paged cache: copied, given to growing and forked sequences (reserve), compacted.
//
// No counts are kept: a page is in use if the first ceil(len / page_size) entries of some row name it. A call
// marks every page that its rows name in an array of one word a page, finds the free ones by a scan over that
// array in the order of the ids, and writes the new table; what has to move goes on a list of (source,
// destination) pages that the copy kernel works off. Everything follows from the inputs alone (marks by
// atomic maximum, ranks by scans), so two runs give the same table.
//
// Bookkeeping is bound by latency: table and marks are a few hundred KB that stay in L2. Marks are scattered 4-byte
// stores, which all SMs share (one cluster alone took 7 us for 65,000 of them); the rest is one cluster of kClusterCtas
// CTAs of kPlanThreads threads, its phases divided by cluster barriers: the CTAs of a cluster are resident together by
// definition. It clears the marks behind itself.
// Copies: HBM-bound, 2 * bytes. CTAs take 16 KB slices of a page, all loads of a slice before its stores (250 pages of 48
// tensors: 135 us, 5,830 GB/s, 0.89 of the measured copy).
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "common.cuh"
#include "kernel_lab_b200.h"
#include "kernel_lab_b200_chunk.h"

namespace klb {
namespace page_pool {

namespace cg = cooperative_groups;

constexpr uint32_t kStatusNoPages = KL_STATUS_NO_PAGES;

// ----------------------------------------------------------------- copies

constexpr int kCopyThreads = 256;
constexpr int kSlice = 16384;     // bytes of a page that a CTA takes at a time
constexpr int kMaxTensors = 64;   // of one launch

struct CopyArgs {
  uint8_t* base[kMaxTensors];
  int64_t stride[kMaxTensors];
  int64_t bytes[kMaxTensors];
  int64_t slice_end[kMaxTensors];  // slices of a page in the tensors up to this one
  uint8_t unit[kMaxTensors];       // bytes of a load: 16, 4 or 1
  int count;
  const int32_t* src;
  const int32_t* dst;
  int64_t pairs;
  const int32_t* pairs_on_device;  // if non-null, their number
  int64_t num_pages;
  uint32_t* status;
};

template <typename U>
__device__ __forceinline__ void copy_slice(uint8_t* to, const uint8_t* from, int bytes) {
  constexpr int K = kSlice / 16 / kCopyThreads;
  const U* s = reinterpret_cast<const U*>(from);
  U* d = reinterpret_cast<U*>(to);
  const int n = bytes / static_cast<int>(sizeof(U));
  for (int base = threadIdx.x; base < n; base += K * kCopyThreads) {
    U v[K];
#pragma unroll
    for (int u = 0; u < K; ++u) {
      if (base + u * kCopyThreads < n) v[u] = s[base + u * kCopyThreads];
    }
#pragma unroll
    for (int u = 0; u < K; ++u) {
      if (base + u * kCopyThreads < n) d[base + u * kCopyThreads] = v[u];
    }
  }
}

__global__ void __launch_bounds__(kCopyThreads) copy_pages(const __grid_constant__ CopyArgs a) {
  wait_prior_grid();
  allow_next_grid();
  const int64_t pairs = a.pairs_on_device ? __ldcg(a.pairs_on_device) : a.pairs;
  const int64_t per_page = a.slice_end[a.count - 1];
  for (int64_t item = blockIdx.x; item < pairs * per_page; item += gridDim.x) {
    const int64_t i = item / per_page, s = item - i * per_page;
    const int from = __ldcg(a.src + i), to = __ldcg(a.dst + i);
    if (from < 0 || to < 0) continue;
    if (from >= a.num_pages || to >= a.num_pages) {
      if (threadIdx.x == 0 && a.status) atomicOr(a.status, kStatusBadPage);
      continue;
    }
    int t = 0, hi = a.count - 1;  // the first tensor with slice_end > s
    while (t < hi) {
      const int mid = (t + hi) >> 1;
      if (a.slice_end[mid] > s) hi = mid; else t = mid + 1;
    }
    const int64_t off = (s - (t ? a.slice_end[t - 1] : 0)) * kSlice;
    const int bytes = static_cast<int>(min(static_cast<int64_t>(kSlice), a.bytes[t] - off));
    const uint8_t* p = a.base[t] + from * a.stride[t] + off;
    uint8_t* q = a.base[t] + to * a.stride[t] + off;
    if (a.unit[t] == 16) copy_slice<uint4>(q, p, bytes);
    else if (a.unit[t] == 4) copy_slice<uint32_t>(q, p, bytes);
    else copy_slice<uint8_t>(q, p, bytes);
  }
}

bool valid(const kl_page_pools_t* pools) {
  if (!pools || pools->count < 0 || (pools->count > 0 && (!pools->base || !pools->stride || !pools->bytes))) return false;
  for (int t = 0; t < pools->count; ++t) {
    if (!pools->base[t] || pools->bytes[t] < 0 || pools->stride[t] < pools->bytes[t]) return false;
  }
  return true;
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  return n;
}

// `pairs`: their number, or with pairs_on_device the most that there can be.
cudaError_t launch_copies(const kl_page_pools_t* pools, const int32_t* src, const int32_t* dst, int64_t pairs,
                          const int32_t* pairs_on_device, int64_t num_pages, uint32_t* status, cudaStream_t st) {
  if (pairs == 0) return cudaSuccess;
  for (int first = 0; first < pools->count; first += kMaxTensors) {
    CopyArgs a{};
    int64_t slices = 0;
    for (int t = first; t < pools->count && t < first + kMaxTensors; ++t) {
      if (pools->bytes[t] == 0) continue;
      const int k = a.count++;
      a.base[k] = static_cast<uint8_t*>(pools->base[t]);
      a.stride[k] = pools->stride[t];
      a.bytes[k] = pools->bytes[t];
      slices += (a.bytes[k] + kSlice - 1) / kSlice;
      a.slice_end[k] = slices;
      const int64_t bits = static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.base[k])) | a.stride[k] | a.bytes[k];
      a.unit[k] = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
    }
    if (a.count == 0) continue;
    a.src = src;
    a.dst = dst;
    a.pairs = pairs;
    a.pairs_on_device = pairs_on_device;
    a.num_pages = num_pages;
    a.status = status;
    const int64_t most = pairs > INT64_MAX / slices ? INT64_MAX : pairs * slices;
    const int64_t grid = std::min<int64_t>(most, static_cast<int64_t>(sm_count()) * 8);
    const cudaError_t e = launch_kernel(true, copy_pages, dim3(static_cast<unsigned>(grid)), dim3(kCopyThreads), 0, st, a);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// ----------------------------------------------------------------- bookkeeping

constexpr int kClusterCtas = 8;
constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kHeld = INT_MAX;  // the mark of a page that a row holds and is not about to write

struct RowPlan;

struct PlanArgs {
  const int32_t* block_table;
  const int32_t* seq_lens;
  const int32_t* new_tokens;  // reserve
  const int32_t* parents;     // reserve; may be null
  int32_t* out_table;
  int32_t* out_lens;          // reserve
  uint8_t* served;            // reserve
  int32_t* used;              // compact
  int64_t bt_stride;
  int64_t num_pages;
  int batch, rows, width, page_size;
  // scratch
  int32_t* mark;       // [num_pages, rounded up to 4]
  int32_t* pool_list;  // [num_pages]: free ids in order (reserve), sources of moves (compact)
  int32_t* src;        // pairs to copy
  int32_t* dst;
  int32_t* count;      // their number
  RowPlan* row_plan;   // [rows] (reserve)
  int64_t* begin;      // [rows]: the row's first page among those given out
  int32_t* copy_begin; // [rows]: its copy's place on the list
  int64_t* totals;     // [0]: pages needed
  uint32_t* status;
};

template <typename N>
struct ScanSpace {
  N warp[kPlanWarps];
  N total;
};

struct Shared {
  ScanSpace<int> pages;
  ScanSpace<long long> needs;
  ScanSpace<int> copies;
  int cta_count;  // read by the other CTAs
};

// Exclusive block-wide prefix sum of a number a thread; the total in sp.total.
template <typename N>
__device__ __forceinline__ N scan(ScanSpace<N>& sp, N v) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  N inc = v;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const N y = __shfl_up_sync(0xffffffffu, inc, m);
    if (lane >= m) inc += y;
  }
  __syncthreads();  // the previous use of the array is over
  if (lane == 31) sp.warp[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const N w = sp.warp[lane];
    N x = w;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const N y = __shfl_up_sync(0xffffffffu, x, m);
      if (lane >= m) x += y;
    }
    sp.warp[lane] = x - w;
    if (lane == 31) sp.total = x;
  }
  __syncthreads();
  return inc - v + sp.warp[warp];
}

// The CTAs' counts: their sum, and that of those before this one.
template <typename Cluster>
__device__ __forceinline__ void counts_before(Cluster& cluster, Shared& sh, int cta, int& before, int& all) {
  const int lane = threadIdx.x & 31;
  const int n = lane < kClusterCtas ? cluster.map_shared_rank(&sh, lane)->cta_count : 0;
  all = __reduce_add_sync(0xffffffffu, n);
  before = __reduce_add_sync(0xffffffffu, lane < cta ? n : 0);
}

struct Row {
  int parent;  // -1: empty
  int len, have;
};

// What the later phases need of a row: its length, how many pages it has, how many tokens are to come, its last page.
struct alignas(16) RowPlan {
  int len, have, add, last;
};

constexpr int kAhead = 8;  // entries of a row in flight a lane: a phase is a chain of round trips to L2

__device__ __forceinline__ Row read_row(const PlanArgs& a, int r, bool report) {
  Row x{r, 0, 0};
  if (a.parents) x.parent = __ldcg(a.parents + r);
  if (x.parent < 0 || x.parent >= a.batch) {
    x.parent = -1;
    return x;
  }
  x.len = max(0, __ldcg(a.seq_lens + x.parent));
  const long long room = static_cast<long long>(a.width) * a.page_size;
  if (x.len > room) {
    x.len = static_cast<int>(room);
    if (report && a.status) atomicOr(a.status, kStatusLenClamped);
  }
  x.have = (x.len + a.page_size - 1) / a.page_size;  // room < 2^31 - page_size
  return x;
}

__device__ __forceinline__ void store_mark(int32_t* p, int v) {
  asm volatile("st.relaxed.gpu.global.s32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}

// This CTA's pages: a multiple of 4 of them, so that marks are read 16 bytes at a time.
__device__ __forceinline__ void own_pages(const PlanArgs& a, int cta, int64_t& lo, int64_t& hi) {
  const int64_t quads = (a.num_pages + 3) / 4, per = (quads + kClusterCtas - 1) / kClusterCtas;
  lo = min(quads, cta * per) * 4;
  hi = min(quads, (cta + 1) * per) * 4;
}

__device__ __forceinline__ int4 marks_at(const PlanArgs& a, int64_t p) {
  int4 m = __ldcg(reinterpret_cast<const int4*>(a.mark + p));
  // Places past the last page count as held.
  if (p + 1 >= a.num_pages) m.y = kHeld;
  if (p + 2 >= a.num_pages) m.z = kHeld;
  if (p + 3 >= a.num_pages) m.w = kHeld;
  return m;
}

__device__ __forceinline__ void clear_marks(const PlanArgs& a, int cta) {
  int64_t lo, hi;
  own_pages(a, cta, lo, hi);
#pragma unroll 4
  for (int64_t p = lo + threadIdx.x * 4; p < hi; p += kPlanThreads * 4) {
    __stcg(reinterpret_cast<int4*>(a.mark + p), make_int4(0, 0, 0, 0));
  }
}

// Marks the pages that the rows name. A row that is to write its last page marks it with rows - r (of several the lowest
// has the largest), any other holder with kHeld. RESERVE: the rows' entries are taken over, too. A warp takes 256
// columns of a row.
constexpr int kMarkThreads = 256;

template <bool RESERVE>
__global__ void __launch_bounds__(kMarkThreads) mark_pages(const __grid_constant__ PlanArgs a) {
  wait_prior_grid();
  allow_next_grid();
  const int lane = threadIdx.x & 31;
  const int64_t parts = (a.width + 32 * kAhead - 1) / (32 * kAhead), items = a.rows * max(parts, int64_t(1));
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * (kMarkThreads / 32) + (threadIdx.x >> 5); item < items;
       item += static_cast<int64_t>(gridDim.x) * (kMarkThreads / 32)) {
    const int r = static_cast<int>(item / max(parts, int64_t(1)));
    const int part = static_cast<int>(item - r * max(parts, int64_t(1)));
    const int asked = RESERVE ? __ldcg(a.new_tokens + r) : 0;
    const Row x = read_row(a, r, part == 0 && lane == 0);
    const int add = x.parent < 0 ? 0 : max(0, asked);
    const bool writes = add > 0 && x.len % a.page_size != 0;
    const int32_t* in = a.block_table + (x.parent < 0 ? 0 : x.parent) * a.bt_stride;
    int32_t* out = a.out_table + static_cast<int64_t>(r) * a.width;
    const int c0 = part * 32 * kAhead + lane;
    int e[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) e[u] = c0 + 32 * u < x.have ? __ldcg(in + c0 + 32 * u) : 0;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int c = c0 + 32 * u;
      if (c < x.have) {
        if (e[u] < 0 || e[u] >= a.num_pages) {
          if (a.status) atomicOr(a.status, kStatusBadPage);
        } else if (RESERVE && writes && c == x.have - 1) {
          atomicMax(a.mark + e[u], a.rows - r);
        } else {
          store_mark(a.mark + e[u], kHeld);
        }
        if (RESERVE && c == x.have - 1) __stcg(reinterpret_cast<int4*>(a.row_plan + r), make_int4(x.len, x.have, add, e[u]));
      }
      if (RESERVE && c < a.width) out[c] = e[u];
    }
    if (RESERVE && part == 0 && lane == 0) {
      a.out_lens[r] = x.len;
      if (x.have == 0) __stcg(reinterpret_cast<int4*>(a.row_plan + r), make_int4(x.len, 0, add, -1));
    }
  }
}

__global__ void __cluster_dims__(kClusterCtas, 1, 1) __launch_bounds__(kPlanThreads)
reserve_plan(const __grid_constant__ PlanArgs a) {
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = static_cast<int>(cluster.block_rank());
  const int lane = threadIdx.x & 31, warp = cta * kPlanWarps + (threadIdx.x >> 5);
  constexpr int kWarps = kClusterCtas * kPlanWarps;
  if (threadIdx.x == 0) sh.cta_count = 0;
  __syncthreads();
  wait_prior_grid();
  allow_next_grid();

  // What each row needs, summed in order (CTA 0); the free pages of each CTA's part.
  int64_t lo, hi;
  own_pages(a, cta, lo, hi);
  int mine = 0;
#pragma unroll 4
  for (int64_t p = lo + threadIdx.x * 4; p < hi; p += kPlanThreads * 4) {
    const int4 m = marks_at(a, p);
    mine += (m.x == 0) + (m.y == 0) + (m.z == 0) + (m.w == 0);
  }
  mine = __reduce_add_sync(0xffffffffu, mine);
  if (lane == 0) atomicAdd(&sh.cta_count, mine);
  if (cta == 0) {
    long long need_before = 0;
    int copies_before = 0;
    for (int base = 0; base < a.rows; base += kPlanThreads) {
      const int r = base + threadIdx.x;
      long long need = 0;
      int copy = 0;
      if (r < a.rows) {
        const int4 v = __ldcg(reinterpret_cast<const int4*>(a.row_plan + r));
        const RowPlan x{v.x, v.y, v.z, v.w};
        const long long end = static_cast<long long>(x.len) + x.add;
        if (end <= static_cast<long long>(a.width) * a.page_size) {
          if (x.add > 0 && x.len % a.page_size != 0 && x.last >= 0 && x.last < a.num_pages) copy = __ldcg(a.mark + x.last) != a.rows - r;
          need = copy + (end + a.page_size - 1) / a.page_size - x.have;
        } else {
          need = -1;  // does not fit
        }
      }
      const bool fits = need >= 0;
      const long long n = scan(sh.needs, fits ? need : 0);
      const int k = scan(sh.copies, copy);
      if (r < a.rows) {
        a.begin[r] = fits ? need_before + n : -1;
        a.copy_begin[r] = copy ? copies_before + k : -1;
      }
      need_before += sh.needs.total;
      copies_before += sh.copies.total;
    }
    if (threadIdx.x == 0) {
      a.totals[0] = need_before;
      *a.count = copies_before;
    }
  }
  cluster.sync();

  // The lowest free pages in order, as many as are needed.
  int before, all;
  counts_before(cluster, sh, cta, before, all);
  const int wanted = static_cast<int>(min(static_cast<long long>(__ldcg(a.totals)), static_cast<long long>(all)));
  for (int64_t p0 = lo; p0 < hi && before < wanted; p0 += kPlanThreads * 4) {
    const int64_t p = p0 + threadIdx.x * 4;
    int4 m = make_int4(kHeld, kHeld, kHeld, kHeld);
    if (p < hi) m = marks_at(a, p);
    int at = before + scan(sh.pages, (m.x == 0) + (m.y == 0) + (m.z == 0) + (m.w == 0));
    const int marks[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (marks[u] == 0) {
        if (at < wanted) __stcg(a.pool_list + at, static_cast<int32_t>(p + u));
        ++at;
      }
    }
    before += sh.pages.total;
  }
  cluster.sync();  // also: no CTA has left while another reads its count
  clear_marks(a, cta);

  for (int r = warp; r < a.rows; r += kWarps) {
    const int4 v = __ldcg(reinterpret_cast<const int4*>(a.row_plan + r));
    const long long begin = __ldcg(a.begin + r);
    const int copy_at = __ldcg(a.copy_begin + r);
    const RowPlan x{v.x, v.y, v.z, v.w};
    const int grown = begin < 0 ? 0 : static_cast<int>((static_cast<long long>(x.len) + x.add + a.page_size - 1) / a.page_size - x.have);
    const int copies = copy_at >= 0;
    const bool ok = begin >= 0 && (grown + copies == 0 || begin + grown + copies <= all);
    int32_t* out = a.out_table + static_cast<int64_t>(r) * a.width;
    if (lane == 0) {
      a.served[r] = ok;
      if (!ok && a.status) atomicOr(a.status, kStatusNoPages);
      if (copies) {
        int from = -1, to = -1;
        if (ok) {
          from = x.last;
          to = __ldcg(a.pool_list + begin);
          out[x.have - 1] = to;
        }
        a.src[copy_at] = from;
        a.dst[copy_at] = to;
      }
    }
    for (int i = lane; ok && i < grown; i += 32) out[x.have + i] = __ldcg(a.pool_list + begin + copies + i);
  }
}

__global__ void __cluster_dims__(kClusterCtas, 1, 1) __launch_bounds__(kPlanThreads)
compact_plan(const __grid_constant__ PlanArgs a) {
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = static_cast<int>(cluster.block_rank());
  const int lane = threadIdx.x & 31, warp = cta * kPlanWarps + (threadIdx.x >> 5);
  constexpr int kWarps = kClusterCtas * kPlanWarps;
  if (threadIdx.x == 0) sh.cta_count = 0;
  __syncthreads();
  wait_prior_grid();
  allow_next_grid();
  int64_t lo, hi;
  own_pages(a, cta, lo, hi);
  int mine = 0;
#pragma unroll 4
  for (int64_t p = lo + threadIdx.x * 4; p < hi; p += kPlanThreads * 4) {
    const int4 m = marks_at(a, p);
    mine += static_cast<int>(min(a.num_pages, p + 4) - p) - ((m.x == 0) + (m.y == 0) + (m.z == 0) + (m.w == 0));
  }
  mine = __reduce_add_sync(0xffffffffu, mine);
  if (lane == 0) atomicAdd(&sh.cta_count, mine);
  cluster.sync();
  int before, used;
  counts_before(cluster, sh, cta, before, used);
  // Page p with L(p) pages in use below it. The free ones below `used` come in order as number p - L(p), the
  // ones in use from `used` on, counted down from the last, as number used - 1 - L(p): as many as the former.
  // In ascending order they are number L(p) - L(used), and L(used) = used - (free ones below it).
  for (int64_t p0 = lo; p0 < hi; p0 += kPlanThreads * 4) {
    const int64_t p = p0 + threadIdx.x * 4;
    int4 m = make_int4(0, 0, 0, 0);
    if (p < hi) m = marks_at(a, p);
    const int marks[4] = {m.x, m.y, m.z, m.w};
    int at = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) at += marks[u] != 0 && p + u < a.num_pages && p < hi;
    at = before + scan(sh.pages, at);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t id = p + u;
      if (p >= hi || id >= a.num_pages) continue;
      const bool in_use = marks[u] != 0;
      if (in_use && id >= used) a.pool_list[used - 1 - at] = static_cast<int32_t>(id);  // last first
      if (!in_use && id < used) __stcg(a.dst + (id - at), static_cast<int32_t>(id));
      if (id == used - 1) *a.count = used - at - in_use;  // free ones below `used`
      at += in_use;
    }
    before += sh.pages.total;
  }
  if (cta == 0 && threadIdx.x == 0) {
    *a.used = used;
    if (used == 0) *a.count = 0;
  }
  cluster.sync();  // also: no CTA has left while another reads its count
  const int moves = __ldcg(a.count);
  for (int i = cta * kPlanThreads + threadIdx.x; i < moves; i += kClusterCtas * kPlanThreads) {
    const int from = __ldcg(a.pool_list + (moves - 1 - i)), to = __ldcg(a.dst + i);
    a.src[i] = from;
    __stcg(a.mark + from, to + 1);  // where the page goes; its mark is not needed any more
  }
  cluster.sync();
  for (int r = warp; r < a.rows; r += kWarps) {
    const Row x = read_row(a, r, false);
    const int32_t* in = a.block_table + static_cast<int64_t>(r) * a.bt_stride;
    int32_t* out = a.out_table + static_cast<int64_t>(r) * a.width;
    for (int c0 = lane; c0 < a.width; c0 += 32 * kAhead) {
      int e[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) e[u] = c0 + 32 * u < x.have ? __ldcg(in + c0 + 32 * u) : 0;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (c0 + 32 * u < x.have && e[u] >= used && e[u] < a.num_pages) e[u] = __ldcg(a.mark + e[u]) - 1;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (c0 + 32 * u < a.width) out[c0 + 32 * u] = e[u];
      }
    }
  }
  cluster.sync();
  clear_marks(a, cta);
}

size_t rounded(size_t n) { return (n + 255) & ~size_t(255); }

// The scratch of a call, cut into its arrays; returns its size.
size_t cut(PlanArgs& a, uint8_t* p, int64_t num_pages, int64_t rows, int64_t pairs) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    uint8_t* at = p + off;
    off += rounded(bytes);
    return at;
  };
  a.totals = reinterpret_cast<int64_t*>(take(16));
  a.count = reinterpret_cast<int32_t*>(take(4));
  a.pool_list = reinterpret_cast<int32_t*>(take(static_cast<size_t>(num_pages) * 4));
  a.src = reinterpret_cast<int32_t*>(take(static_cast<size_t>(pairs) * 4));
  a.dst = reinterpret_cast<int32_t*>(take(static_cast<size_t>(pairs) * 4));
  a.row_plan = reinterpret_cast<RowPlan*>(take(static_cast<size_t>(rows) * sizeof(RowPlan)));
  a.begin = reinterpret_cast<int64_t*>(take(static_cast<size_t>(rows) * 8));
  a.copy_begin = reinterpret_cast<int32_t*>(take(static_cast<size_t>(rows) * 4));
  return off;
}

// Status word and marks, which every call leaves zero.
constexpr size_t kMarksAt = 256;
size_t sync_size(int64_t num_pages) { return kMarksAt + static_cast<size_t>(num_pages + 3) / 4 * 16; }

cudaError_t launch_marks(void (*kernel)(PlanArgs), const PlanArgs& a, cudaStream_t st) {
  const int64_t parts = std::max<int64_t>(1, (a.width + 32 * kAhead - 1) / (32 * kAhead));
  const int64_t warps = kMarkThreads / 32, blocks = (a.rows * parts + warps - 1) / warps;
  return launch_kernel(true, kernel, dim3(static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(blocks, 1), sm_count() * 8))),
                       dim3(kMarkThreads), 0, st, a);
}

// The marks and the plan after them, which zeroes the marks. Where it cannot be launched, they are zeroed all the same.
cudaError_t launch_plan(void (*marks)(PlanArgs), void (*plan)(PlanArgs), const PlanArgs& a, cudaStream_t st) {
  cudaError_t e = launch_marks(marks, a, st);
  if (e != cudaSuccess) return e;
  e = launch_kernel(true, plan, dim3(kClusterCtas), dim3(kPlanThreads), 0, st, a);
  if (e != cudaSuccess) (void)cudaMemsetAsync(a.mark, 0, sync_size(a.num_pages) - kMarksAt, st);
  return e;
}

constexpr int kMaxRows = 1 << 24;

bool sizes_ok(int batch, int rows, int width, int page_size, int64_t bt_stride, int64_t num_pages) {
  return batch >= 0 && rows >= 0 && rows <= kMaxRows && width >= 0 && page_size > 0 && bt_stride >= width && num_pages >= 0 &&
         num_pages <= INT32_MAX - 8 && static_cast<int64_t>(width) * page_size <= INT32_MAX - page_size;
}

bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na > 0 && nb > 0 && x < y + static_cast<uintptr_t>(nb) && y < x + static_cast<uintptr_t>(na);
}

// Whether an output lies over an input or another output: some rows are written while others are read. The lengths alone may
// be updated in place, where every row is its own parent.
bool outputs_overlap(const PlanArgs& a) {
  struct Region {
    const void* at;
    int64_t bytes;
  };
  const int64_t rows = a.rows;
  const Region out[] = {{a.out_table, rows * a.width * 4}, {a.out_lens, a.out_lens ? rows * 4 : 0}, {a.served, a.served ? rows : 0}, {a.used, a.used ? 4 : 0}};
  const Region in[] = {{a.block_table, a.batch > 0 ? ((a.batch - 1) * a.bt_stride + a.width) * 4 : 0},
                       {a.seq_lens, int64_t(a.batch) * 4},
                       {a.new_tokens, a.new_tokens ? rows * 4 : 0},
                       {a.parents, a.parents ? rows * 4 : 0}};
  const bool in_place = !a.parents && a.out_lens == a.seq_lens;
  for (int o = 0; o < 4; ++o) {
    for (int i = 0; i < 4; ++i) {
      if (o == 1 && i == 1 && in_place) continue;
      if (overlap(out[o].at, out[o].bytes, in[i].at, in[i].bytes)) return true;
    }
    for (int i = 0; i < o; ++i) {
      if (overlap(out[o].at, out[o].bytes, out[i].at, out[i].bytes)) return true;
    }
  }
  return false;
}

}  // namespace page_pool
}  // namespace klb

extern "C" int kl_paged_copy_pages(const kl_page_pools_t* pools, const int32_t* src, const int32_t* dst, int64_t pairs,
                                   int64_t num_pages, uint32_t* status, void* stream) {
  using namespace klb::page_pool;
  if (!valid(pools) || pairs < 0 || pairs > INT32_MAX || num_pages < 0 || num_pages > INT32_MAX || (pairs > 0 && (!src || !dst))) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  if (pairs == 0) return 0;
  return static_cast<int>(launch_copies(pools, src, dst, pairs, nullptr, num_pages, status, static_cast<cudaStream_t>(stream)));
}

extern "C" int kl_paged_reserve_workspace_size(int64_t num_pages, int rows, size_t* scratch_bytes, size_t* sync_bytes) {
  using namespace klb::page_pool;
  if (num_pages < 0 || num_pages > INT32_MAX - 8 || rows < 0 || rows > kMaxRows || !scratch_bytes || !sync_bytes) return static_cast<int>(cudaErrorInvalidValue);
  PlanArgs a{};
  *scratch_bytes = cut(a, nullptr, num_pages, rows, rows);
  *sync_bytes = sync_size(num_pages);
  return 0;
}

extern "C" int kl_paged_reserve(const kl_page_pools_t* pools, int32_t* out_table, int32_t* out_lens, uint8_t* served,
                                const int32_t* block_table, const int32_t* seq_lens, const int32_t* new_tokens,
                                const int32_t* parents, int batch, int rows, int width, int page_size,
                                int64_t block_table_stride, int64_t num_pages, void* scratch, size_t scratch_bytes,
                                void* sync, size_t sync_bytes, void* stream) {
  using namespace klb::page_pool;
  const int invalid = static_cast<int>(cudaErrorInvalidValue);
  if (!valid(pools) || !sizes_ok(batch, rows, width, page_size, block_table_stride, num_pages)) return invalid;
  if (!parents && rows != batch) return invalid;
  if (rows == 0) return 0;
  if (!out_lens || !served || !new_tokens || (batch > 0 && !seq_lens) || (width > 0 && (!out_table || (batch > 0 && !block_table)))) return invalid;
  PlanArgs a{};
  const size_t need = cut(a, static_cast<uint8_t*>(scratch), num_pages, rows, rows);
  if (!scratch || scratch_bytes < need || !sync || sync_bytes < sync_size(num_pages)) return invalid;
  if (reinterpret_cast<uintptr_t>(scratch) % 16 || reinterpret_cast<uintptr_t>(sync) % 16) return invalid;
  a.status = static_cast<uint32_t*>(sync);
  a.mark = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(sync) + kMarksAt);
  a.block_table = block_table;
  a.seq_lens = seq_lens;
  a.new_tokens = new_tokens;
  a.parents = parents;
  a.out_table = out_table;
  a.out_lens = out_lens;
  a.served = served;
  a.bt_stride = block_table_stride;
  a.num_pages = num_pages;
  a.batch = batch;
  a.rows = rows;
  a.width = width;
  a.page_size = page_size;
  if (outputs_overlap(a)) return invalid;
  const auto st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = launch_plan(mark_pages<true>, reserve_plan, a, st);
  if (e != cudaSuccess) return static_cast<int>(e);
  return static_cast<int>(launch_copies(pools, a.src, a.dst, rows, a.count, num_pages, a.status, st));
}

extern "C" int kl_paged_compact_workspace_size(int64_t num_pages, size_t* scratch_bytes, size_t* sync_bytes) {
  using namespace klb::page_pool;
  if (num_pages < 0 || num_pages > INT32_MAX - 8 || !scratch_bytes || !sync_bytes) return static_cast<int>(cudaErrorInvalidValue);
  PlanArgs a{};
  *scratch_bytes = cut(a, nullptr, num_pages, 0, num_pages);
  *sync_bytes = sync_size(num_pages);
  return 0;
}

extern "C" int kl_paged_compact(const kl_page_pools_t* pools, int32_t* out_table, int32_t* used,
                                const int32_t* block_table, const int32_t* seq_lens, int batch, int width,
                                int page_size, int64_t block_table_stride, int64_t num_pages, void* scratch,
                                size_t scratch_bytes, void* sync, size_t sync_bytes, void* stream) {
  using namespace klb::page_pool;
  const int invalid = static_cast<int>(cudaErrorInvalidValue);
  if (!valid(pools) || !sizes_ok(batch, batch, width, page_size, block_table_stride, num_pages) || !used) return invalid;
  if (batch > 0 && (!seq_lens || (width > 0 && (!out_table || !block_table)))) return invalid;
  PlanArgs a{};
  const size_t need = cut(a, static_cast<uint8_t*>(scratch), num_pages, 0, num_pages);
  if (!scratch || scratch_bytes < need || !sync || sync_bytes < sync_size(num_pages)) return invalid;
  if (reinterpret_cast<uintptr_t>(scratch) % 16 || reinterpret_cast<uintptr_t>(sync) % 16) return invalid;
  a.status = static_cast<uint32_t*>(sync);
  a.mark = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(sync) + kMarksAt);
  a.block_table = block_table;
  a.seq_lens = seq_lens;
  a.out_table = out_table;
  a.used = used;
  a.bt_stride = block_table_stride;
  a.num_pages = num_pages;
  a.batch = batch;
  a.rows = batch;
  a.width = width;
  a.page_size = page_size;
  if (outputs_overlap(a)) return invalid;
  const auto st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = launch_plan(mark_pages<false>, compact_plan, a, st);
  if (e != cudaSuccess) return static_cast<int>(e);
  // Pages with ids of `used` and more that go below it: at most half of them.
  return static_cast<int>(launch_copies(pools, a.src, a.dst, num_pages / 2, a.count, num_pages, a.status, st));
}
