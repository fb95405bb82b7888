// Single-token decode attention over a paged cache held in 8 bits (e4m3 or int8) with a scale for
// each page and KV head, for sm_100a: over all pages of a sequence, or over a list of pages for each
// sequence and KV head (block-sparse decode).
//
//   s_t = scale * k_scale[page(t), h] * sum_d q_d ck_{t,d}
//   out = (sum_t 2^(s_t - m) * v_scale[page(t), h] * cv_t) / sum_t 2^(s_t - m)     (s in base 2)
//
// HBM-bound: every code is read once and used for the group's query heads (4 to 16 operations a byte).
// CTAs of eight warps. A "tile" is 16 tokens of one KV head, 2 * 16 * head_dim bytes; each
// warp (or team of warps, below) streams its own tiles through its own ring of shared-memory stages
// with 16-byte cp.async, so no warp waits for another while it streams and page and token strides
// may be any. Rows past the sequence's end are zero-filled by the copy: code 0 is 0 in both formats, so
// whatever the page holds there (NaN codes included) never reaches a product.
//
// Warps of a CTA. Up to 8 * NT query heads of one KV head share a warp's products, so that codes are
// widened once for them: NT = 1 for groups of at most 8, 2 up to 16, 4 beyond for head_dim up to 64. (For 128 the
// outputs of 32 query heads fill the registers: 168 us against 120 on 128 ragged int8 sequences, 101
// against 70 for a group of 64. For 64 it is 48 against 55 us, 64 x 4000 tokens of 64/2 heads.) With NT = 4
// a lane keeps its query fragments in shared memory. Larger groups take HG warps, which form a team: they share one ring, each copies 1/HG of a tile and meets the others
// at a named barrier once a step. The CTA's teams are HB KV heads times TS parts of the token range; the
// TS parts' states are joined through shared memory at the end of a
// range. Many parallel KV heads and one part where there is work for every warp (fewest joins, and
// a page's heads are read together), more parts of fewer heads where the whole call is small. A warp
// takes two tiles a step: a tile is a chain of dependent steps, and two of them fill each other's gaps. One
// for head_dim above 128, whose ring has no room for more, and for NT = 4, whose four products a
// fragment are independent already (39.0 us against 41.2, 16 x 4000-8000 tokens of 128/2 heads of 64).
//
// Balance. Rows (sequence, block of HB heads) are laid end to end, each as long as its tiles plus a
// fixed charge for starting it, and CTA c takes the c-th equal piece, found by every CTA alone from
// seq_lens (no host synchronisation). A row that a boundary cuts has chunks: each chunk publishes
// its unnormalised state (fp32) and counts itself; the one that completes the count joins all of
// them in chunk order, so the result does not depend on which came last, and sets the counter back to
// zero. Nobody waits for another CTA.
//
// Measured (e4m3, 32/8 heads of 128, pages of 16), ten calls in a row and, after the bar, calls for 1.5 seconds under
// the card's power cap: 64 x 4096 tokens 93.4 | 107 us (5.8 | 5.0 TB/s, 0.88 | 0.77 of the copy peak; about 12 us are
// launch, first loads and joins), 128 x 8192 of 64/8 heads 338 | 411 us (0.98 | 0.80), 8 x 4096 22.9 | 22.5 us (0.45).
// Groups above 8 are bound by the latency of a warp's dependent steps with two warps a scheduler: 128
// ragged sequences of one int8 KV head for 32 query heads 122 us (2.0 TB/s, 0.31; issue 44 % busy).
//
// Products. S = K.Q^T and O^T += V^T.P^T by mma.m16n8k16 in f16 with fp32 accumulation: codes widen
// to f16 exactly, a bf16 q is divided by a power of two so that f16 holds it, k_scale and that power enter
// with the softmax scale. p is at most 2^8 (the running maximum is only raised when a score passes it
// by 8). What is rounded to f16 is P = p * v_scale / w: w, a power of two, is the head's own measure of its
// largest p * v_scale so far, so that neither the scales' magnitude nor a page of large values and
// vanishing probability takes bits from the tokens that count. It is taken anew whenever the maximum is raised
// (the weights before shrink with it) and when a step's v_scale passes w by 2^7, which keeps P at most 2^15
// between. A token's P is thus off by 2^-11 of itself or by 2^-25 of the largest p * v_scale.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "block8.cuh"
#include "kernel_lab_b200_block8.h"

namespace klb {
// A namespace with a name: an unnamed one's symbols carry a hash of the file's text, and with them the
// compiler's register allocation would change with a comment.
namespace block8_decode {

constexpr int kB8Warps = 8;
constexpr int kB8Threads = 32 * kB8Warps;
constexpr int kB8Tile = 16;
constexpr int kB8Meta = 32;        // bytes of a stage after its codes: scales (k, v) of its octets, valid counts
constexpr float kRaiseBy = 8.0f;   // the running maximum is raised when a score passes it by this (base 2)
constexpr float kNoMax = -1e30f;   // running maximum before the first score
constexpr float kLeastWeight = 0x1p-126f, kMostWeight = 0x1p126f;  // w and 1 / w are normal numbers
constexpr float kWeightRange = 128.0f;  // w is taken anew when a v_scale passes it by this
constexpr int kMaxShared = 227 * 1024 - 128;  // dynamic, beside the plan's static part
constexpr int kTeamBarrier = 1, kGroupBarrier = 8;  // named barriers: 1.. teams, 8.. groups

struct Block8Args {
  void* out;
  const void* q;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_table;
  const int32_t* seq_lens;
  const int32_t* selected;  // null: every page
  int32_t page_stride, token_stride, head_stride;
  int64_t bt_stride;
  int64_t num_pages;
  int batch, num_q_heads, num_kv_heads, group, head_dim, page_size, max_pages;
  int num_selected;
  int q_bf16;
  float scale_log2;
  int hb, ts, units;   // KV heads and token parts of a CTA; units = ceil(num_kv_heads / hb)
  int min_tiles;       // least length of a CTA's piece
  int row_charge;      // tiles' worth of time charged for starting a row
  uint32_t* sync;      // [0] status, [1 + (b * num_kv_heads + h) * HG + hg] arrival counters
  float* part_o;       // [slot][8 / ts][8 * NT][DP]
  float2* part_ml;     // [slot][8 / ts][8 * NT]: (maximum, sum)
};

// Tiles of a step, and stages (of a step's tiles) of a team's ring: what 227 KB hold beside the boxes of
// the joins.
__host__ __device__ constexpr int step_tiles(int dp, int nt) { return dp == 256 || nt == 4 ? 1 : 2; }
__host__ __device__ constexpr int ring_stages(int dp, int nt, int hg) {
  const int per_warp = dp != 64 ? 3 : nt == 4 ? 8 : 6;
  return hg * per_warp < 12 ? hg * per_warp : 12;
}
// Bytes in which a warp keeps its 32 query heads' fragments (none where registers hold them).
__host__ __device__ constexpr int query_bytes(int dp, int nt) { return nt == 4 ? 8 * nt * dp * 2 : 0; }
// Floats a lane hands over at a time in a join: the maxima and sums of 8 query heads and half of their
// outputs.
__host__ __device__ constexpr int box_floats(int dp) { return 4 + dp / 8; }

// The power of two at or below v, kept to where its reciprocal is a normal number too.
__device__ __forceinline__ float weight_unit(float v) {
  return __uint_as_float(__float_as_uint(fminf(fmaxf(v, kLeastWeight), kMostWeight)) & 0x7f800000u);
}
__device__ __forceinline__ float reciprocal_of_power(float w) { return __uint_as_float(0x7f000000u - __float_as_uint(w)); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes),
               "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// Four codes of a word -> two f16 pairs, exactly.
template <typename Code>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi);
template <>
__device__ __forceinline__ void widen<E4m3Code>(uint32_t w, uint32_t& lo, uint32_t& hi) {
  lo = e4m3x2_lo_to_f16x2(w);
  hi = e4m3x2_hi_to_f16x2(w);
}
// The byte c + 128 below the exponent of 1024 is the f16 1024 + 128 + c.
template <>
__device__ __forceinline__ void widen<Int8Code>(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u;
  const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
  const uint32_t l = __byte_perm(u, 0x64646464u, 0x4140), h = __byte_perm(u, 0x64646464u, 0x4342);
  const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&l), bias);
  const __half2 b = __hsub2(*reinterpret_cast<const __half2*>(&h), bias);
  lo = *reinterpret_cast<const uint32_t*>(&a);
  hi = *reinterpret_cast<const uint32_t*>(&b);
}

// Byte offset of 16-byte unit `u` of token row `r` of a tile: rows DP bytes apart, the units of each
// 128 bytes permuted so that the score product's reads (8 lanes: 2 rows x 4 units) and the value
// product's (8 lanes: rows 0, 2, 4, 6 or 1, 3, 5, 7 x 2 units) each meet 8 different units. Rows 8
// apart are permuted alike; the permutation is an exclusive or that is linear in the row's bits.
template <int DP>
__host__ __device__ constexpr uint32_t unit_offset(int r, int u) {
  if (DP == 64) return (r >> 1) * 128 + ((((r & 1) * 4 + u) ^ (((r >> 1) & 3) << 1)) << 4);
  const int f = (((r ^ (r >> 2)) & 1) << 2) | (r & 2);
  return r * DP + ((u ^ f) << 4);
}
// unit_offset(r + sub, u) from unit_offset(sub, u), for rows r that are a multiple of a copy's rows.
template <int DP>
__device__ __forceinline__ uint32_t row_block(uint32_t offset, int r) {
  const uint32_t flips = DP == 64 ? 0u : unit_offset<DP>(r, 0) & 127u;
  return (offset ^ flips) + r * DP;
}

struct Segment {
  int b, u;         // row: sequence, block of heads
  int x0, x1;       // tiles
  int tiles;        // of the whole row
  int len;
  int start;        // position of the row's first tile, relative to the CTA's piece
};

// Walks the rows of a CTA's piece; positions are relative to its begin.
struct RowWalk {
  int p, p1, start;  // start: position of row (b, u)
  int b, u, len, tiles;

  __device__ __forceinline__ void read_row(const Block8Args& a) {
    const int cap = a.max_pages * a.page_size;
    len = b < a.batch ? max(0, min(a.seq_lens[b], cap)) : 0;
    tiles = row_tiles(a, len);
  }
  static __device__ __forceinline__ int row_tiles(const Block8Args& a, int len) {
    const int n = a.selected ? a.num_selected * a.page_size : len;
    return len > 0 && n > 0 ? (n - 1) / kB8Tile + 1 : 1;  // an empty row has one tile, all masked
  }
  __device__ __forceinline__ bool next(const Block8Args& a, Segment& s) {
    while (p < p1) {
      const int x0 = p - start;
      const bool some = x0 < tiles;
      s = Segment{b, u, x0, min(tiles, p1 - start), tiles, len, start};
      start += tiles + a.row_charge;
      p = start;
      if (++u == a.units) {
        u = 0;
        ++b;
        read_row(a);
      }
      if (some) return true;
    }
    return false;
  }
};

struct PlanShared {
  long long warp_sum[kB8Warps + 1];
  long long before;  // positions of the sequences before the first one, divided by units
  int b;
};

// All threads: this CTA's piece and the row it starts in; returns false for an empty piece.
__device__ __forceinline__ bool plan_piece(const Block8Args& a, PlanShared* ps, RowWalk& w, int64_t& piece) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.batch + kB8Threads - 1) / kB8Threads;
  const int lo = min(a.batch, tid * per), hi = min(a.batch, lo + per);
  const int cap = a.max_pages * a.page_size;
  long long local = 0;
  bool over = false;
  for (int b = lo; b < hi; ++b) {
    const int len = a.seq_lens[b];
    over |= len > cap;
    local += RowWalk::row_tiles(a, max(0, min(len, cap))) + a.row_charge;
  }
  if (over && blockIdx.x == 0) atomicOr(a.sync, kStatusLenClamped);
  long long inc = local;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) ps->warp_sum[warp] = inc;
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < kB8Warps; ++i) {
    const long long v = ps->warp_sum[i];
    if (i < warp) before += v;
    total += v;
  }
  before += inc - local;
  total *= a.units;
  piece = max(static_cast<long long>(a.min_tiles), (total + gridDim.x - 1) / gridDim.x);
  const int64_t p0 = piece * blockIdx.x;
  if (p0 >= total) return false;
  if (p0 >= before * a.units && p0 < (before + local) * a.units) {  // one thread's
    int b = lo;
    for (; b < hi - 1; ++b) {
      const int cost = RowWalk::row_tiles(a, max(0, min(a.seq_lens[b], cap))) + a.row_charge;
      if (p0 < (before + cost) * a.units) break;
      before += cost;
    }
    ps->b = b;
    ps->before = before;
  }
  __syncthreads();
  w.b = ps->b;
  w.read_row(a);
  const int cost = w.tiles + a.row_charge;
  const int64_t first = ps->before * a.units;
  w.u = static_cast<int>((p0 - first) / cost);
  w.start = static_cast<int>(first + static_cast<int64_t>(w.u) * cost - p0);
  w.p = 0;
  w.p1 = static_cast<int>(min(piece, static_cast<int64_t>(total) - p0));
  return true;
}

// DP: head_dim rounded up to 64, 128 or 256 (the copies zero-fill the rest). NT: groups of 8 query
// heads a warp. HG: warps a team.
template <typename Code, int DP, int NT, int HG>
__global__ void __launch_bounds__(kB8Threads, 1) decode_block8_kernel(const Block8Args a) {
  constexpr int kTiles = step_tiles(DP, NT);
  constexpr int kStages = ring_stages(DP, NT, HG);
  constexpr int kTileBytes = kB8Tile * DP;
  constexpr int kPlace = 2 * kTileBytes + kB8Meta;  // a tile's codes (keys, values) and what goes with them
  constexpr int kStageBytes = kTiles * kPlace;
  constexpr int kUnits = DP / 16;             // 16-byte units of a row
  constexpr int kRows = 32 / kUnits;          // rows one copy instruction of a warp covers
  constexpr int kBlocks = kB8Tile / kRows;    // copy instructions of one tensor's tile
  constexpr int kHalves = DP == 256 ? 2 : 1;  // 128-byte parts of a row
  constexpr int kM = DP == 64 ? 4 : 8;        // value products (16 output channels) of a part
  constexpr int kSteps = DP / 16;             // score products (16 channels)
  constexpr int NH = 8 * NT;
  constexpr bool kQRegs = query_bytes(DP, NT) == 0;

  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ PlanShared s_plan;
  __shared__ int s_last[kB8Warps];

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int team = warp / HG, hg = warp % HG;
  const int hb = team / a.ts, ts = team % a.ts;
  const int groups = kB8Warps / a.ts;      // (hb, hg) pairs of the CTA
  const int grp = hb * HG + hg;

  wait_prior_grid();
  allow_next_grid();
  RowWalk cons;
  int64_t piece;
  if (!plan_piece(a, &s_plan, cons, piece)) return;
  // No block-wide barrier from here on: teams without a head leave.

  const uint32_t ring = smem_u32(smem) + team * (kStages * kStageBytes);
  constexpr int kRings = (kB8Warps / HG) * kStages * kStageBytes;
  // The lane's own query fragments, where they are not in registers: 16 bytes are two steps of one n.
  const uint32_t q_at = smem_u32(smem) + kRings + warp * query_bytes(DP, NT) + lane * 16;
  float* const joint = reinterpret_cast<float*>(smem + kRings + kB8Warps * query_bytes(DP, NT));
  const uint64_t policy = l2_policy_evict_first();

  // ---- loading side: the team's next tile
  RowWalk ahead = cons;
  int l_t = 0, l_t1 = 0;          // tiles left of the segment's part
  int l_entry = 0, l_sub = 0;     // page entry of the next tile and the tile's place in that page
  int l_win = 0;                  // first entry of the window
  int w_page = -1, w_col = 0, n_page = -1, n_col = 0;  // this lane's entry of the window, of the next one
  int l_b = 0, l_h = 0, l_len = 0;
  const int page_tiles = a.page_size / kB8Tile;  // 0: pages of 8 tokens
  const int unit = lane % kUnits, sub = lane / kUnits;
  const uint32_t unit_bytes = unit * 16 < a.head_dim ? 16u : 0u;  // channels past head_dim are zero-filled
  const uint32_t dst0 = unit_offset<DP>(sub, unit);

  const auto read_entry = [&](int e, int& page, int& col) {
    page = -1;
    col = e;
    const uint32_t page_size = static_cast<uint32_t>(a.page_size);  // the sum may pass 31 bits
    const int used = static_cast<int>((static_cast<uint32_t>(l_len) + page_size - 1u) / page_size);
    if (a.selected) {
      col = -1;
      if (e < a.num_selected) {
        col = a.selected[(static_cast<int64_t>(l_b) * a.num_kv_heads + l_h) * a.num_selected + e];
      }
    }
    if (col < 0 || col >= used) return;
    page = a.block_table[l_b * a.bt_stride + col];
    if (page < 0 || page >= a.num_pages) {
      atomicOr(a.sync, kStatusBadPage);
      page = -1;
    }
  };

  // Copies the team's next step to a stage; a segment's last step may end in tiles of nothing.
  const auto issue = [&](int slot) {
    while (l_t >= l_t1) {
      Segment s;
      if (!ahead.next(a, s)) {
        cp_async_commit();
        return;
      }
      l_b = s.b;
      l_h = s.u * a.hb + hb;
      l_len = s.len;
      if (l_h >= a.num_kv_heads) continue;
      const int part = (s.x1 - s.x0 + a.ts - 1) / a.ts;
      l_t = s.x0 + ts * part;
      l_t1 = min(s.x1, l_t + part);
      if (l_t >= l_t1) continue;
      if (page_tiles == 0) {
        l_entry = 2 * l_t;
      } else {
        l_entry = l_t / page_tiles;
        l_sub = l_t - l_entry * page_tiles;
      }
      l_win = l_entry;
      read_entry(l_win + lane, w_page, w_col);
      read_entry(l_win + 32 + lane, n_page, n_col);
    }
    const uint8_t* const base = a.k_cache + static_cast<int64_t>(l_h) * a.head_stride +
                                static_cast<int64_t>(sub) * a.token_stride + unit * 16;
    const int64_t to_values = a.v_cache - a.k_cache;
#pragma unroll
    for (int q = 0; q < kTiles; ++q, ++l_t) {
      const uint32_t stage = ring + slot * kStageBytes + q * kPlace;
      if (l_entry - l_win >= 32) {
        l_win += 32;
        w_page = n_page;
        w_col = n_col;
        read_entry(l_win + 32 + lane, n_page, n_col);
      }
      int page0 = __shfl_sync(0xffffffffu, w_page, l_entry - l_win), page1 = page0;
      const int col = a.selected ? __shfl_sync(0xffffffffu, w_col, l_entry - l_win) : l_entry;
      int valid0, valid1;  // tokens of the tile's two octets
      const bool some = l_t < l_t1;
      // A row past the valid ones is still a row of its page (or of page 0): only its size is 0.
      if (page_tiles != 0) {
        const int left = some && page0 >= 0 ? l_len - col * a.page_size - l_sub * kB8Tile : 0;
        const uint8_t* const src = base + static_cast<int64_t>(max(page0, 0)) * a.page_stride +
                                   static_cast<int64_t>(l_sub * kB8Tile) * a.token_stride;
        valid0 = max(0, min(8, left));
        valid1 = max(0, min(8, left - 8));
        const int64_t step = static_cast<int64_t>(kRows) * a.token_stride;
#pragma unroll
        for (int i = 0; i < (2 * kBlocks + HG - 1) / HG; ++i) {
          const int blk = i * HG + hg;
          if (2 * kBlocks % HG == 0 || blk < 2 * kBlocks) {
            const int tensor = blk / kBlocks, j = blk % kBlocks;
            cp_async16(stage + tensor * kTileBytes + row_block<DP>(dst0, j * kRows),
                       src + j * step + (tensor ? to_values : 0), j * kRows + sub < left ? unit_bytes : 0u, policy);
          }
        }
        if (++l_sub == page_tiles) {
          l_sub = 0;
          ++l_entry;
        }
      } else {  // two pages of 8 tokens
        page1 = __shfl_sync(0xffffffffu, w_page, l_entry + 1 - l_win);
        const int col1 = a.selected ? __shfl_sync(0xffffffffu, w_col, l_entry + 1 - l_win) : l_entry + 1;
        valid0 = some && page0 >= 0 ? max(0, min(8, l_len - col * 8)) : 0;
        valid1 = some && page1 >= 0 ? max(0, min(8, l_len - col1 * 8)) : 0;
#pragma unroll
        for (int i = 0; i < (2 * kBlocks + HG - 1) / HG; ++i) {
          const int blk = i * HG + hg;
          if (2 * kBlocks % HG == 0 || blk < 2 * kBlocks) {
            const int tensor = blk / kBlocks, j = blk % kBlocks;
            const bool second = j * kRows >= 8;
            const int in_page = j * kRows & 7;
            const uint8_t* src = base + static_cast<int64_t>(max(second ? page1 : page0, 0)) * a.page_stride +
                                 static_cast<int64_t>(in_page) * a.token_stride + (tensor ? to_values : 0);
            cp_async16(stage + tensor * kTileBytes + row_block<DP>(dst0, j * kRows), src,
                       in_page + sub < (second ? valid1 : valid0) ? unit_bytes : 0u, policy);
          }
        }
        l_entry += 2;
      }
      if (hg == 0 && lane < 5) {  // (k, v) scale of either octet; the valid counts
        const uint32_t meta = stage + 2 * kTileBytes + lane * 4;
        if (lane < 4) {
          const int page = lane < 2 ? page0 : page1;
          const bool there = (lane < 2 ? valid0 : valid1) > 0;
          const float* src = (lane & 1 ? a.v_scale : a.k_scale) +
                             (there ? static_cast<int64_t>(page) * a.num_kv_heads + l_h : 0);
          cp_async4(meta, src, there ? 4u : 0u);
        } else {
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(meta), "r"(valid0 | valid1 << 16) : "memory");
        }
      }
    }
    cp_async_commit();
  };
  const auto team_barrier = [&]() {
    if constexpr (HG == 1) {
      __syncwarp();
    } else {
      named_barrier(kTeamBarrier + team, 32 * HG);
    }
  };
  const auto group_barrier = [&]() {
    if (a.ts == 1) {
      __syncwarp();
    } else {
      named_barrier(kGroupBarrier + grp, 32 * a.ts);
    }
  };

#pragma unroll 1
  for (int i = 0; i < kStages - 1; ++i) issue(i);
  int slot = 0;
  // Where this lane reads: rows g and g + 8 of the keys; rows 2c, 2c + 1, 2c + 8, 2c + 9 of the values.
  const uint32_t k_at = unit_offset<DP>(g, c);
  const uint32_t v_at = DP == 64 ? unit_offset<DP>(2 * c, g >> 1) + (g & 1) * 8 : unit_offset<DP>(2 * c, g);

  Segment s;
  while (cons.next(a, s)) {
    const int h = s.u * a.hb + hb;
    if (h >= a.num_kv_heads) continue;
    const int heads = max(0, min(NH, a.group - hg * NH));  // query heads of this warp
    const int64_t q_row = static_cast<int64_t>(s.b) * a.num_q_heads + h * a.group + hg * NH;

    // Q as the score product's B operand: lane (g, c) holds query head g of each group of 8. The
    // contraction runs over a row's codes in the order in which a lane's 16-byte reads deliver them.
    uint32_t qf[kQRegs ? NT : 1][kSteps][2];
    float q_mul[NT][2];  // scale of the scores of this lane's two heads (2c, 2c + 1)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float v[kSteps][4];
      float top = 0.0f;
      const bool mine = n * 8 + g < heads;
#pragma unroll
      for (int j = 0; j < kSteps / 4; ++j) {
        const int d = (j * 4 + c) * 16;
        uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (mine && d < a.head_dim) {
          const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) +
                                                          (q_row + n * 8 + g) * a.head_dim + d);
          raw[0] = __ldg(p);
          raw[1] = __ldg(p + 1);
        }
        const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 f = a.q_bf16 ? Storage<__nv_bfloat16>::unpack2(w[i]) : Storage<__half>::unpack2(w[i]);
          v[j * 4 + i / 2][(i & 1) * 2] = f.x;
          v[j * 4 + i / 2][(i & 1) * 2 + 1] = f.y;
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // An fp16 q goes in as it is. A bf16 q is divided by the 2^e that puts its largest element between 2^14 and
      // 2^15, so that f16's bits reach 2^-31 of it without loss; e is kept to where 2^-e is a normal number too.
      const int e = a.q_bf16 ? max(-126, min(113, static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14)) : 0;
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * a.scale_log2;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        qf[kQRegs ? n : 0][i][0] = Storage<__half>::pack2(v[i][0] * down, v[i][1] * down);
        qf[kQRegs ? n : 0][i][1] = Storage<__half>::pack2(v[i][2] * down, v[i][3] * down);
      }
      if constexpr (!kQRegs) {
#pragma unroll
        for (int i = 0; i < kSteps / 2; ++i) {
          sts128(q_at + (n * (kSteps / 2) + i) * 512,
                 make_uint4(qf[0][2 * i][0], qf[0][2 * i][1], qf[0][2 * i + 1][0], qf[0][2 * i + 1][1]));
        }
      }
      q_mul[n][0] = __shfl_sync(0xffffffffu, up, 8 * c);
      q_mul[n][1] = __shfl_sync(0xffffffffu, up, 8 * c + 4);
    }

    float acc[NT][kHalves][kM][4];
    float m[NT][2], l[NT][2];
    float per[NT][2];              // 1 / w: acc is in units of w
    float most_per = 1.0f / kLeastWeight;  // the largest of this lane's
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = kNoMax;
      per[n][0] = per[n][1] = 1.0f / kLeastWeight;
      l[n][0] = l[n][1] = 0.0f;
#pragma unroll
      for (int f = 0; f < kHalves; ++f)
#pragma unroll
        for (int i = 0; i < kM; ++i) acc[n][f][i][0] = acc[n][f][i][1] = acc[n][f][i][2] = acc[n][f][i][3] = 0.0f;
    }

    const int part = (s.x1 - s.x0 + a.ts - 1) / a.ts;
    const int t0 = s.x0 + ts * part, t1 = min(s.x1, t0 + part);
#pragma unroll 1
    for (int t = t0; t < t1; t += kTiles) {
      cp_async_wait<kStages - 2>();
      team_barrier();
      issue(slot == 0 ? kStages - 1 : slot - 1);
      const uint32_t kt = ring + slot * kStageBytes, vt = kt + kTileBytes, meta = vt + kTileBytes;
      slot = slot + 1 == kStages ? 0 : slot + 1;

      // S = K.Q^T: rows (tokens) g and g + 8, columns (heads) 2c and 2c + 1.
      float sc[kTiles][NT][4];
#pragma unroll
      for (int q = 0; q < kTiles; ++q)
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[q][n][0] = sc[q][n][1] = sc[q][n][2] = sc[q][n][3] = 0.0f;
#pragma unroll
      for (int j = 0; j < kSteps / 4; ++j) {
        uint4 k0[kTiles], k1[kTiles];
#pragma unroll
        for (int q = 0; q < kTiles; ++q) {
          const uint32_t at = kt + q * kPlace + (k_at ^ ((j & 1) * 64)) + (j >> 1) * 128;
          k0[q] = lds128(at);
          k1[q] = lds128(at + 8 * DP);
        }
        uint4 qs[NT];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (!kQRegs) {
            if (i % 2 == 0) {
#pragma unroll
              for (int n = 0; n < NT; ++n) qs[n] = lds128(q_at + (n * (kSteps / 2) + j * 2 + i / 2) * 512);
            }
          }
#pragma unroll
          for (int q = 0; q < kTiles; ++q) {
            const uint32_t w0 = i == 0 ? k0[q].x : i == 1 ? k0[q].y : i == 2 ? k0[q].z : k0[q].w;
            const uint32_t w1 = i == 0 ? k1[q].x : i == 1 ? k1[q].y : i == 2 ? k1[q].z : k1[q].w;
            uint32_t a0, a1, a2, a3;
            widen<Code>(w0, a0, a2);
            widen<Code>(w1, a1, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if constexpr (kQRegs) {
                Mma<__half>::run(sc[q][n], a0, a1, a2, a3, qf[n][j * 4 + i][0], qf[n][j * 4 + i][1]);
              } else {
                Mma<__half>::run(sc[q][n], a0, a1, a2, a3, i % 2 ? qs[n].z : qs[n].x, i % 2 ? qs[n].w : qs[n].y);
              }
            }
          }
        }
      }

      float ks[kTiles][2], vs[kTiles][2];  // scales of the octets
      bool there[kTiles][2];               // rows g and g + 8 within the length
      float v_top = 0.0f;
#pragma unroll
      for (int q = 0; q < kTiles; ++q) {
        const uint4 v = lds128(meta + q * kPlace);
        ks[q][0] = __uint_as_float(v.x), vs[q][0] = __uint_as_float(v.y);
        ks[q][1] = __uint_as_float(v.z), vs[q][1] = __uint_as_float(v.w);
        v_top = fmaxf(v_top, fmaxf(fabsf(vs[q][0]), fabsf(vs[q][1])));
        const uint32_t valid = lds32(meta + q * kPlace + 16);
        there[q][0] = g < static_cast<int>(valid & 0xffffu);
        there[q][1] = g < static_cast<int>(valid >> 16);
      }

      // Scores less the running maximum, in base 2; rows past the end at -infinity.
      float x[kTiles][NT][4];
      float most = -INFINITY;
#pragma unroll
      for (int q = 0; q < kTiles; ++q)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = fmaf(sc[q][n][e], q_mul[n][e & 1] * ks[q][e >> 1], -m[n][e & 1]);
            x[q][n][e] = there[q][e >> 1] ? v : -INFINITY;
            most = fmaxf(most, x[q][n][e]);
          }
      if (__any_sync(0xffffffffu, most > kRaiseBy || v_top * most_per > kWeightRange)) {
        most_per = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = -INFINITY;
#pragma unroll
            for (int q = 0; q < kTiles; ++q)
#pragma unroll
              for (int o = 0; o < 2; ++o) {
                x[q][n][2 * o + e] = there[q][o] ? sc[q][n][2 * o + e] * (q_mul[n][e] * ks[q][o]) : -INFINITY;
                top = fmaxf(top, x[q][n][2 * o + e]);
              }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float next = fmaxf(m[n][e], top);
            const float f = exp2_fast(m[n][e] - next);
            m[n][e] = next;
            float heaviest = reciprocal_of_power(per[n][e]) * f;
            const float before = heaviest;
#pragma unroll
            for (int q = 0; q < kTiles; ++q)
#pragma unroll
              for (int o = 0; o < 2; ++o) {
                x[q][n][2 * o + e] -= next;
                heaviest = fmaxf(heaviest, exp2_fast(x[q][n][2 * o + e]) * fabsf(vs[q][o]));
              }
            heaviest = fmaxf(heaviest, __shfl_xor_sync(0xffffffffu, heaviest, 4));
            heaviest = fmaxf(heaviest, __shfl_xor_sync(0xffffffffu, heaviest, 8));
            heaviest = fmaxf(heaviest, __shfl_xor_sync(0xffffffffu, heaviest, 16));
            per[n][e] = reciprocal_of_power(weight_unit(heaviest));
            most_per = fmaxf(most_per, per[n][e]);
            const float k = before * per[n][e];  // below 2
            l[n][e] *= f;
#pragma unroll
            for (int y = 0; y < kHalves; ++y)
#pragma unroll
              for (int i = 0; i < kM; ++i) {
                acc[n][y][i][e] *= k;
                acc[n][y][i][2 + e] *= k;
              }
          }
        }
      }

      // P^T as the value product's B operand.
      uint32_t p0[kTiles][NT], p1[kTiles][NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int q = 0; q < kTiles; ++q) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[e] = exp2_fast(x[q][n][e]);
            l[n][e & 1] += p[e];
            p[e] *= vs[q][e >> 1] * per[n][e & 1];
          }
          p0[q][n] = movmatrix_trans(Storage<__half>::pack2(p[0], p[1]));
          p1[q][n] = movmatrix_trans(Storage<__half>::pack2(p[2], p[3]));
        }
      }

      // O^T += V^T.P^T: a lane reads the same channels of tokens 2c, 2c + 1, 2c + 8, 2c + 9 and pairs
      // tokens bytewise before widening; rows g and g + 8 of product i are channels 2i and 2i + 1 of
      // the lane's unit.
#pragma unroll
      for (int y = 0; y < kHalves; ++y) {
#pragma unroll
        for (int q = 0; q < kTiles; ++q) {
          constexpr int kWords = DP == 64 ? 2 : 4;
          constexpr uint32_t kNext = unit_offset<DP>(1, 0) & 127;  // the permutation's change from row 2c to 2c + 1
          uint32_t w[4][kWords];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t at = vt + q * kPlace + (k & 1 ? (v_at ^ kNext) + (DP == 64 ? 0 : DP) : v_at) +
                                (k >> 1) * 8 * DP + y * 128;
            if constexpr (DP == 64) {
              const uint2 u = lds64(at);
              w[k][0] = u.x, w[k][1] = u.y;
            } else {
              const uint4 u = lds128(at);
              w[k][0] = u.x, w[k][1] = u.y, w[k][2] = u.z, w[k][3] = u.w;
            }
          }
#pragma unroll
          for (int i = 0; i < kM; ++i) {
            const uint32_t sel = i & 1 ? 0x7362u : 0x5140u;
            uint32_t a0, a1, a2, a3;
            widen<Code>(__byte_perm(w[0][i / 2], w[1][i / 2], sel), a0, a1);
            widen<Code>(__byte_perm(w[2][i / 2], w[3][i / 2], sel), a2, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n) Mma<__half>::run(acc[n][y][i], a0, a1, a2, a3, p0[q][n], p1[q][n]);
          }
        }
      }
    }

    // ---- end of the segment: this warp's state, values in units of 1
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 4);
        l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 8);
        l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 16);
      }
#pragma unroll
      for (int y = 0; y < kHalves; ++y)
#pragma unroll
        for (int i = 0; i < kM; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][y][i][e] *= reciprocal_of_power(per[n][e & 1]);
    }
    // Join the TS parts: the upper half hands its state to the lower half, fragment by fragment, half
    // of the outputs of 8 query heads at a time.
    for (int half = a.ts >> 1; half > 0; half >>= 1) {
      float* const box = joint + ((grp * (a.ts >> 1) + (ts % half)) * box_floats(DP)) * 32 + lane;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float mine[2], other[2];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          if (ts >= half && ts < 2 * half) {
            int k = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              box[32 * k++] = m[n][e];
              box[32 * k++] = l[n][e];
            }
#pragma unroll
            for (int y = 0; y < kHalves; ++y)
#pragma unroll
              for (int i = 0; i < kM / 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) box[32 * k++] = acc[n][y][hf * (kM / 2) + i][e];
          }
          group_barrier();
          if (ts < half) {
            int k = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float om = box[32 * k++], ol = box[32 * k++];
              if (hf == 0) {
                const float next = fmaxf(m[n][e], om);
                mine[e] = exp2_fast(m[n][e] - next);
                other[e] = exp2_fast(om - next);
                m[n][e] = next;
                l[n][e] = l[n][e] * mine[e] + ol * other[e];
              }
            }
#pragma unroll
            for (int y = 0; y < kHalves; ++y)
#pragma unroll
              for (int i = 0; i < kM / 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  float& v = acc[n][y][hf * (kM / 2) + i][e];
                  v = v * mine[e & 1] + box[32 * k++] * other[e & 1];
                }
          }
          group_barrier();  // the boxes are free again
        }
      }
    }

    const int64_t row_start = piece * blockIdx.x + s.start;
    const int64_t c_first = row_start / piece;
    const int chunks = static_cast<int>((row_start + s.tiles - 1) / piece - c_first) + 1;
    const auto store_out = [&](int64_t row, int d, float v0, float v1, float v2, float v3) {
      uint2 w;
      if (a.q_bf16) {
        w = make_uint2(Storage<__nv_bfloat16>::pack2(v0, v1), Storage<__nv_bfloat16>::pack2(v2, v3));
      } else {
        w = make_uint2(Storage<__half>::pack2(v0, v1), Storage<__half>::pack2(v2, v3));
      }
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + row * a.head_dim + d) = w;
    };
    const auto slot_rows = [&](int64_t chunk) {  // first row of a chunk's partial state
      const int64_t sl = (c_first + chunk) * 2 + (chunk == 0 ? 1 : 0);
      return (sl * groups + grp) * NH;
    };
    if (ts == 0) {
      // f(head of this warp, channel, 4 values) over the lane's values, four channels at a time.
      const auto for_values = [&](auto&& f) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = n * 8 + 2 * c + e;
            if (r >= heads) continue;
#pragma unroll
            for (int y = 0; y < kHalves; ++y)
#pragma unroll
              for (int i = 0; i < kM; i += 2) {
                const int d = y * 128 + g * (2 * kM) + 2 * i;
                if (d < a.head_dim) f(r, n, e, d, acc[n][y][i][e], acc[n][y][i][2 + e], acc[n][y][i + 1][e], acc[n][y][i + 1][2 + e]);
              }
          }
      };
      if (chunks == 1) {
        for_values([&](int r, int n, int e, int d, float v0, float v1, float v2, float v3) {
          const float f = l[n][e] != 0.0f ? 1.0f / l[n][e] : 0.0f;
          store_out(q_row + r, d, v0 * f, v1 * f, v2 * f, v3 * f);
        });
      } else {
        const int64_t row = slot_rows(static_cast<int64_t>(blockIdx.x) - c_first);
        for_values([&](int r, int, int, int d, float v0, float v1, float v2, float v3) {
          *reinterpret_cast<float4*>(a.part_o + (row + r) * DP + d) = make_float4(v0, v1, v2, v3);
        });
        if (g == 0) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int r = n * 8 + 2 * c + e;
              if (r < heads) a.part_ml[row + r] = make_float2(m[n][e], l[n][e]);
            }
        }
        __syncwarp();
        if (lane == 0) {
          uint32_t* counter = a.sync + 1 + (static_cast<int64_t>(s.b) * a.num_kv_heads + h) * HG + hg;
          const uint32_t old = atom_add_acq_rel_gpu(counter, 1);
          const bool last = old == static_cast<uint32_t>(chunks - 1);
          if (last) *counter = 0;
          s_last[grp] = last;
        }
      }
    }
    if (chunks > 1) {
      group_barrier();
      if (s_last[grp]) {
        // The group's threads share out (head, 4 channels). Chunks in order, eight loads in flight.
        constexpr int kAhead = 8;
        const int quads = a.head_dim / 4;
        for (int i = ts * 32 + lane; i < heads * quads; i += 32 * a.ts) {
          const int r = i / quads, d = (i - r * quads) * 4;
          float top = kNoMax, sum = 0.0f;
          float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (int k0 = 0; k0 < chunks; k0 += kAhead) {
            float2 ml[kAhead];
            float4 v[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
              ml[k] = make_float2(kNoMax, 0.0f);
              v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              if (k0 + k < chunks) {
                const int64_t row = slot_rows(k0 + k) + r;
                ml[k] = __ldcg(&a.part_ml[row]);
                v[k] = __ldcg(reinterpret_cast<const float4*>(a.part_o + row * DP + d));
              }
            }
            float next = top;
#pragma unroll
            for (int k = 0; k < kAhead; ++k) next = fmaxf(next, ml[k].x);
            const float f = exp2_fast(top - next);
            top = next;
            sum *= f;
            o.x *= f, o.y *= f, o.z *= f, o.w *= f;
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
              const float w = exp2_fast(ml[k].x - top);
              sum = fmaf(w, ml[k].y, sum);
              o.x = fmaf(w, v[k].x, o.x);
              o.y = fmaf(w, v[k].y, o.y);
              o.z = fmaf(w, v[k].z, o.z);
              o.w = fmaf(w, v[k].w, o.w);
            }
          }
          const float f = sum != 0.0f ? 1.0f / sum : 0.0f;
          store_out(q_row + r, d, o.x * f, o.y * f, o.z * f, o.w * f);
        }
      }
      group_barrier();  // s_last may be written again
    }
  }
  cp_async_wait<0>();
}

// ------------------------------------------------------------------------- host side

struct Block8Plan {
  int dp, nt, hg, hb, ts, units, min_tiles, row_charge, grid;
  size_t smem, partial_bytes, sync_bytes;
};

// False: the shape is not supported.
bool make_block8_plan(int batch, int hq, int hkv, int d, int page, int max_pages, int selected, Block8Plan& p) {
  if (batch < 0 || hkv <= 0 || hq <= 0 || hq % hkv != 0 || d <= 0 || d % 16 != 0 || d > 256 || page <= 0 ||
      (page != 8 && page % 16 != 0) || max_pages < 0 || selected < 0 ||
      static_cast<int64_t>(max_pages) * page > INT32_MAX - 64 || static_cast<int64_t>(selected) * page > INT32_MAX - 64) {
    return false;
  }
  const int group = hq / hkv;
  p.dp = d <= 64 ? 64 : d <= 128 ? 128 : 256;
  if (group > (p.dp == 256 ? 64 : 128)) return false;
  p.nt = group <= 8 || p.dp == 256 ? 1 : group <= 16 || p.dp == 128 ? 2 : 4;
  p.hg = 1;
  while (p.hg * 8 * p.nt < group) p.hg *= 2;
  const int teams = kB8Warps / p.hg;
  const int ctas = sm_count();
  const int64_t tokens = selected > 0 ? static_cast<int64_t>(selected) * page : static_cast<int64_t>(max_pages) * page;
  const int64_t tiles = std::max<int64_t>(1, (tokens + kB8Tile - 1) / kB8Tile);
  // As many heads side by side as fill the CTA, halved while the rows are under a fifth of the CTAs: a
  // row that many CTAs share is joined from as many states. Measured (us, 32/8 heads of 128; HB 8, 4,
  // 2, 1): batch 1 x 32768 tokens 78, 35, 25.6, 23.4; 8 x 4096 30.1, 24.1, 22.9, 24.6; 16 x 2048 27.0,
  // 22.5, 24.2, 27.2; 64 x 4096 93.9, 93.9, 98.6, 108.
  p.hb = 1;
  while (2 * p.hb <= teams && 2 * p.hb <= hkv) p.hb *= 2;
  while (p.hb > 1 && batch * static_cast<int64_t>((hkv + p.hb - 1) / p.hb) * 5 < ctas) p.hb /= 2;
  p.ts = teams / p.hb;
  p.units = (hkv + p.hb - 1) / p.hb;
  const int least = std::max(4, step_tiles(p.dp, p.nt) * p.ts);
  // Starting a row costs a CTA a few microseconds whatever its heads, 8 tiles of every one of its TS
  // parts; a short row, split or not, is not worth charging more than half of itself. No piece, and no row's
  // charge, is less than a step of every warp: two short rows in one CTA, or a chunk that leaves half of the
  // warps idle, cost more than the CTAs saved (us without the rule and with it: 1 x 16 tokens 13.9, 8.4; 1 x 256
  // 10.8, 9.6; 8 x 1024 of 32/1 heads 19.8, 17.2).
  p.row_charge = static_cast<int>(std::min<int64_t>(8 * p.ts, std::max<int64_t>(least, tiles / 2)));
  p.min_tiles = least;
  const int64_t most = batch * static_cast<int64_t>(p.units) * (tiles + p.row_charge);
  p.grid = static_cast<int>(std::min<int64_t>(ctas, std::max<int64_t>(1, (most + p.min_tiles - 1) / p.min_tiles)));
  if (most / p.grid >= INT32_MAX - p.min_tiles) return false;  // positions within a piece are 32 bits
  const int stages = ring_stages(p.dp, p.nt, p.hg);
  p.smem = static_cast<size_t>(kB8Warps / p.hg) * stages * step_tiles(p.dp, p.nt) * (2 * kB8Tile * p.dp + kB8Meta) +
           static_cast<size_t>(kB8Warps) * query_bytes(p.dp, p.nt);
  if (p.ts > 1) p.smem += static_cast<size_t>(kB8Warps / 2) * box_floats(p.dp) * 32 * sizeof(float);
  const size_t rows = static_cast<size_t>(p.grid) * 2 * (kB8Warps / p.ts) * 8 * p.nt;
  p.partial_bytes = rows * (p.dp * sizeof(float) + sizeof(float2));
  p.sync_bytes = (1 + static_cast<size_t>(batch) * hkv * p.hg) * sizeof(uint32_t);
  return true;
}

bool decode_pdl() {  // the same switch as the other decode kernels'
  static const bool on = env_switch_on("KL_DECODE_PDL");
  return on;
}

template <typename Code, int DP, int NT, int HG>
cudaError_t launch_block8(const Block8Args& a, const Block8Plan& p, cudaStream_t st) {
  const auto kernel = decode_block8_kernel<Code, DP, NT, HG>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_shared_memory(kernel, kMaxShared, done);
  if (e != cudaSuccess) return e;
  return launch_kernel(decode_pdl(), kernel, dim3(static_cast<unsigned>(p.grid)), dim3(kB8Threads), p.smem, st, a);
}

template <typename Code, int DP, int NT>
cudaError_t launch_heads(const Block8Args& a, const Block8Plan& p, cudaStream_t st) {
  switch (p.hg) {
    case 1: return launch_block8<Code, DP, NT, 1>(a, p, st);
    case 2: return launch_block8<Code, DP, NT, 2>(a, p, st);
    case 4: return launch_block8<Code, DP, NT, 4>(a, p, st);
    default: return launch_block8<Code, DP, NT, 8>(a, p, st);
  }
}

template <typename Code>
cudaError_t launch_code(const Block8Args& a, const Block8Plan& p, cudaStream_t st) {
  if (p.dp == 256) return launch_heads<Code, 256, 1>(a, p, st);
  if (p.nt == 1) return p.dp == 64 ? launch_block8<Code, 64, 1, 1>(a, p, st) : launch_block8<Code, 128, 1, 1>(a, p, st);
  if (p.dp == 128) return launch_heads<Code, 128, 2>(a, p, st);
  if (p.nt == 2) return launch_block8<Code, 64, 2, 1>(a, p, st);
  switch (p.hg) {  // up to 128 query heads are four warps of 32
    case 1: return launch_block8<Code, 64, 4, 1>(a, p, st);
    case 2: return launch_block8<Code, 64, 4, 2>(a, p, st);
    default: return launch_block8<Code, 64, 4, 4>(a, p, st);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace block8_decode
}  // namespace klb

extern "C" int kl_paged_decode_block8_workspace_size(int batch, int num_q_heads, int num_kv_heads, int head_dim,
                                                     int page_size, int max_pages_per_seq, int num_selected,
                                                     size_t* partial_bytes, size_t* sync_bytes) {
  if (!partial_bytes || !sync_bytes) return static_cast<int>(cudaErrorInvalidValue);
  *partial_bytes = 0;
  *sync_bytes = sizeof(uint32_t);
  if (batch == 0) return 0;
  klb::block8_decode::Block8Plan p;
  if (!klb::block8_decode::make_block8_plan(batch, num_q_heads, num_kv_heads, head_dim, page_size, max_pages_per_seq, num_selected, p)) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  *partial_bytes = p.partial_bytes;
  *sync_bytes = p.sync_bytes;
  return 0;
}

extern "C" int kl_paged_decode_block8(int dtype, int code_type, void* out, const void* q, const void* k_cache,
                                      const void* v_cache, const float* k_scale, const float* v_scale,
                                      const int32_t* block_table, const int32_t* seq_lens, const int32_t* selected,
                                      int batch, int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                                      int64_t page_stride, int64_t token_stride, int64_t head_stride,
                                      int64_t block_table_stride, int max_pages_per_seq, int64_t num_pages,
                                      int num_selected, float scale, void* partials, size_t partial_bytes, void* sync,
                                      size_t sync_bytes, void* stream) {
  using namespace klb;
  using namespace klb::block8_decode;
  constexpr int kInvalid = static_cast<int>(cudaErrorInvalidValue);
  if (batch == 0) return 0;
  if ((dtype != KL_FLOAT16 && dtype != KL_BFLOAT16) || (code_type != KL_CODE_E4M3 && code_type != KL_CODE_INT8) ||
      !out || !q || !k_cache || !v_cache || !k_scale || !v_scale || !block_table || !seq_lens || !sync ||
      num_pages < 0 || num_pages > INT32_MAX || block_table_stride < max_pages_per_seq ||
      (selected == nullptr) != (num_selected == 0) || page_stride < 0 || token_stride < 0 || head_stride < 0 || page_stride > INT32_MAX ||
      token_stride > INT32_MAX || head_stride > INT32_MAX || page_stride % 16 != 0 || token_stride % 16 != 0 || head_stride % 16 != 0 || !aligned16(k_cache) ||
      !aligned16(v_cache) || !aligned16(q) || !aligned16(out)) {
    return kInvalid;
  }
  Block8Plan p;
  if (!make_block8_plan(batch, num_q_heads, num_kv_heads, head_dim, page_size, max_pages_per_seq, num_selected, p)) {
    return kInvalid;
  }
  if (partial_bytes < p.partial_bytes || sync_bytes < p.sync_bytes || !partials || !aligned16(partials)) return kInvalid;
  Block8Args a{};
  a.out = out;
  a.q = q;
  a.k_cache = static_cast<const uint8_t*>(k_cache);
  a.v_cache = static_cast<const uint8_t*>(v_cache);
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.block_table = block_table;
  a.seq_lens = seq_lens;
  a.selected = selected;
  a.page_stride = static_cast<int32_t>(page_stride);
  a.token_stride = static_cast<int32_t>(token_stride);
  a.head_stride = static_cast<int32_t>(head_stride);
  a.bt_stride = block_table_stride;
  a.num_pages = num_pages;
  a.batch = batch;
  a.num_q_heads = num_q_heads;
  a.num_kv_heads = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.head_dim = head_dim;
  a.page_size = page_size;
  a.max_pages = max_pages_per_seq;
  a.num_selected = num_selected;
  a.q_bf16 = dtype == KL_BFLOAT16;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.hb = p.hb;
  a.ts = p.ts;
  a.units = p.units;
  a.min_tiles = p.min_tiles;
  a.row_charge = p.row_charge;
  a.sync = static_cast<uint32_t*>(sync);
  a.part_o = static_cast<float*>(partials);
  const size_t rows = static_cast<size_t>(p.grid) * 2 * (kB8Warps / p.ts) * 8 * p.nt;
  a.part_ml = reinterpret_cast<float2*>(a.part_o + rows * p.dp);
  const auto st = static_cast<cudaStream_t>(stream);
  return static_cast<int>(code_type == KL_CODE_E4M3 ? launch_code<E4m3Code>(a, p, st) : launch_code<Int8Code>(a, p, st));
}
