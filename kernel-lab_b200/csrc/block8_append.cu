// Append to a paged cache held in 8 bits with a scale for each page and KV head, for sm_100a: one
// new token a sequence, or a prompt's tokens.
//
// The work falls into units of one page, KV head and tensor: the largest magnitude of the page's
// new elements gives the scale, so a unit is a reduction and then an elementwise pass over the same
// elements. A team of one warp (pages of up to 4096 elements a head) or of four warps takes a unit
// and copies its new elements to shared memory, all in flight at once and without registers, so that
// it reads them once; larger pages re-read theirs from L2. HBM-bound for prompts (the new rows in, half
// or a quarter of their bytes out), latency-bound for single tokens, where the chain is indptr / position,
// block-table entry, new row.
// Measured: 33.4k prompt tokens of 8 heads of 128, e4m3 with bounds, 42.0 us (5.0 TB/s of the 210 MB it has to
// move, 0.76 of the copy peak); 37 int8 chunks of up to 257 tokens 21 us; one token of each of 64 sequences
// 4.9 us. A window that holds many short sequences takes them one after another: a chunk of 4000 tokens among 63
// single ones 48 us, alone 7.6.
//
// No host knows where pages begin in the ragged rows, so a team takes a window of the flattened new
// tokens and looks for the tokens in it that are the first of their sequence in a page; the window is
// one token when sequences bring one each, else one page's length, or up to four pages' in a large call:
// the sequence is found once for them, and while a page filled whole is quantised the next one's rows are
// on their way (one page at a time 51.4 us, two 46, four 42.0; eight 49.6, too few teams). The parts of
// a page lie side by side in the grid, so that neighbouring heads are read and written together (1.1 us).
//
// Bounds: rounding is monotone, so the least and largest code of a channel are the codes of the
// least and largest scaled element, and only those two are rounded; they are combined over the
// team's tokens through shared memory.
//
// 16-bit elements are compared two at a time as they are (packed maximum of magnitudes, packed
// extremes), which is exact; only a unit that holds a NaN or an infinity takes the element-wise path.
#include <algorithm>
#include <cfloat>
#include <cstdint>
#include <type_traits>

#include <cuda_runtime.h>

#include "block8.cuh"
#include "kernel_lab_b200_block8.h"

namespace klb {
// A namespace with a name: an unnamed one's symbols carry a hash of the file's text, and with them the
// compiler's register allocation would change with a comment.
namespace block8_append {

constexpr int kBlock8AppendThreads = 128;
constexpr int kMaxGridY = 65535;
// Blocks an SM that the registers are held to. With 4, 5, 6: 33.4k prompt tokens 44.9, 42.1, 42.7 us; 37 int8
// chunks 21.2, 21.2, 21.9 us (whose shared memory, 16 packs a lane, allows 4; 6 spills).
constexpr int kAppendBlocks = 5;

struct Block8AppendArgs {
  uint8_t* k_cache;
  uint8_t* v_cache;
  float* k_scale;
  float* v_scale;
  int8_t* k_bounds;        // may be null
  const void* k_new;
  const void* v_new;
  const int32_t* block_table;
  const int32_t* positions;
  const int32_t* indptr;   // null: one token a sequence
  uint32_t* status;        // may be null
  int64_t page_stride, token_stride, head_stride;  // bytes (= elements)
  int64_t bt_stride;
  int64_t new_stride;      // elements between consecutive new rows
  int64_t num_pages;
  int64_t tokens;
  int batch, num_kv_heads, head_dim, page_size, max_pages;
  int window;              // new tokens a team looks at
  int across, down;        // channel units (of VEC) side by side in a team, tokens beside them
  uint32_t per_across;     // 65536 / across + 1: thread / across without a division
  uint32_t per_down;       // 2^32 / down + 1 (0 where down is 1): tokens / down likewise
  int keep;                // packs a thread can keep in shared memory
};

// Last b with indptr[b] <= t, by all lanes of a warp (32 samples a step).
__device__ __forceinline__ int sequence_of(const int32_t* indptr, int batch, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = batch;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int i = lo + lane * step;
    const unsigned le = __ballot_sync(0xffffffffu, lane * step < n && indptr[i] <= t);
    const int k = le ? 31 - __clz(le) : 0;
    n = min(step, n - k * step);
    lo += k * step;
  }
  return lo;
}

// Which sequence a new row belongs to, its rows and its first position. For up to 127 sequences each
// warp reads the whole of indptr and positions at once (one latency, not one for each step of a search).
struct Sequences {
  static constexpr int kWords = 4;
  int ptr[kWords], pos[kWords];
  bool whole;
  __device__ __forceinline__ void read(const Block8AppendArgs& a) {
    whole = a.indptr != nullptr && a.batch < 32 * kWords;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      const int i = 32 * k + lane;
      ptr[k] = whole && i <= a.batch ? a.indptr[i] : INT32_MAX;
      pos[k] = whole && i < a.batch ? a.positions[i] : -1;
    }
  }
  __device__ __forceinline__ int pick(const int (&v)[kWords], int i) const {
    const int w = i >> 5;
    const int got = w == 0 ? v[0] : w == 1 ? v[1] : w == 2 ? v[2] : v[3];
    return __shfl_sync(0xffffffffu, got, i & 31);
  }
  __device__ __forceinline__ void find(const Block8AppendArgs& a, int t, int& b, int& begin, int& end, int& start) const {
    if (whole) {
      int count = 0;
#pragma unroll
      for (int k = 0; k < kWords; ++k) count += __popc(__ballot_sync(0xffffffffu, ptr[k] <= t));
      b = max(0, min(count, a.batch) - 1);
      begin = pick(ptr, b);
      end = pick(ptr, b + 1);
      start = pick(pos, b);
    } else if (a.indptr) {
      b = sequence_of(a.indptr, a.batch, t);
      begin = a.indptr[b];
      end = a.indptr[b + 1];
      start = a.positions[b];
    } else {
      b = t;
      begin = t;
      end = t + 1;
      start = a.positions[b];
    }
    end = min(end, static_cast<int>(a.tokens));
  }
};

// VEC consecutive elements of a new row (VEC 8: 16-byte aligned), as loaded.
template <typename E, int VEC>
struct NewPack {
  alignas(VEC == 8 ? 16 : sizeof(E)) E v[VEC];
  __device__ __forceinline__ void load(const E* p) {
    if constexpr (VEC == 8) {
      constexpr int kWords = sizeof(E) * 8 / 16;
#pragma unroll
      for (int i = 0; i < kWords; ++i) reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      v[0] = *p;
    }
  }
  __device__ __forceinline__ void unpack(float (&f)[VEC]) const {
    if constexpr (VEC == 8 && sizeof(E) == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 p = Storage<E>::unpack2(reinterpret_cast<const uint32_t*>(v)[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = Storage<E>::load(v[j]);
    }
  }
};

// Extremes of packs element by element and the largest magnitude, in the element type (exact). NaN
// and infinities show in the magnitude (not finite), after which the extremes are not used.
template <typename E, int VEC>
struct PackExtremes {
  static constexpr bool kPairs = VEC == 8 && sizeof(E) == 2;
  using Pair = std::conditional_t<std::is_same_v<E, __half>, __half2, __nv_bfloat162>;
  static constexpr int kN = kPairs ? 4 : VEC;
  using Unit = std::conditional_t<kPairs, Pair, float>;
  Unit lo[kN], hi[kN];
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if constexpr (std::is_same_v<Unit, __half2>) {
        lo[i] = __half2half2(__ushort_as_half(0x7c00)), hi[i] = __half2half2(__ushort_as_half(0xfc00));
      } else if constexpr (std::is_same_v<Unit, __nv_bfloat162>) {
        lo[i] = __bfloat162bfloat162(__ushort_as_bfloat16(0x7f80));
        hi[i] = __bfloat162bfloat162(__ushort_as_bfloat16(0xff80));
      } else {
        lo[i] = INFINITY, hi[i] = -INFINITY;
      }
    }
  }
  __device__ __forceinline__ void add(const NewPack<E, VEC>& p) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if constexpr (kPairs) {
        const Unit u = reinterpret_cast<const Unit*>(p.v)[i];
        lo[i] = __hmin2(lo[i], u);
        hi[i] = __hmax2(hi[i], u);
      } else {
        const float u = Storage<E>::load(p.v[i]);
        lo[i] = fminf(lo[i], u);
        hi[i] = fmaxf(hi[i], u);
      }
    }
  }
  // With the extremes of the lane `o` away.
  __device__ __forceinline__ void combine_lanes(int o) {
    static_assert(kPairs);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const uint32_t l = __shfl_xor_sync(0xffffffffu, reinterpret_cast<const uint32_t&>(lo[i]), o);
      const uint32_t h = __shfl_xor_sync(0xffffffffu, reinterpret_cast<const uint32_t&>(hi[i]), o);
      lo[i] = __hmin2(lo[i], reinterpret_cast<const Unit&>(l));
      hi[i] = __hmax2(hi[i], reinterpret_cast<const Unit&>(h));
    }
  }
  __device__ __forceinline__ void get(float (&l)[VEC], float (&h)[VEC]) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if constexpr (kPairs) {
        const float2 a = Storage<E>::unpack2(reinterpret_cast<const uint32_t*>(lo)[i]);
        const float2 b = Storage<E>::unpack2(reinterpret_cast<const uint32_t*>(hi)[i]);
        l[2 * i] = a.x, l[2 * i + 1] = a.y;
        h[2 * i] = b.x, h[2 * i + 1] = b.y;
      } else {
        l[i] = lo[i], h[i] = hi[i];
      }
    }
  }
};

template <typename E, int VEC>
struct Magnitude {
  using X = PackExtremes<E, VEC>;
  typename X::Unit top;
  __device__ __forceinline__ void reset() {
    if constexpr (X::kPairs) {
      const uint32_t zero = 0;
      top = *reinterpret_cast<const typename X::Unit*>(&zero);
    } else {
      top = 0.0f;
    }
  }
  __device__ __forceinline__ void add(const NewPack<E, VEC>& p) {
#pragma unroll
    for (int i = 0; i < X::kN; ++i) {
      if constexpr (X::kPairs) {
        top = __hmax2_nan(top, __habs2(reinterpret_cast<const typename X::Unit*>(p.v)[i]));
      } else {
        const float f = fabsf(Storage<E>::load(p.v[i]));
        top = f > top || f != f ? f : top;  // NaN stays
      }
    }
  }
  __device__ __forceinline__ float get() const {  // NaN or infinity if an element was
    if constexpr (X::kPairs) {
      const float2 p = Storage<E>::unpack2(*reinterpret_cast<const uint32_t*>(&top));
      return p.x != p.x ? p.x : p.y != p.y ? p.y : fmaxf(p.x, p.y);
    } else {
      return top;
    }
  }
};

template <typename Code, int VEC>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&y)[VEC], bool in_range) {
  if constexpr (VEC == 8) {
    uint2 w;
    if (in_range) {
      w.x = Code::code4_in_range(y[0], y[1], y[2], y[3]);
      w.y = Code::code4_in_range(y[4], y[5], y[6], y[7]);
    } else {
      w.x = Code::code4(y[0], y[1], y[2], y[3]);
      w.y = Code::code4(y[4], y[5], y[6], y[7]);
    }
    *reinterpret_cast<uint2*>(p) = w;
  } else {
    *p = static_cast<uint8_t>(Code::code(y[0]));
  }
}

template <typename Code, int VEC>
__device__ __forceinline__ void load_codes(const uint8_t* p, float (&y)[VEC]) {
  if constexpr (VEC == 8) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[i] = Code::value(w.x >> (8 * i));
      y[4 + i] = Code::value(w.y >> (8 * i));
    }
  } else {
    y[0] = Code::value(*p);
  }
}

// N channels' bounds (UP: the upper ones) of extremes times `by`, as bytes: the code's value in units, outward.
template <typename Code, bool UP, int N>
__device__ __forceinline__ uint32_t bound_codes(const float* x, float by) {
  constexpr float kPerUnit = 1.0f / Code::kBoundUnit;  // a power of two
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float v = Code::value(Code::code(x[j] * by)) * kPerUnit;
    const int r = UP ? __float2int_ru(v) : __float2int_rd(v);
    w |= static_cast<uint32_t>(r & 0xff) << (8 * j);
  }
  return w;
}

// Extremes of scaled elements; NaN counts as 0.
template <int VEC>
struct Extremes {
  float lo[VEC], hi[VEC];
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int j = 0; j < VEC; ++j) lo[j] = FLT_MAX, hi[j] = -FLT_MAX;
  }
  __device__ __forceinline__ void add(const float (&y)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float v = y[j] == y[j] ? y[j] : 0.0f;
      lo[j] = fminf(lo[j], v);
      hi[j] = fmaxf(hi[j], v);
    }
  }
};

// A team of TEAM threads and the unit's units of VEC channels: thread t takes channel unit
// c0 + t % across of the tokens t / across, t / across + down, ...
template <int TEAM>
__device__ __forceinline__ void team_sync() {
  if constexpr (TEAM == 32) __syncwarp(); else __syncthreads();
}

template <typename E, int VEC, int TEAM>
__host__ __device__ constexpr int team_bytes(int keep) {
  const int codes = keep * VEC, extremes = 2 * VEC * static_cast<int>(sizeof(float));
  return TEAM * (keep * static_cast<int>(sizeof(E)) * VEC + (codes > extremes ? codes : extremes));
}

template <int TEAM>
__device__ __forceinline__ bool team_all(bool v) {
  if constexpr (TEAM == 32) return __all_sync(0xffffffffu, v);
  else return __syncthreads_and(v);
}

template <int TEAM>
__device__ __forceinline__ float team_max(float v, float* red) {
  v = warp_allreduce_max(v);
  if constexpr (TEAM > 32) {
    __syncthreads();  // `red` is free
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TEAM / 32; ++w) v = fmaxf(v, red[w]);
  }
  return v;
}

// Eight packs a lane of a page that is filled whole by one call (the bulk of a prompt): straight-line,
// in registers. `staged` holds the lane's packs; `next` is called when they have been read, to ask for the
// next part's in their place. Returns false, with nothing written or asked for, when the page holds a
// NaN or an infinity.
constexpr int kWhole = 8;
template <typename E, typename Code, typename Next>
__device__ __forceinline__ bool append_whole_page(const NewPack<E, 8>* staged, uint8_t* dst, int64_t dst_step,
                                                  float* scale_at, int8_t* bounds, int head_dim, int across,
                                                  Next&& next) {
  using Pack = NewPack<E, 8>;
  Pack p[kWhole];
#pragma unroll
  for (int i = 0; i < kWhole; ++i) p[i].load(staged[i * 32].v);
  Magnitude<E, 8> mag;
  mag.reset();
#pragma unroll
  for (int i = 0; i < kWhole; ++i) mag.add(p[i]);
  float amax = mag.get();
  if (!__all_sync(0xffffffffu, amax <= FLT_MAX)) return false;  // every lane has its packs
  next();
  amax = warp_allreduce_max(amax);
  const float scale = Code::scale_for(amax);
  const float inv = reciprocal_scale(scale);
  const int lane = threadIdx.x & 31;
  if (lane == 0) *scale_at = scale;
#pragma unroll
  for (int i = 0; i < kWhole; ++i, dst += dst_step) {
    float y[8];
    p[i].unpack(y);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] *= inv;
    *reinterpret_cast<uint2*>(dst) = make_uint2(Code::code4_in_range(y[0], y[1], y[2], y[3]),
                                                Code::code4_in_range(y[4], y[5], y[6], y[7]));
  }
  if (bounds) {
    PackExtremes<E, 8> x;
    x.reset();
#pragma unroll
    for (int i = 0; i < kWhole; ++i) x.add(p[i]);
    for (int o = across; o < 32; o <<= 1) x.combine_lanes(o);
    if (lane < across) {
      float lo[8], hi[8];
      x.get(lo, hi);
      uint32_t low[2], high[2];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        low[w] = bound_codes<Code, false, 4>(lo + 4 * w, inv);
        high[w] = bound_codes<Code, true, 4>(hi + 4 * w, inv);
      }
      *reinterpret_cast<uint2*>(bounds + lane * 8) = make_uint2(low[0], low[1]);
      *reinterpret_cast<uint2*>(bounds + head_dim + lane * 8) = make_uint2(high[0], high[1]);
    }
  }
  return true;
}

template <typename E, typename Code, int VEC, int TEAM>
__global__ void __launch_bounds__(kBlock8AppendThreads, kAppendBlocks) kv_append_block8(const Block8AppendArgs a) {
  constexpr int kTeams = kBlock8AppendThreads / TEAM;
  using Pack = NewPack<E, VEC>;
  // Per team: the kept packs [keep][TEAM]; then a page's present codes (VEC bytes a thread and row)
  // and, after those are used, the threads' extremes [2][TEAM * VEC].
  extern __shared__ __align__(16) uint8_t s_dyn[];
  __shared__ float s_red[kBlock8AppendThreads / 32];
  const int team = threadIdx.x / TEAM, tid = threadIdx.x % TEAM;
  Pack* const s_new = reinterpret_cast<Pack*>(s_dyn + team * team_bytes<E, VEC, TEAM>(a.keep));
  uint8_t* const s_codes = reinterpret_cast<uint8_t*>(s_new + a.keep * TEAM);
  float* const s_lo = reinterpret_cast<float*>(s_codes);
  float* const s_hi = s_lo + TEAM * VEC;
  wait_prior_grid();
  allow_next_grid();
  const int part = blockIdx.x * kTeams + team;  // 2 * head + (0: keys, 1: values)
  if (part >= 2 * a.num_kv_heads) return;       // whole warps; with TEAM 128 there is one team a block
  const int64_t window = static_cast<int64_t>(blockIdx.z) * kMaxGridY + blockIdx.y;
  if (window * a.window >= a.tokens) return;
  const int h = part >> 1;
  const bool keys = (part & 1) == 0;
  const bool bounds = keys && a.k_bounds != nullptr;

  const int units = a.head_dim / VEC;
  const int across = a.across, down = a.down;
  const int my_tok = static_cast<int>((static_cast<uint32_t>(tid) * a.per_across) >> 16);
  const int my_unit = tid - my_tok * across;
  const bool active = my_tok < down;
  const int64_t src_step = down * a.new_stride, dst_step = down * a.token_stride;
  const auto barrier = [] { team_sync<TEAM>(); };

  Sequences seqs;
  seqs.read(a);
  const int w1 = static_cast<int>(min(a.tokens, (window + 1) * a.window));
  int begin, end = -1;  // rows of sequence b, whose first position is start
  int b, start;
  bool asked = false;  // the new packs of the page at t are on their way to s_new
  for (int t = static_cast<int>(window * a.window); t < w1;) {
    if (t >= end) seqs.find(a, t, b, begin, end, start);
    if (t < begin || t >= end) {  // a row of no sequence
      ++t;
      end = -1;
      continue;
    }
    if (start < 0) {
      t = end;
      continue;
    }
    const uint32_t pos = static_cast<uint32_t>(start) + static_cast<uint32_t>(t) - static_cast<uint32_t>(begin);  // below 2^32
    const uint32_t col = pos / static_cast<uint32_t>(a.page_size);
    const int s0 = static_cast<int>(pos - col * static_cast<uint32_t>(a.page_size));
    const int n = min(a.page_size - s0, end - t);
    const int first = t;
    t += n;
    if (first != begin && s0 != 0) continue;  // not the sequence's first token in this page

    // Tokens of [0, m) that are this thread's: my_tok, my_tok + down, ...
    const auto mine = [&](int m) {
      if (!active || m <= my_tok) return 0;
      const uint32_t x = static_cast<uint32_t>(m - my_tok + down - 1);
      return static_cast<int>(a.per_down ? __umulhi(x, a.per_down) : x);
    };
    const int my_new = mine(n), my_old = mine(s0);
    int64_t page = -1;
    if (col < static_cast<uint32_t>(a.max_pages)) page = a.block_table[b * a.bt_stride + col];
    const bool kept = VEC == 8 && units <= across && n <= a.keep * down;  // they fit in shared memory
    const bool staged = VEC == 8 && units <= across && s0 <= a.keep * down;
    // The whole page at once, eight packs a lane, channel units a power of two.
    const bool whole = VEC == 8 && n == a.page_size && n == kWhole * down && across * down == 32 && units == across;
    const int64_t row = static_cast<int64_t>(first + my_tok) * a.new_stride + my_unit * VEC;
    const int64_t place = page * a.page_stride + my_tok * a.token_stride + my_unit * VEC;

    const bool have = asked;
    const bool more = t < w1 && end - t >= a.page_size;  // the window's next page is filled whole too
    asked = false;
    const E* const src = static_cast<const E*>(keys ? a.k_new : a.v_new) + row + h * a.head_dim;
    if constexpr (TEAM == 32 && PackExtremes<E, VEC>::kPairs) {
      if (whole && page >= 0 && page < a.num_pages) {
        uint8_t* const to = (keys ? a.k_cache : a.v_cache) + place + h * a.head_stride;
        float* const scale_at = (keys ? a.k_scale : a.v_scale) + page * a.num_kv_heads + h;
        int8_t* const out = bounds ? a.k_bounds + ((page * a.num_kv_heads + h) * 2) * a.head_dim : nullptr;
        const auto ask = [&](const E* from) {
          const uint32_t at = smem_u32(s_new + tid);
#pragma unroll
          for (int i = 0; i < kWhole; ++i) cp_async16(at + i * TEAM * sizeof(Pack), from + i * src_step);
        };
        if (!have) ask(src);
        cp_async_wait_all();
        const auto next = [&] {
          if (more) ask(src + a.page_size * a.new_stride);
          asked = more;
        };
        if (append_whole_page<E, Code>(s_new + tid, to, dst_step, scale_at, out, a.head_dim, across, next)) continue;
      }
    }
    // The new packs first (they need no page), then the page, its present scale and its codes.
    if constexpr (VEC == 8) {
      if (kept && !have) {
        const uint8_t* from = reinterpret_cast<const uint8_t*>(src);
        uint32_t to = smem_u32(s_new + tid);
#pragma unroll 4
        for (int i = 0; i < my_new; ++i) {
#pragma unroll
          for (int k = 0; k < static_cast<int>(sizeof(Pack)); k += 16) cp_async16(to + k, from + k);
          from += src_step * static_cast<int64_t>(sizeof(E));
          to += TEAM * sizeof(Pack);
        }
      }
    }
    if (page < 0 || page >= a.num_pages) {
      if (tid == 0 && a.status) atomicOr(a.status, kStatusBadPage);
      cp_async_wait_all();  // the next unit's copies may take the same places
      continue;
    }
    float* scale_at = (keys ? a.k_scale : a.v_scale) + page * a.num_kv_heads + h;
    const float old = s0 > 0 ? *scale_at : 0.0f;
    // This thread's first slot; slot s0 + my_tok is its first new one.
    uint8_t* const dst = (keys ? a.k_cache : a.v_cache) + place + h * a.head_stride;
    if (staged) {
      uint32_t to = smem_u32(s_codes) + tid * VEC;
      const uint8_t* from = dst;
#pragma unroll 4
      for (int i = 0; i < my_old; ++i, from += dst_step, to += TEAM * VEC) cp_async8(to, from);
    }
    cp_async_wait_all();  // each thread reads back what it copied itself

    // f(pack) over this thread's new packs of channel units c0, c0 + 1, ..., in token order.
    const auto for_new = [&](int c0, auto&& f) {
      if (kept) {
        const Pack* at = s_new + tid;
#pragma unroll 4
        for (int i = 0; i < my_new; ++i, at += TEAM) {
          Pack p;
          p.load(at->v);
          f(p);
        }
      } else if (c0 + my_unit < units) {
        const E* at = src + c0 * VEC;
#pragma unroll 1
        for (int i = 0; i < my_new; ++i, at += src_step) {
          Pack p;
          p.load(at);
          f(p);
        }
      }
    };

    Magnitude<E, VEC> mag;
    mag.reset();
    for (int c0 = 0; c0 < units; c0 += across) for_new(c0, [&](const Pack& p) { mag.add(p); });
    float amax = mag.get();
    const bool plain = team_all<TEAM>(amax <= FLT_MAX);  // no NaN, no infinity in the unit
    if (!plain) {
      amax = 0.0f;
      for (int c0 = 0; c0 < units; c0 += across) {
        for_new(c0, [&](const Pack& p) {
          float f[VEC];
          p.unpack(f);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            if (fabsf(f[j]) <= FLT_MAX) amax = fmaxf(amax, fabsf(f[j]));
          }
        });
      }
    }
    amax = team_max<TEAM>(amax, s_red);
    const float scale = fmaxf(old, Code::scale_for(amax));
    const float inv = reciprocal_scale(scale);
    const bool grew = s0 > 0 && scale > old;
    const float ratio = grew ? old / scale : 1.0f;
    barrier();  // every thread has read the old scale
    if (tid == 0) *scale_at = scale;

    for (int c0 = 0; c0 < units; c0 += across) {
      Extremes<VEC> ext;
      ext.reset();
      uint8_t* put = dst + c0 * VEC + s0 * a.token_stride;
      const auto quantise = [&](const Pack& p) {
        float y[VEC];
        p.unpack(y);
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] *= inv;
        store_codes<Code, VEC>(put, y, plain);  // plain: |y| is at most a rounding above the largest code
        put += dst_step;
      };
      if (bounds) {
        PackExtremes<E, VEC> raw;
        raw.reset();
        for_new(c0, [&](const Pack& p) {
          quantise(p);
          raw.add(p);
        });
        if (plain && my_new > 0) {  // this thread's own extremes, scaled
          raw.get(ext.lo, ext.hi);
#pragma unroll
          for (int j = 0; j < VEC; ++j) ext.lo[j] *= inv, ext.hi[j] *= inv;
        }
      } else {
        for_new(c0, quantise);
      }
      // Codes of the slots in use: those kept, and the new ones where the packs' extremes do not serve.
      const auto for_codes = [&](int count, uint8_t* at, float by, bool write, bool in_shared) {
        if (c0 + my_unit >= units) return;
        const uint8_t* in = in_shared ? s_codes + tid * VEC : at;
        const int64_t in_step = in_shared ? TEAM * VEC : dst_step;
#pragma unroll 2
        for (int i = 0; i < count; ++i, at += dst_step, in += in_step) {
          float y[VEC];
          load_codes<Code, VEC>(in, y);
#pragma unroll
          for (int j = 0; j < VEC; ++j) y[j] *= by;
          if (write) store_codes<Code, VEC>(at, y, false);
          if (bounds) ext.add(y);
        }
      };
      if (grew || bounds) for_codes(my_old, dst + c0 * VEC, ratio, grew, staged);
      if (bounds && !plain) {
        barrier();
        for_codes(my_new, dst + c0 * VEC + s0 * a.token_stride, 1.0f, false, false);
      }
      if (bounds) {
        const int width = across * VEC;
        barrier();
        if (active) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            s_lo[my_tok * width + my_unit * VEC + j] = ext.lo[j];
            s_hi[my_tok * width + my_unit * VEC + j] = ext.hi[j];
          }
        }
        barrier();
        int8_t* out = a.k_bounds + ((page * a.num_kv_heads + h) * 2) * a.head_dim + c0 * VEC;
        const int here = min(width, a.head_dim - c0 * VEC);
        constexpr int kAtOnce = VEC == 8 ? 4 : 1;  // channels a thread writes
        for (int i = tid * kAtOnce; i < here; i += TEAM * kAtOnce) {
          float l[kAtOnce], m[kAtOnce];
#pragma unroll
          for (int j = 0; j < kAtOnce; ++j) l[j] = FLT_MAX, m[j] = -FLT_MAX;
          for (int k = 0; k < down; ++k) {
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
              l[j] = fminf(l[j], s_lo[k * width + i + j]);
              m[j] = fmaxf(m[j], s_hi[k * width + i + j]);
            }
          }
          if constexpr (VEC == 8) {
            *reinterpret_cast<uint32_t*>(out + i) = bound_codes<Code, false, 4>(l, 1.0f);
            *reinterpret_cast<uint32_t*>(out + a.head_dim + i) = bound_codes<Code, true, 4>(m, 1.0f);
          } else {
            out[i] = static_cast<int8_t>(bound_codes<Code, false, 1>(l, 1.0f));
            out[a.head_dim + i] = static_cast<int8_t>(bound_codes<Code, true, 1>(m, 1.0f));
          }
        }
      }
    }
    barrier();  // another unit may follow: the extremes' place is free again
  }
}

bool append_pdl() {  // the same switch as the 16-bit append's
  static const bool on = env_switch_on("KL_APPEND_PDL");
  return on;
}

template <typename E, typename Code, int VEC, int TEAM>
cudaError_t launch_team(Block8AppendArgs a, cudaStream_t st) {
  a.across = std::min(a.head_dim / VEC, TEAM);
  a.down = TEAM / a.across;
  a.per_across = 65536u / static_cast<uint32_t>(a.across) + 1u;
  a.per_down = a.down == 1 ? 0u : 0xffffffffu / static_cast<uint32_t>(a.down) + 1u;
  // A page's packs a thread, up to 16 (of a larger page all are read again).
  const int64_t packs = (static_cast<int64_t>(a.page_size) + a.down - 1) / a.down;
  a.keep = VEC == 8 ? static_cast<int>(std::min<int64_t>(packs, 16)) : 0;
  constexpr int kTeams = kBlock8AppendThreads / TEAM;
  const int blocks = (2 * a.num_kv_heads + kTeams - 1) / kTeams;
  // Up to four pages a window, as many as leave 2.5 waves of blocks, and no more than a sequence brings.
  const int64_t waves = (a.tokens + a.window - 1) / a.window * blocks / (static_cast<int64_t>(sm_count()) * kAppendBlocks);
  a.window = static_cast<int>(std::min<int64_t>(a.window * std::max<int64_t>(1, std::min<int64_t>(waves * 2 / 5, 4)),
                                                std::max<int64_t>(1, a.tokens / a.batch)));
  const int64_t windows = (a.tokens + a.window - 1) / a.window;
  const unsigned y = static_cast<unsigned>(std::min<int64_t>(windows, kMaxGridY));
  const dim3 grid(static_cast<unsigned>(blocks), y, static_cast<unsigned>((windows + kMaxGridY - 1) / kMaxGridY));
  const int bytes = kTeams * team_bytes<E, VEC, TEAM>(a.keep);
  const auto kernel = kv_append_block8<E, Code, VEC, TEAM>;
  if (bytes > 48 * 1024 - 64) {
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_shared_memory(kernel, kTeams * team_bytes<E, VEC, TEAM>(16), done);
    if (e != cudaSuccess) return e;
  }
  return launch_kernel(append_pdl(), kernel, grid, dim3(kBlock8AppendThreads), static_cast<size_t>(bytes), st, a);
}

template <typename E, typename Code>
cudaError_t launch_codes(const Block8AppendArgs& a, bool vec, cudaStream_t st) {
  if (!vec) return launch_team<E, Code, 1, kBlock8AppendThreads>(a, st);
  // A warp keeps up to 16 packs of 8 elements a lane.
  const bool small = static_cast<int64_t>(a.page_size) * a.head_dim <= 4096 && a.head_dim <= 256;
  return small ? launch_team<E, Code, 8, 32>(a, st) : launch_team<E, Code, 8, kBlock8AppendThreads>(a, st);
}

template <typename E>
cudaError_t launch_elements(const Block8AppendArgs& a, int code_type, bool vec, cudaStream_t st) {
  return code_type == KL_CODE_E4M3 ? launch_codes<E, E4m3Code>(a, vec, st) : launch_codes<E, Int8Code>(a, vec, st);
}

bool multiple_of(int64_t n, const void* p) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace block8_append
}  // namespace klb

extern "C" int kl_paged_kv_append_block8(int dtype, int code_type, void* k_cache, void* v_cache, float* k_scale,
                                         float* v_scale, void* k_bounds, const void* k_new, const void* v_new,
                                         const int32_t* block_table, const int32_t* positions, const int32_t* indptr,
                                         int batch, int64_t tokens, int num_kv_heads, int head_dim, int page_size,
                                         int64_t page_stride, int64_t token_stride, int64_t head_stride,
                                         int64_t block_table_stride, int max_pages_per_seq, int64_t num_pages,
                                         int64_t new_row_stride, uint32_t* status, void* stream) {
  using namespace klb;
  using namespace klb::block8_append;
  constexpr int kInvalid = static_cast<int>(cudaErrorInvalidValue);
  if (batch == 0 || tokens == 0) return 0;
  if (batch < 0 || tokens < 0 || tokens > INT32_MAX || num_kv_heads <= 0 || num_kv_heads > 32767 || head_dim <= 0 ||
      head_dim > 1024 || page_size <= 0 || max_pages_per_seq < 0 || block_table_stride < max_pages_per_seq ||
      num_pages < 0 || page_stride < 0 || token_stride < 0 || head_stride < 0 ||
      new_row_stride < static_cast<int64_t>(num_kv_heads) * head_dim || (!indptr && tokens != batch) || !k_cache ||
      !v_cache || !k_scale || !v_scale || !k_new || !v_new || !block_table || !positions) {
    return kInvalid;
  }
  if (code_type != KL_CODE_E4M3 && code_type != KL_CODE_INT8) return kInvalid;
  Block8AppendArgs a{};
  a.k_cache = static_cast<uint8_t*>(k_cache);
  a.v_cache = static_cast<uint8_t*>(v_cache);
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.k_bounds = static_cast<int8_t*>(k_bounds);
  a.k_new = k_new;
  a.v_new = v_new;
  a.block_table = block_table;
  a.positions = positions;
  a.indptr = indptr;
  a.status = status;
  a.page_stride = page_stride;
  a.token_stride = token_stride;
  a.head_stride = head_stride;
  a.bt_stride = block_table_stride;
  a.new_stride = new_row_stride;
  a.num_pages = num_pages;
  a.tokens = tokens;
  a.batch = batch;
  a.num_kv_heads = num_kv_heads;
  a.head_dim = head_dim;
  a.page_size = page_size;
  a.max_pages = max_pages_per_seq;
  // A window holds about one first-in-page token: a page's length of tokens of long pieces, one
  // token where sequences bring one each.
  a.window = static_cast<int>(std::min<int64_t>(page_size, std::max<int64_t>(1, tokens / batch)));
  const int elem = dtype == KL_FLOAT32 ? 4 : 2;
  const bool vec = head_dim % 8 == 0 && (new_row_stride * elem) % 16 == 0 && multiple_of(16, k_new) &&
                   multiple_of(16, v_new) && multiple_of(8, k_cache) && multiple_of(8, v_cache) &&
                   page_stride % 8 == 0 && token_stride % 8 == 0 && head_stride % 8 == 0 && multiple_of(8, k_bounds);
  const auto st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case KL_FLOAT32: return static_cast<int>(launch_elements<float>(a, code_type, vec, st));
    case KL_FLOAT16: return static_cast<int>(launch_elements<__half>(a, code_type, vec, st));
    case KL_BFLOAT16: return static_cast<int>(launch_elements<__nv_bfloat16>(a, code_type, vec, st));
    default: return kInvalid;
  }
}
