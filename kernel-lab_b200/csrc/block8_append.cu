// Append to a paged cache held in 8 bits with a scale for each page and KV head, for sm_100a: one
// new token a sequence, or a prompt's tokens.
//
// The work falls into units of one page, KV head and tensor: the largest magnitude of the page's
// new elements gives the scale, so a unit is a reduction and then an elementwise pass over the same
// elements. A team of one warp (pages of up to 2048 elements a head) or of four warps takes a unit
// and copies its new elements to shared memory, all in flight at once and without registers, so that
// it reads them once; larger pages re-read theirs from L2. HBM-bound for prompts (the new rows in, half or a quarter of their bytes out),
// latency-bound for single tokens, where the chain is indptr / position, block-table entry, new row.
//
// No host knows where pages begin in the ragged rows, so a team takes a window of the flattened new
// tokens and looks for the tokens in it that are the first of their sequence in a page; the window
// is a page's length when sequences bring many tokens and one token when they bring one each.
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
namespace {

constexpr int kBlock8AppendThreads = 128;

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
};

// Last b with indptr[b] <= t, by all lanes of a warp (32 samples a step).
__device__ __forceinline__ int sequence_of(const int32_t* indptr, int batch, int64_t t) {
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
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&y)[VEC]) {
  if constexpr (VEC == 8) {
    *reinterpret_cast<uint2*>(p) =
        make_uint2(Code::code4(y[0], y[1], y[2], y[3]), Code::code4(y[4], y[5], y[6], y[7]));
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

template <typename E, typename Code, int VEC, int TEAM>
__global__ void __launch_bounds__(kBlock8AppendThreads) kv_append_block8(const Block8AppendArgs a) {
  constexpr int kTeams = kBlock8AppendThreads / TEAM;
  using Pack = NewPack<E, VEC>;
  constexpr int kKeep = VEC == 8 ? 8 : 1;  // packs a thread keeps in shared memory
  __shared__ __align__(16) Pack s_new[kTeams][kKeep][TEAM];
  __shared__ __align__(16) float s_ext[kTeams][2][TEAM * VEC];
  __shared__ float s_red[kBlock8AppendThreads / 32];
  const int team = threadIdx.x / TEAM, tid = threadIdx.x % TEAM;
  const int h = blockIdx.y * kTeams + team;
  wait_prior_grid();
  allow_next_grid();
  if (h >= a.num_kv_heads) return;  // whole warps; with TEAM 128 there is one team a block
  const bool keys = blockIdx.z == 0;
  const bool bounds = keys && a.k_bounds != nullptr;

  const int units = a.head_dim / VEC;
  const int across = min(units, TEAM), down = TEAM / across;
  const int my_tok = tid / across, my_unit = tid % across;
  const bool active = my_tok < down;

  const int64_t w1 = min(a.tokens, (static_cast<int64_t>(blockIdx.x) + 1) * a.window);
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * a.window; t < w1;) {
    int64_t begin = t, end = t + 1;
    int b = static_cast<int>(t);
    if (a.indptr) {
      b = sequence_of(a.indptr, a.batch, t);
      begin = a.indptr[b];
      end = min(static_cast<int64_t>(a.indptr[b + 1]), a.tokens);
    }
    if (t < begin || t >= end) {  // a row of no sequence
      ++t;
      continue;
    }
    const int start = a.positions[b];
    if (start < 0) {
      t = end;
      continue;
    }
    const int64_t pos = start + (t - begin);
    const int64_t col = pos / a.page_size;
    const int s0 = static_cast<int>(pos - col * a.page_size);
    const int n = static_cast<int>(min(static_cast<int64_t>(a.page_size - s0), end - t));
    const int64_t first = t;
    t += n;
    if (first != begin && s0 != 0) continue;  // not the sequence's first token in this page

    // The new packs first (they need no page), then the page and its present scale.
    const E* src = static_cast<const E*>(keys ? a.k_new : a.v_new) + first * a.new_stride +
                   static_cast<int64_t>(h) * a.head_dim + my_unit * VEC;
    const bool kept = VEC == 8 && units <= across && n <= kKeep * down;  // they fit in shared memory
    if constexpr (VEC == 8) {
      if (kept && active) {
        for (int i = 0, tok = my_tok; tok < n; ++i, tok += down) {
#pragma unroll
          for (int k = 0; k < static_cast<int>(sizeof(Pack)); k += 16) {
            cp_async16(smem_u32(&s_new[team][i][tid]) + k, reinterpret_cast<const uint8_t*>(src + tok * a.new_stride) + k);
          }
        }
      }
    }
    int64_t page = -1;
    if (col < a.max_pages) page = a.block_table[b * a.bt_stride + col];
    if (page < 0 || page >= a.num_pages) {
      if (tid == 0 && a.status) atomicOr(a.status, kStatusBadPage);
      cp_async_wait_all();  // the next unit's copies may take the same places
      continue;
    }
    float* scale_at = (keys ? a.k_scale : a.v_scale) + page * a.num_kv_heads + h;
    const float old = s0 > 0 ? *scale_at : 0.0f;
    uint8_t* dst = (keys ? a.k_cache : a.v_cache) + page * a.page_stride + h * a.head_stride + my_unit * VEC;

    cp_async_wait_all();  // each thread reads back what it copied itself

    // f(pack, token) over this thread's new packs of channel units c0, c0 + 1, ...
    const auto for_new = [&](int c0, auto&& f) {
      if (!active || c0 + my_unit >= units) return;
      const E* at = kept ? s_new[team][0][tid].v : src + my_tok * a.new_stride + c0 * VEC;
      const int64_t step = kept ? static_cast<int64_t>(TEAM) * VEC : down * a.new_stride;
#pragma unroll 2
      for (int tok = my_tok; tok < n; tok += down, at += step) {
        Pack p;
        p.load(at);
        f(p, tok);
      }
    };

    Magnitude<E, VEC> mag;
    mag.reset();
    for (int c0 = 0; c0 < units; c0 += across) for_new(c0, [&](const Pack& p, int) { mag.add(p); });
    float amax = mag.get();
    const bool plain = team_all<TEAM>(amax <= FLT_MAX);  // no NaN, no infinity in the unit
    if (!plain) {
      amax = 0.0f;
      for (int c0 = 0; c0 < units; c0 += across) {
        for_new(c0, [&](const Pack& p, int) {
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
    team_sync<TEAM>();  // every thread has read the old scale
    if (tid == 0) *scale_at = scale;

    for (int c0 = 0; c0 < units; c0 += across) {
      Extremes<VEC> ext;
      {
        PackExtremes<E, VEC> raw;
        raw.reset();
        for_new(c0, [&](const Pack& p, int tok) {
          float y[VEC];
          p.unpack(y);
#pragma unroll
          for (int j = 0; j < VEC; ++j) y[j] *= inv;
          store_codes<Code, VEC>(dst + c0 * VEC + (s0 + tok) * a.token_stride, y);
          if (bounds) raw.add(p);
        });
        raw.get(ext.lo, ext.hi);
      }
      const bool had = plain && active && my_tok < n;  // this thread's own extremes, to be scaled
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        ext.lo[j] = had ? ext.lo[j] * inv : FLT_MAX;
        ext.hi[j] = had ? ext.hi[j] * inv : -FLT_MAX;
      }
      // Codes of the slots in use: those kept, and the new ones where the packs' extremes do not serve.
      const auto for_codes = [&](int from, int to, float by, bool write) {
        if (!active || c0 + my_unit >= units) return;
#pragma unroll 2
        for (int tok = from + my_tok; tok < to; tok += down) {
          uint8_t* at = dst + c0 * VEC + tok * a.token_stride;
          float y[VEC];
          load_codes<Code, VEC>(at, y);
#pragma unroll
          for (int j = 0; j < VEC; ++j) y[j] *= by;
          if (write) store_codes<Code, VEC>(at, y);
          if (bounds) ext.add(y);
        }
      };
      if (grew || bounds) for_codes(0, s0, ratio, grew);
      if (bounds && !plain) {
        team_sync<TEAM>();
        for_codes(s0, s0 + n, 1.0f, false);
      }
      if (bounds) {
        float* lo = s_ext[team][0];
        float* hi = s_ext[team][1];
        const int width = across * VEC;
        team_sync<TEAM>();
        if (active) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            lo[my_tok * width + my_unit * VEC + j] = ext.lo[j];
            hi[my_tok * width + my_unit * VEC + j] = ext.hi[j];
          }
        }
        team_sync<TEAM>();
        int8_t* out = a.k_bounds + ((page * a.num_kv_heads + h) * 2) * a.head_dim + c0 * VEC;
        const int here = min(width, a.head_dim - c0 * VEC);
        for (int i = tid; i < here; i += TEAM) {
          float l = FLT_MAX, m = -FLT_MAX;
          for (int k = 0; k < down; ++k) {
            l = fminf(l, lo[k * width + i]);
            m = fmaxf(m, hi[k * width + i]);
          }
          constexpr float kPerUnit = 1.0f / Code::kBoundUnit;  // a power of two
          out[i] = static_cast<int8_t>(floorf(Code::value(Code::code(l)) * kPerUnit));
          out[a.head_dim + i] = static_cast<int8_t>(ceilf(Code::value(Code::code(m)) * kPerUnit));
        }
      }
    }
  }
}

bool append_pdl() {  // the same switch as the 16-bit append's
  static const bool on = env_switch_on("KL_APPEND_PDL");
  return on;
}

template <typename E, typename Code, int VEC, int TEAM>
cudaError_t launch_team(const Block8AppendArgs& a, cudaStream_t st) {
  constexpr int kTeams = kBlock8AppendThreads / TEAM;
  const int64_t windows = (a.tokens + a.window - 1) / a.window;
  const dim3 grid(static_cast<unsigned>(windows), static_cast<unsigned>((a.num_kv_heads + kTeams - 1) / kTeams), 2);
  return launch_kernel(append_pdl(), kv_append_block8<E, Code, VEC, TEAM>, grid, dim3(kBlock8AppendThreads), 0, st, a);
}

template <typename E, typename Code>
cudaError_t launch_codes(const Block8AppendArgs& a, bool vec, cudaStream_t st) {
  if (!vec) return launch_team<E, Code, 1, kBlock8AppendThreads>(a, st);
  // A warp keeps 8 packs of 8 elements a lane.
  const bool small = static_cast<int64_t>(a.page_size) * a.head_dim <= 2048 && a.head_dim <= 256;
  return small ? launch_team<E, Code, 8, 32>(a, st) : launch_team<E, Code, 8, kBlock8AppendThreads>(a, st);
}

template <typename E>
cudaError_t launch_elements(const Block8AppendArgs& a, int code_type, bool vec, cudaStream_t st) {
  return code_type == KL_CODE_E4M3 ? launch_codes<E, E4m3Code>(a, vec, st) : launch_codes<E, Int8Code>(a, vec, st);
}

bool multiple_of(int64_t n, const void* p) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace klb

extern "C" int kl_paged_kv_append_block8(int dtype, int code_type, void* k_cache, void* v_cache, float* k_scale,
                                         float* v_scale, void* k_bounds, const void* k_new, const void* v_new,
                                         const int32_t* block_table, const int32_t* positions, const int32_t* indptr,
                                         int batch, int64_t tokens, int num_kv_heads, int head_dim, int page_size,
                                         int64_t page_stride, int64_t token_stride, int64_t head_stride,
                                         int64_t block_table_stride, int max_pages_per_seq, int64_t num_pages,
                                         int64_t new_row_stride, uint32_t* status, void* stream) {
  using namespace klb;
  constexpr int kInvalid = static_cast<int>(cudaErrorInvalidValue);
  if (batch == 0 || tokens == 0) return 0;
  if (batch < 0 || tokens < 0 || tokens > INT32_MAX || num_kv_heads <= 0 || num_kv_heads > 65535 || head_dim <= 0 ||
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
                   page_stride % 8 == 0 && token_stride % 8 == 0 && head_stride % 8 == 0;
  const auto st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case KL_FLOAT32: return static_cast<int>(launch_elements<float>(a, code_type, vec, st));
    case KL_FLOAT16: return static_cast<int>(launch_elements<__half>(a, code_type, vec, st));
    case KL_BFLOAT16: return static_cast<int>(launch_elements<__nv_bfloat16>(a, code_type, vec, st));
    default: return kInvalid;
  }
}
