// RMSNorm and fused residual-add + RMSNorm with an e4m3 output for sm_100a.
//
//   r' = T(float(x) + float(r))            (with a residual; bit-exact, as kl_rms_norm forms it)
//   y  = r' * rstd * w,  rstd = 1 / sqrt(mean(r'^2) + eps)            (never rounded to T)
//   a  = max |y| over a group of columns (NaN ignored): a whole row, or group_size columns
//   scale = a / 448,  code = e4m3(y * 448 / a), nearest-even, saturating
// rstd is common to y and a, so the codes need none of it: with t = r' * w (exact in fp32 for 16-bit
// types) and b = max |t|, code = e4m3(t * (448 / b)) and a = b * rstd: one product and few roundings
// an element. A group whose a or b is below 2^-100 (448 / b would overflow) gets scale
// 0 and codes 0; a row whose rstd is NaN or infinite gets NaN codes, as its y are.
//
// HBM-bound: x, residual in; residual out, one byte an element and the scales out. As in the 16-bit
// kernel one CTA takes a row, every thread issues all its 16-byte loads before it uses any, and the
// row stays in registers, so each tensor crosses HBM once. With one scale a row, b needs no barrier
// of its own: it is reduced along with the sum of squares. With a scale a group, a group's columns sit in adjacent lanes of one warp (16
// lanes for 128 columns of a 16-bit type), and its maximum is a few shuffles.
//
// Measured (bf16 with a residual): 4096 x 8192 with a scale for each 128 columns 37.4 us, 6.3 TB/s of the
// 236 MB (0.96 of the copy peak); 16 x 8192 with a scale a row 2.3 us a call in a graph. At first the
// conversions took 36 instructions an element and bound it (66 us); packed conversions and
// mixed-precision multiply-adds on register halves, and codes that need no rstd, took that to 12.
//
// Widths or pointers that 16-byte loads cannot take, groups that are not 1 to 32 whole packs (a
// power of two of them) and rows wider than the registers hold run in a fallback that re-reads its
// row from L2 (1000 x 5001 fp16 24 us, 512 x 20000 bf16 48 us: 0.2 of the copy peak).
#include <algorithm>
#include <cstdint>

#include <cuda_runtime.h>

#include "block8.cuh"
#include "kernel_lab_b200_block8.h"

namespace klb {
// A namespace with a name: an unnamed one's symbols carry a hash of the file's text, and with them the
// compiler's register allocation would change with a comment.
namespace rmsnorm_fp8 {

constexpr float kE4m3Max = 448.0f;
constexpr float kPerE4m3Max = 1.0f / 448.0f;
constexpr float kLeastAmax = 0x1p-100f;  // below it a group's scale is 0

// lo += a.low * b.low, hi += a.high * b.high for packed 16-bit pairs, by mixed-precision multiply-adds
// (no unpacking into floats first).
template <typename T>
__device__ __forceinline__ void fma_pair_to(uint32_t a, uint32_t b, float& lo, float& hi);
template <>
__device__ __forceinline__ void fma_pair_to<__nv_bfloat16>(uint32_t a, uint32_t b, float& lo, float& hi) {
  asm("{\n.reg .b16 al, ah, bl, bh;\nmov.b32 {al, ah}, %2;\nmov.b32 {bl, bh}, %3;\n"
      "fma.rn.f32.bf16 %0, al, bl, %0;\nfma.rn.f32.bf16 %1, ah, bh, %1;\n}"
      : "+f"(lo), "+f"(hi)
      : "r"(a), "r"(b));
}
template <>
__device__ __forceinline__ void fma_pair_to<__half>(uint32_t a, uint32_t b, float& lo, float& hi) {
  asm("{\n.reg .b16 al, ah, bl, bh;\nmov.b32 {al, ah}, %2;\nmov.b32 {bl, bh}, %3;\n"
      "fma.rn.f32.f16 %0, al, bl, %0;\nfma.rn.f32.f16 %1, ah, bh, %1;\n}"
      : "+f"(lo), "+f"(hi)
      : "r"(a), "r"(b));
}

// lo = a.low * b.low, hi = a.high * b.high (exact).
template <typename T>
__device__ __forceinline__ void mul_pair(uint32_t a, uint32_t b, float& lo, float& hi);
template <>
__device__ __forceinline__ void mul_pair<__nv_bfloat16>(uint32_t a, uint32_t b, float& lo, float& hi) {
  asm("{\n.reg .b16 al, ah, bl, bh;\nmov.b32 {al, ah}, %2;\nmov.b32 {bl, bh}, %3;\n"
      "fma.rn.f32.bf16 %0, al, bl, %4;\nfma.rn.f32.bf16 %1, ah, bh, %4;\n}"
      : "=f"(lo), "=f"(hi)
      : "r"(a), "r"(b), "f"(0.0f));
}
template <>
__device__ __forceinline__ void mul_pair<__half>(uint32_t a, uint32_t b, float& lo, float& hi) {
  asm("{\n.reg .b16 al, ah, bl, bh;\nmov.b32 {al, ah}, %2;\nmov.b32 {bl, bh}, %3;\n"
      "fma.rn.f32.f16 %0, al, bl, %4;\nfma.rn.f32.f16 %1, ah, bh, %4;\n}"
      : "=f"(lo), "=f"(hi)
      : "r"(a), "r"(b), "f"(0.0f));
}

// 16 bytes of a row.
template <typename T>
struct RowPack {
  static constexpr int N = 16 / sizeof(T);
  uint32_t w[4];
  __device__ __forceinline__ void load(uint4 v) { w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w; }
  __device__ __forceinline__ uint4 raw() const { return make_uint4(w[0], w[1], w[2], w[3]); }
  // this = T(float(this) + float(r))
  __device__ __forceinline__ void add(const RowPack& r) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (N == 8) {
        float2 f = Storage<T>::unpack2(r.w[i]);
        add_pair_to<T>(w[i], f.x, f.y);
        w[i] = Storage<T>::pack2(f.x, f.y);
      } else {
        w[i] = __float_as_uint(__uint_as_float(w[i]) + __uint_as_float(r.w[i]));
      }
    }
  }
  __device__ __forceinline__ void add_squares(float& s0, float& s1) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (N == 8) {
        fma_pair_to<T>(w[i], w[i], s0, s1);
      } else {
        float& s = i & 1 ? s1 : s0;
        s = fmaf(__uint_as_float(w[i]), __uint_as_float(w[i]), s);
      }
    }
  }
  // t = this * weights
  __device__ __forceinline__ void times(const RowPack& k, float (&t)[N]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (N == 8) {
        mul_pair<T>(w[i], k.w[i], t[2 * i], t[2 * i + 1]);
      } else {
        t[i] = __uint_as_float(w[i]) * __uint_as_float(k.w[i]);
      }
    }
  }
};

template <int N>
__device__ __forceinline__ float largest(const float (&t)[N], float top) {
#pragma unroll
  for (int j = 0; j < N; ++j) top = fmaxf(top, fabsf(t[j]));
  return top;
}

// What a group's t are multiplied by for its codes, and the scale that undoes it for y.
struct GroupScale {
  float inv, scale;
  __device__ __forceinline__ GroupScale(float b, float rstd) {
    const float a = b * rstd;
    const bool some = a >= kLeastAmax && b >= kLeastAmax;  // false for NaN too; b is at most 2^126
    inv = some ? __fdividef(kE4m3Max, b) : 0.0f * rstd;  // within 2 units in the last place
    scale = some ? a * kPerE4m3Max : 0.0f;
  }
};

struct SumMax {
  float sum, max;
};

// Sum and maximum over the block; every thread gets both. `red` holds one pair per warp.
__device__ __forceinline__ SumMax block_allreduce(float sum, float max, SumMax* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  sum = warp_allreduce_sum(sum);
  max = warp_allreduce_max(max);
  if (lane == 0) red[warp] = SumMax{sum, max};
  __syncthreads();
  SumMax t{0.0f, 0.0f};
  for (int w = 0; w < nwarps; ++w) {
    t.sum += red[w].sum;
    t.max = fmaxf(t.max, red[w].max);
  }
  return t;
}

struct NormFp8Args {
  uint8_t* codes;
  float* scales;
  void* residual_out;
  const void* x;
  const void* residual;
  const void* weight;
  int hidden;
  int group;       // columns of a group
  int groups;      // groups of a row
  int64_t x_row_stride;
  float eps;
};

// One CTA per row; each thread owns NPT 16-byte packs of the row, strided by blockDim. GROUPS: a
// scale for each `lanes` packs (adjacent lanes), else one for the row (four packs a thread of a 16-bit type spill 8
// to 16 bytes then).
template <typename T, int NPT, bool RES, bool GROUPS>
__global__ void __launch_bounds__(512, 2) rmsnorm_fp8_row_regs(const NormFp8Args g, int lanes) {
  using P = RowPack<T>;
  __shared__ SumMax red[32];
  const int packs = g.hidden / P::N;
  const int64_t row = blockIdx.x;
  const uint4* xr = reinterpret_cast<const uint4*>(static_cast<const T*>(g.x) + row * g.x_row_stride);
  const uint4* rr = reinterpret_cast<const uint4*>(static_cast<const T*>(g.residual) + row * g.hidden);
  uint4* ro = reinterpret_cast<uint4*>(static_cast<T*>(g.residual_out) + row * g.hidden);
  const uint4* wr = reinterpret_cast<const uint4*>(g.weight);
  uint8_t* codes = g.codes + row * g.hidden;
  float* scales = g.scales + row * g.groups;

  P a[NPT], r[NPT], w[NPT];
  wait_prior_grid();
#pragma unroll
  for (int i = 0; i < NPT; ++i) {
    const int pk = threadIdx.x + i * blockDim.x;
    const uint4 none = make_uint4(0, 0, 0, 0);  // packs past the row add nothing
    a[i].load(pk < packs ? __ldcs(xr + pk) : none);
    if constexpr (RES) r[i].load(pk < packs ? __ldcs(rr + pk) : none);
    if constexpr (!GROUPS) w[i].load(pk < packs ? __ldg(wr + pk) : none);
  }

  float s0 = 0.0f, s1 = 0.0f, top = 0.0f;
#pragma unroll
  for (int i = 0; i < NPT; ++i) {
    const int pk = threadIdx.x + i * blockDim.x;
    if constexpr (RES) {
      a[i].add(r[i]);
      if (pk < packs) ro[pk] = a[i].raw();
    }
    a[i].add_squares(s0, s1);
    if constexpr (!GROUPS) {
      float t[P::N];
      a[i].times(w[i], t);
      top = largest(t, top);
    }
  }

  if constexpr (GROUPS) {  // needed only from here on: in the residual's registers, under the reduction
#pragma unroll
    for (int i = 0; i < NPT; ++i) {
      const int pk = threadIdx.x + i * blockDim.x;
      w[i].load(pk < packs ? __ldg(wr + pk) : make_uint4(0, 0, 0, 0));
    }
  }
  const SumMax all = block_allreduce(s0 + s1, top, red);
  const float rstd = 1.0f / sqrtf(all.sum / static_cast<float>(g.hidden) + g.eps);
  allow_next_grid();
  float inv = 0.0f;
  if constexpr (!GROUPS) {
    const GroupScale whole(all.max, rstd);
    inv = whole.inv;
    if (threadIdx.x == 0) scales[0] = whole.scale;
  }

#pragma unroll
  for (int i = 0; i < NPT; ++i) {
    const int pk = threadIdx.x + i * blockDim.x;
    float t[P::N];
    a[i].times(w[i], t);
    if constexpr (GROUPS) {
      float b = largest(t, 0.0f);
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) {
        if (m < lanes) b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, m));
      }
      const GroupScale s(b, rstd);
      inv = s.inv;
      if (pk < packs && (pk & (lanes - 1)) == 0) scales[pk >> (31 - __clz(lanes))] = s.scale;
    }
    if (pk < packs) {
      uint32_t c[P::N / 4];
#pragma unroll
      for (int j = 0; j < P::N; j += 4) {
        c[j / 4] = E4m3Code::code4(t[j] * inv, t[j + 1] * inv, t[j + 2] * inv, t[j + 3] * inv);
      }
      if constexpr (P::N == 8) {
        *reinterpret_cast<uint2*>(codes + pk * 8) = make_uint2(c[0], c[1]);
      } else {
        *reinterpret_cast<uint32_t*>(codes + pk * 4) = c[0];
      }
    }
  }
}

// General fallback: any width, alignment and group. Pass 1 forms (and stores) the rounded sum and
// the sum of squares; then each warp takes a group at a time (the whole block with one scale a row),
// finds its maximum and quantises it, re-reading the row from L2.
template <typename T, bool RES>
__global__ void __launch_bounds__(1024) rmsnorm_fp8_row_general(const NormFp8Args g) {
  __shared__ SumMax red[32];
  const int64_t row = blockIdx.x;
  const T* xr = static_cast<const T*>(g.x) + row * g.x_row_stride;
  const T* rr = static_cast<const T*>(g.residual) + row * g.hidden;
  T* ro = static_cast<T*>(g.residual_out) + row * g.hidden;
  const T* w = static_cast<const T*>(g.weight);
  uint8_t* codes = g.codes + row * g.hidden;
  float* scales = g.scales + row * g.groups;

  wait_prior_grid();
  float ss = 0.0f;
  for (int i = threadIdx.x; i < g.hidden; i += blockDim.x) {
    float f = Storage<T>::load(xr[i]);
    if constexpr (RES) {
      const T s = Storage<T>::store(f + Storage<T>::load(rr[i]));
      ro[i] = s;
      f = Storage<T>::load(s);
    }
    ss = fmaf(f, f, ss);
  }
  const float mean = block_allreduce(ss, 0.0f, red).sum / static_cast<float>(g.hidden);
  const float rstd = 1.0f / sqrtf(mean + g.eps);
  allow_next_grid();
  __syncthreads();  // every column of the row is stored, and `red` is free again
  const T* src = RES ? ro : xr;
  const auto t = [&](int i) { return Storage<T>::load(src[i]) * Storage<T>::load(w[i]); };
  const auto put = [&](int i, float inv) {
    codes[i] = static_cast<uint8_t>(E4m3Code::code(t(i) * inv));
  };
  if (g.groups == 1) {
    float top = 0.0f;
    for (int i = threadIdx.x; i < g.hidden; i += blockDim.x) top = fmaxf(top, fabsf(t(i)));
    const GroupScale s(block_allreduce(0.0f, top, red).max, rstd);
    if (threadIdx.x == 0) scales[0] = s.scale;
    for (int i = threadIdx.x; i < g.hidden; i += blockDim.x) put(i, s.inv);
    return;
  }
  const int lane = threadIdx.x & 31;
  for (int k = threadIdx.x >> 5; k < g.groups; k += blockDim.x >> 5) {
    const int lo = k * g.group, hi = min(g.hidden, lo + g.group);
    float top = 0.0f;
    for (int i = lo + lane; i < hi; i += 32) top = fmaxf(top, fabsf(t(i)));
    const GroupScale s(warp_allreduce_max(top), rstd);
    if (lane == 0) scales[k] = s.scale;
    for (int i = lo + lane; i < hi; i += 32) put(i, s.inv);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool use_pdl() {  // the same switch as the 16-bit kernels'
  static const bool on = env_switch_on("KL_RMSNORM_PDL");
  return on;
}

template <typename... Params, typename... Args>
cudaError_t launch_rows(void (*kernel)(Params...), int rows, int threads, cudaStream_t st, const Args&... args) {
  return launch_kernel(use_pdl(), kernel, dim3(static_cast<unsigned>(rows)), dim3(static_cast<unsigned>(threads)), 0,
                       st, args...);
}

template <typename T, int NPT>
cudaError_t launch_regs(const NormFp8Args& g, int rows, int threads, int lanes, cudaStream_t st) {
  if (g.groups > 1) {
    return g.residual ? launch_rows(rmsnorm_fp8_row_regs<T, NPT, true, true>, rows, threads, st, g, lanes)
                      : launch_rows(rmsnorm_fp8_row_regs<T, NPT, false, true>, rows, threads, st, g, lanes);
  }
  return g.residual ? launch_rows(rmsnorm_fp8_row_regs<T, NPT, true, false>, rows, threads, st, g, lanes)
                    : launch_rows(rmsnorm_fp8_row_regs<T, NPT, false, false>, rows, threads, st, g, lanes);
}

template <typename T>
cudaError_t launch_typed(const NormFp8Args& g, int rows, cudaStream_t st) {
  constexpr int N = 16 / sizeof(T);
  const int packs = g.hidden / N;
  const int lanes = g.groups == 1 ? 0 : g.group / N;
  const bool grouped = g.groups == 1 || (g.group % N == 0 && lanes <= 32 && (lanes & (lanes - 1)) == 0);
  const bool vec = g.hidden % N == 0 && g.x_row_stride % N == 0 && aligned16(g.codes) && aligned16(g.x) &&
                   aligned16(g.weight) && (!g.residual || (aligned16(g.residual) && aligned16(g.residual_out)));
  if (vec && grouped && packs <= 4 * 512) {
    // As for the 16-bit output: enough packs a thread to keep several loads in flight on wide rows.
    const int npt = packs <= 128 ? 1 : packs <= 512 ? 2 : 4;
    const int threads = std::min(512, std::max(32, ((packs + npt - 1) / npt + 31) / 32 * 32));
    switch (npt) {
      case 1: return launch_regs<T, 1>(g, rows, threads, lanes, st);
      case 2: return launch_regs<T, 2>(g, rows, threads, lanes, st);
      default: return launch_regs<T, 4>(g, rows, threads, lanes, st);
    }
  }
  const int threads = std::min(1024, std::max(32, (g.hidden + 31) / 32 * 32));
  return g.residual ? launch_rows(rmsnorm_fp8_row_general<T, true>, rows, threads, st, g)
                    : launch_rows(rmsnorm_fp8_row_general<T, false>, rows, threads, st, g);
}

}  // namespace rmsnorm_fp8
}  // namespace klb

extern "C" int kl_rms_norm_fp8(int dtype, void* codes, float* scales, void* residual_out, const void* x,
                               const void* residual, const void* weight, int rows, int hidden, int64_t x_row_stride,
                               int group_size, float eps, void* stream) {
  using namespace klb;
  using namespace klb::rmsnorm_fp8;
  if (rows == 0) return 0;
  if (rows < 0 || hidden <= 0 || x_row_stride < 0 || group_size < 0 || !codes || !scales || !x || !weight ||
      (residual == nullptr) != (residual_out == nullptr)) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  NormFp8Args g{};
  g.codes = static_cast<uint8_t*>(codes);
  g.scales = scales;
  g.residual_out = residual_out;
  g.x = x;
  g.residual = residual;
  g.weight = weight;
  g.hidden = hidden;
  g.group = group_size == 0 ? hidden : std::min(group_size, hidden);
  g.groups = (hidden - 1) / g.group + 1;
  g.x_row_stride = x_row_stride;
  g.eps = eps;
  const auto st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case KL_FLOAT32: return static_cast<int>(launch_typed<float>(g, rows, st));
    case KL_FLOAT16: return static_cast<int>(launch_typed<__half>(g, rows, st));
    case KL_BFLOAT16: return static_cast<int>(launch_typed<__nv_bfloat16>(g, rows, st));
    default: return static_cast<int>(cudaErrorInvalidValue);
  }
}
