// What the kernels of the block-scaled 8-bit cache share: the two code types.
#pragma once

#include <atomic>

#include "common.cuh"

namespace klb {

// Scales below this have no finite reciprocal worth using: codes of 0.
constexpr float kLeastScale = 0x1p-126f;
constexpr float kPer127 = 1.0f / 127.0f;  // int8 scales are products with this, one rounding, no division

struct E4m3Code {
  static constexpr int kBoundUnit = 4;  // 448 / 4 = 112 fits int8
  // The least power of two 2^k, k >= -126, with a <= 448 * 2^k: powers of two lose nothing (a code's
  // relative precision does not depend on the scale) and make a later growth exact. From the bits
  // of a = f * 2^e, f in [1, 2): 448 = 1.75 * 2^8, so k = e - 8, one more when f > 1.75.
  static __device__ __forceinline__ float scale_for(float amax) {
    if (!(amax > 0.0f)) return 0.0f;
    const uint32_t bits = __float_as_uint(amax);
    const int k = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return __uint_as_float(static_cast<uint32_t>(max(k, -126) + 127) << 23);
  }
  static __device__ __forceinline__ float value(uint32_t code) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(e4m3x2_lo_to_f16x2(code & 0xffu) & 0xffffu)));
  }
  static __device__ __forceinline__ uint32_t code(float v) {
    return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
  }
  // code() of four at once.
  static __device__ __forceinline__ uint32_t code4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
  // code4() for numbers within the codes' range.
  static __device__ __forceinline__ uint32_t code4_in_range(float a, float b, float c, float d) {
    return code4(a, b, c, d);
  }
};

struct Int8Code {
  static constexpr int kBoundUnit = 1;
  static __device__ __forceinline__ float scale_for(float amax) {
    return amax > 0.0f ? fmaxf(amax * kPer127, kLeastScale) : 0.0f;
  }
  static __device__ __forceinline__ float value(uint32_t code) {
    return static_cast<float>(static_cast<int8_t>(code & 0xffu));
  }
  // Rounds to nearest even; NaN converts to 0.
  static __device__ __forceinline__ uint32_t code(float v) {
    return static_cast<uint32_t>(max(-127, min(127, __float2int_rn(v)))) & 0xffu;
  }
  static __device__ __forceinline__ uint32_t code4(float a, float b, float c, float d) {
    return code(a) | (code(b) << 8) | (code(c) << 16) | (code(d) << 24);
  }
  // Adding 1.5 * 2^23 rounds to a whole number (nearest even) and leaves it in the low bits; never
  // fused with the product that made the number, which would round once instead of twice.
  static __device__ __forceinline__ uint32_t code4_in_range(float a, float b, float c, float d) {
    constexpr float kRound = 12582912.0f;
    const uint32_t lo = __byte_perm(__float_as_uint(__fadd_rn(a, kRound)), __float_as_uint(__fadd_rn(b, kRound)), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(__fadd_rn(c, kRound)), __float_as_uint(__fadd_rn(d, kRound)), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  }
};

__device__ __forceinline__ float reciprocal_scale(float scale) { return scale >= kLeastScale ? 1.0f / scale : 0.0f; }

// 16 bytes from global to shared memory, asynchronously (both 16-byte aligned).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Host side: lets `kernel` use up to `bytes` of dynamic shared memory on the current device, asked
// of the runtime once for each kernel and device.
template <typename... Params>
inline cudaError_t allow_shared_memory(void (*kernel)(Params...), int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// SMs of the current device.
inline int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
  return n;
}

}  // namespace klb
