// q8.hpp -- what the 8-bit operators (q8.hip, kv8.hip) share: element types, row quantisation, host-side checks.
#pragma once

#include <math.h>

#include "kernels.hpp"

namespace wj {

// the calling thread's device is put back on every way out of an entry point
struct DeviceScope {
  int prev = -1;
  hipError_t enter(int device) {
    hipError_t e = hipGetDevice(&prev);
    if (e != hipSuccess) { prev = -1; return e; }
    if (prev == device) { prev = -1; return hipSuccess; }
    return hipSetDevice(device);
  }
  ~DeviceScope() { if (prev >= 0) (void)hipSetDevice(prev); }
};

inline bool known_dtype(int dtype) { return dtype == WJ_F32 || is16(dtype); }
inline bool aligned_to(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// bfloat16 of any float, NaN included (f2bf's carry can turn a NaN's payload into an infinity): one instruction on gfx950
__device__ __forceinline__ bf16_t f2bf_any(float v) { return __builtin_bit_cast(bf16_t, static_cast<__bf16>(v)); }
template <typename T> __device__ __forceinline__ T to_T(float v);
template <> __device__ __forceinline__ float to_T<float>(float v) { return v; }
template <> __device__ __forceinline__ f16_t to_T<f16_t>(float v) { return f2h(v); }
template <> __device__ __forceinline__ bf16_t to_T<bf16_t>(float v) { return f2bf_any(v); }

// one element of a row whose type is known at run time only (wave-uniform)
__device__ __forceinline__ void st_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == WJ_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dtype == WJ_F16) reinterpret_cast<f16_t*>(p)[i] = f2h(v);
  else reinterpret_cast<bf16_t*>(p)[i] = f2bf_any(v);
}

// magnitude that carries "not finite" through a maximum: fmaxf alone drops a NaN
__device__ __forceinline__ float mag(float v) { const float a = fabsf(v); return a < INFINITY ? a : INFINITY; }

// The quantiser of a row with maximum magnitude `amax` (INFINITY: the row holds a NaN or an infinity): scale = amax / 127, code =
// rint(127 v / amax).  The quotient is the rounded one (a reciprocal, then one correction) and 127 v is exact for 16-bit values, so that a
// tie is one: v = amax / 2 is 63.5 and common among 16-bit values.  Rounding v / scale instead, where scale itself was rounded, or missing
// the tie by a product with 127 / amax, moves codes of many rows (128 bfloat16 columns: 5.8e-4 off, relative to the row's norm, against 4.0e-4).
// Below 1e-30 and above 1e30 values and maximum are lifted by a power of two first, where the products would leave float32's range.
struct RowQuant {
  float scale, lift, top, inv;
  bool live;
  __device__ __forceinline__ explicit RowQuant(float amax) {
    live = amax > 0.f && amax < INFINITY;
    const float by = amax < 1e-30f ? 1.2089258196146292e24f : amax > 1e30f ? 8.271806125530277e-25f : 1.f;      // 2^80, 2^-80
    lift = by * 127.f;
    top = live ? amax * by : 1.f;
    inv = 1.f / top;
    scale = amax < INFINITY ? amax / 127.f : __uint_as_float(0x7fc00000u);
  }
  __device__ __forceinline__ int code(float v) const {
    const float x = v * lift, t = x * inv;
    return live ? (int)rintf(fmaf(fmaf(-t, top, x), inv, t)) : 0;
  }
};

// 8 consecutive elements, at any alignment: gfx950 serves wide unaligned accesses
template <typename T> struct Raw8 { uint32_t w[8 * sizeof(T) / 4]; };      // 8 elements as they lie in memory
template <typename T> __device__ __forceinline__ Raw8<T> ld_raw8(const T* p) {
  Raw8<T> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
__device__ __forceinline__ void widen8(const Raw8<float>& r, float v[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(r.w[e]);
}
__device__ __forceinline__ void widen8(const Raw8<f16_t>& r, float v[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) unpack2<f16_t>(r.w[e], v[2 * e], v[2 * e + 1]);
}
__device__ __forceinline__ void widen8(const Raw8<bf16_t>& r, float v[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) unpack2<bf16_t>(r.w[e], v[2 * e], v[2 * e + 1]);
}
template <typename T> __device__ __forceinline__ void st8(T* p, const float v[8]) {
  T t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = to_T<T>(v[e]);
  __builtin_memcpy(p, t, sizeof(t));
}

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return (uint32_t)(a & 255) | ((uint32_t)(b & 255) << 8) | ((uint32_t)(c & 255) << 16) | ((uint32_t)d << 24);
}

}  // namespace wj
