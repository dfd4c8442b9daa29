// Vector loads and stores of V neighbouring fp32 or bf16 values per thread, and
// the 8-bit group codes that several kernels read and write.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "common.cuh"
#include "recurrence.h"

namespace su {

#ifdef __CUDACC__

template <int BYTES>
struct RawOf;
template <>
struct RawOf<1> { using type = uint8_t; };
template <>
struct RawOf<2> { using type = uint16_t; };
template <>
struct RawOf<4> { using type = uint32_t; };
template <>
struct RawOf<8> { using type = uint2; };
template <>
struct RawOf<16> { using type = uint4; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v) {  // round to nearest even
  if constexpr (sizeof(T) == 2)
    return __float2bfloat16(v);
  else
    return v;
}

// V values of T as one register vector; the address is V * sizeof(T) aligned.
template <class T, int V>
struct Pack {
  using Raw = typename RawOf<sizeof(T) * V>::type;
  Raw raw;
  __device__ __forceinline__ void load(const T* p) { raw = __ldcs(reinterpret_cast<const Raw*>(p)); }
  __device__ __forceinline__ void zero() { raw = Raw{}; }
  __device__ __forceinline__ void get(float (&f)[V]) const {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f32(e[i]);
  }
  __device__ __forceinline__ void set(const float (&f)[V]) {
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_f32<T>(f[i]);
  }
  __device__ __forceinline__ void store(T* p) const { __stcs(reinterpret_cast<Raw*>(p), raw); }
};

// one value of a parameter vector held in fp32 or bf16
__device__ __forceinline__ float param_at(const void* p, int is_bf16, int64_t i) {
  return is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void param_store(void* p, int is_bf16, int64_t i, float v) {
  if (is_bf16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16(v);
  else
    static_cast<float*>(p)[i] = v;
}

// Logistic function: ex2 and reciprocal approximations, ~2e-7 relative. exp(-v) = inf gives 0.
__device__ __forceinline__ float sigmoid_f(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }

// ---------------------------------------------------------------------------
// 8-bit codes: per group of 32 values of a row, scale = amax / 127 and
// code = rint(v * (127 / amax)). The largest magnitude is taken on the bits, so
// NaN and infinity win; such a group gets the scale NaN (all of it reads back as
// NaN), a group below 2^-100 the scale 0 (127 / amax would overflow).
// ---------------------------------------------------------------------------
struct Scale8 {
  float inv;
  float scale;
};
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ Scale8 scale8(uint32_t top) {
  Scale8 s;
  const float amax = __uint_as_float(top);
  s.inv = __fdiv_rn(127.f, amax);
  s.scale = __fmul_rn(amax, static_cast<float>(1.0 / 127.0));
  if (top < 0x0d800000u) {  // 2^-100
    s.inv = 0.f;
    s.scale = 0.f;
  } else if (top >= 0x7f800000u) {
    s.inv = 0.f;
    s.scale = __uint_as_float(0x7fc00000u);
  }
  return s;
}

// The largest magnitude of a group that LANES neighbouring lanes hold (LANES a power of
// two, aligned inside the warp; every lane of the group calls).
template <int LANES>
__device__ __forceinline__ uint32_t group_top(uint32_t top) {
  const unsigned lane = threadIdx.x & 31;
  const unsigned mask = LANES == 32 ? 0xffffffffu : (((1u << LANES) - 1u) << (lane & ~(LANES - 1u)));
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(mask, top, o));
  return top;
}

// codes and scale of V values per lane
template <int V>
__device__ __forceinline__ float encode8(const float (&f)[V], int8_t (&code)[V]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) top = max(top, abs_bits(f[i]));
  const Scale8 s = scale8(group_top<kGroup8 / V>(top));
  // inv = 0 and f = inf would be NaN, which converts to 0 as well
#pragma unroll
  for (int i = 0; i < V; ++i) code[i] = static_cast<int8_t>(__float2int_rn(__fmul_rn(f[i], s.inv)));
  return s.scale;
}

template <int V>
__device__ __forceinline__ void store_codes(int8_t* p, const int8_t (&code)[V]) {
  typename RawOf<V>::type raw;
  int8_t* e = reinterpret_cast<int8_t*>(&raw);
#pragma unroll
  for (int i = 0; i < V; ++i) e[i] = code[i];
  __stcs(reinterpret_cast<typename RawOf<V>::type*>(p), raw);
}
template <int V>
__device__ __forceinline__ void load_codes(const int8_t* p, float scale, float (&f)[V]) {
  const typename RawOf<V>::type raw = __ldcs(reinterpret_cast<const typename RawOf<V>::type*>(p));
  const int8_t* e = reinterpret_cast<const int8_t*>(&raw);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = __fmul_rn(static_cast<float>(e[i]), scale);
}

#endif  // __CUDACC__

}  // namespace su
