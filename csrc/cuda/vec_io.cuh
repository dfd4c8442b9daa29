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
  // for values that a later pass reads again
  __device__ __forceinline__ void load_keep(const T* p) { raw = __ldg(reinterpret_cast<const Raw*>(p)); }
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

// Copies of 4, 8 or 16 bytes from global to shared memory that the thread does not wait for:
// committed in groups, of which wait_copies leaves the newest N under way. What a thread
// copied is its own to read after that.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* smem, const void* p) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(p) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(smem)), "l"(p), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

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

// Single instructions of the special-function unit (each within 2 ulp or so), subnormals
// flushed: the plain functions spend several instructions more on subnormals.
__device__ __forceinline__ float ex2_f(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp_f(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float sqrt_f(float v) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rsqrt_f(float v) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// Logistic function, ~3e-7 relative; exp(-v) = inf gives 0.
__device__ __forceinline__ float sigmoid_f(float v) { return rcp_f(1.f + ex2_f(-kLog2e * v)); }

// ---------------------------------------------------------------------------
// 8-bit codes: per group of 32 values of a row, scale = amax / 127 and
// code = rint(v * (127 / amax)). A NaN or an infinity wins the maximum; such a group gets
// the scale NaN (all of it reads back as NaN) and codes 0, a group below 2^-100 the scale 0
// (127 / amax would overflow).
//
// Rounding and conversion go through the FMA pipe: v + 1.5 * 2^23 rounds v to an integer
// (to nearest even) and has it in its low bits; the conversion instructions run at the
// special-function unit's rate, which the kernels that encode and decode need for
// exponentials.
// ---------------------------------------------------------------------------
struct Scale8 {
  float inv;
  float scale;
  bool bad;
};
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ Scale8 scale8(float amax) {
  Scale8 s;
  s.bad = !(amax < __int_as_float(0x7f800000));
  const bool tiny = amax < 7.888609052210118e-31f;  // 2^-100
  s.inv = tiny ? 0.f : __fdiv_rn(127.f, amax);
  s.scale = tiny ? 0.f : __fmul_rn(amax, static_cast<float>(1.0 / 127.0));
  if (s.bad) s.scale = __int_as_float(0x7fc00000);
  return s;
}

// The largest magnitude of a group that FULL neighbouring lanes hold, or with NARROW `lanes` of
// them (powers of two, aligned inside the warp; every lane of the group calls).
template <int FULL, bool NARROW>
__device__ __forceinline__ float group_top(float top, int lanes) {
  const unsigned lane = threadIdx.x & 31;
  if constexpr (!NARROW) {
    const unsigned mask = FULL == 32 ? 0xffffffffu : (((1u << FULL) - 1u) << (lane & ~(FULL - 1u)));
#pragma unroll
    for (int o = FULL / 2; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(mask, top, o));
  } else {
    const unsigned mask = ((1u << lanes) - 1u) << (lane & ~(lanes - 1u));
    for (int o = lanes / 2; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(mask, top, o));
  }
  return top;
}
// Lanes that a group takes at V values each: fewer than 32 / V where the row is less than a group
// (NARROW kernels; the others unroll their five, four or three exchanges).
__host__ __device__ inline int group_lanes(int width, int V) {
  int lanes = 1;
  while (lanes < kGroup8 / V && lanes * V < width) lanes *= 2;
  return lanes;
}

// V codes side by side, lowest address first
template <int V>
struct Codes {
  typename RawOf<V>::type raw;
  __device__ __forceinline__ void store(int8_t* p) const { __stcs(reinterpret_cast<typename RawOf<V>::type*>(p), raw); }
  __device__ __forceinline__ void load(const int8_t* p) { raw = __ldcs(reinterpret_cast<const typename RawOf<V>::type*>(p)); }
  __device__ __forceinline__ void zero() { raw = 0; }
  __device__ __forceinline__ void get(float scale, float (&f)[V]) const {
    const uint32_t word = static_cast<uint32_t>(raw) ^ 0x80808080u;  // code + 128, 0 to 255
#pragma unroll
    for (int i = 0; i < V; ++i) {
      // 2^23 + (code + 128), exactly
      const float t = __uint_as_float(__byte_perm(word, 0x4b000000u, 0x7440 + i));
      f[i] = __fmul_rn(t - (8388608.f + 128.f), scale);
    }
  }
};

// codes of V values per lane, `lanes` lanes a group where NARROW; returns the group's scale
template <bool NARROW, int V>
__device__ __forceinline__ float encode8(const float (&f)[V], Codes<V>& code, int lanes) {
  float top = fabsf(f[0]);
#pragma unroll
  for (int i = 1; i < V; ++i) top = max_nan(top, fabsf(f[i]));
  const Scale8 s = scale8(group_top<kGroup8 / V, NARROW>(top, lanes));
  uint32_t n[V];
#pragma unroll
  for (int i = 0; i < V; ++i) n[i] = __float_as_uint(__fadd_rn(__fmul_rn(f[i], s.inv), 12582912.f));
  uint32_t word;
  if constexpr (V == 4)
    word = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
  else if constexpr (V == 2)
    word = __byte_perm(n[0], n[1], 0x0040);
  else
    word = n[0];
  code.raw = static_cast<typename RawOf<V>::type>(s.bad ? 0u : word);
  return s.scale;
}

#endif  // __CUDACC__

}  // namespace su
