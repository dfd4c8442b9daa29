// Arithmetic of one step of the gated linear recurrence (forward and gradients), shared
// by the kernels of both directions.
//
//   z = -c softplus(decay) sigmoid(r)      a = exp(z)          s = sqrt(1 - a^2)
//   h_t = a h_{t-1} + s sigmoid(i) x
//
// and backwards, with g_t = dh_t + a_{t+1} g_{t+1}:
//
//   dx = g s sigmoid(i)                    di = dx x (1 - sigmoid(i))
//   dz = g (a h_{t-1} - (a^2 / s) sigmoid(i) x)
//   dr = dz z (1 - sigmoid(r))             ddecay = -c sigmoid(decay) sum dz sigmoid(r)
//
// Everything is computed in fp32. 1 - a comes from the series of 1 - exp(z) where z is
// small, so that a close to 1 (memories of thousands of steps) loses nothing, and a from
// the exponential where it is not, so that neither does an a close to 0:
// s = sqrt((1 - a)(1 + a)). Where s^2 is 0 or subnormal (a closed gate) 1 / s is held
// at its value for the smallest normal s^2: its product with z tends to 0.
#pragma once

#include "recurrence.h"
#include "vec_io.cuh"

namespace su {

// V channels of a thread. Pairs of them go through the packed fp32 instructions (one issue
// slot for two products or sums, each rounded as its scalar form): the kernels of bf16 inputs
// are bound by issue slots and the special-function unit, not by bytes.
template <int V>
struct Vf {
  float v[V];
  __device__ __forceinline__ float& operator[](int i) { return v[i]; }
  __device__ __forceinline__ float operator[](int i) const { return v[i]; }
};

__device__ __forceinline__ void pair_fma(float& d0, float& d1, float a0, float a1, float b0, float b1, float c0,
                                         float c1) {
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void pair_mul(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void pair_add(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}

template <int V>
__device__ __forceinline__ Vf<V> splat(float x) {
  Vf<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = x;
  return r;
}
template <int V>
__device__ __forceinline__ Vf<V> fma(const Vf<V>& a, const Vf<V>& b, const Vf<V>& c) {
  Vf<V> r;
  if constexpr (V == 1) {
    r.v[0] = fmaf(a.v[0], b.v[0], c.v[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2)
      pair_fma(r.v[i], r.v[i + 1], a.v[i], a.v[i + 1], b.v[i], b.v[i + 1], c.v[i], c.v[i + 1]);
  }
  return r;
}
template <int V>
__device__ __forceinline__ Vf<V> operator*(const Vf<V>& a, const Vf<V>& b) {
  Vf<V> r;
  if constexpr (V == 1) {
    r.v[0] = __fmul_rn(a.v[0], b.v[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) pair_mul(r.v[i], r.v[i + 1], a.v[i], a.v[i + 1], b.v[i], b.v[i + 1]);
  }
  return r;
}
template <int V>
__device__ __forceinline__ Vf<V> operator+(const Vf<V>& a, const Vf<V>& b) {
  Vf<V> r;
  if constexpr (V == 1) {
    r.v[0] = __fadd_rn(a.v[0], b.v[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) pair_add(r.v[i], r.v[i + 1], a.v[i], a.v[i + 1], b.v[i], b.v[i + 1]);
  }
  return r;
}
// 1 - a
template <int V>
__device__ __forceinline__ Vf<V> rest_of(const Vf<V>& a) {
  return fma(a, splat<V>(-1.f), splat<V>(1.f));
}
template <int V>
__device__ __forceinline__ Vf<V> sigmoid(const Vf<V>& a) {
  Vf<V> e = a * splat<V>(-kLog2e);
#pragma unroll
  for (int i = 0; i < V; ++i) e.v[i] = ex2_f(e.v[i]);
  e = e + splat<V>(1.f);
#pragma unroll
  for (int i = 0; i < V; ++i) e.v[i] = rcp_f(e.v[i]);
  return e;
}


// a = exp(-y) and em = 1 - a for V values y >= 0, each to a few units of its own last place: the
// gradients are multiples of a where it is small and of em where that is. Where y <= 0.25 em is Taylor's
// series up to y^6 (remainder below 0.25^6 / 7! = 5e-8 of it) and a the rest, above 0.77; elsewhere a is
// the exponential and em the rest, above 0.22. A thread whose V values are all small, the rule for
// a memory of many steps, branches past the exponentials: the special-function unit is what
// bounds bf16 inputs.
template <int V>
struct Decay {
  Vf<V> a, em;
};
template <int V>
__device__ __forceinline__ Decay<V> decay_from(const Vf<V>& y) {
  Vf<V> t = fma(y, splat<V>(-1.f / 720.f), splat<V>(1.f / 120.f));
  t = fma(y, t, splat<V>(-1.f / 24.f));
  t = fma(y, t, splat<V>(1.f / 6.f));
  t = fma(y, t, splat<V>(-0.5f));
  t = fma(y, t, splat<V>(1.f));
  Decay<V> d;
  d.em = y * t;
  d.a = rest_of(d.em);
  float most = y.v[0];
#pragma unroll
  for (int i = 1; i < V; ++i) most = fmaxf(most, y.v[i]);
  if (most > 0.25f) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float e = ex2_f(-kLog2e * y.v[i]);
      d.a.v[i] = y.v[i] > 0.25f ? e : d.a.v[i];
      d.em.v[i] = y.v[i] > 0.25f ? 1.f - e : d.em.v[i];
    }
  }
  return d;
}

// c softplus(decay), so that z = -k sigmoid(r)
__device__ __forceinline__ float decay_factor(float decay, float rate) {
  return rate * (fmaxf(decay, 0.f) + log1pf(expf(-fabsf(decay))));
}

// What a step maps the state with: h -> a h + add.
template <int V>
struct Step {
  Vf<V> a, add;
};
template <int V>
__device__ __forceinline__ Step<V> step_of(const Vf<V>& x, const Vf<V>& r, const Vf<V>& i, const Vf<V>& k) {
  const Decay<V> d = decay_from(k * sigmoid(r));
  Step<V> g;
  g.a = d.a;
  Vf<V> s = fma(d.em, d.a, d.em);
#pragma unroll
  for (int v = 0; v < V; ++v) s.v[v] = sqrt_f(s.v[v]);
  g.add = s * sigmoid(i) * x;
  return g;
}
template <int V>
__device__ __forceinline__ Vf<V> decay_of(const Vf<V>& r, const Vf<V>& k) {
  return decay_from(k * sigmoid(r)).a;
}

// One step's gradients are products with g, the gradient at h_t: dx = g x, dr = g r,
// di = g i, the share of ddecay's sum is -g l and a g goes on to h_{t-1}. `Gate` is what the
// inputs alone give; the state before the step turns it into `Slope`. Each is evaluated once.
template <int V>
struct Gate {
  Vf<V> a, x, i, add, q, y, sr;
};
template <int V>
__device__ __forceinline__ Gate<V> gate_of(const Vf<V>& x, const Vf<V>& r, const Vf<V>& i, const Vf<V>& k) {
  Gate<V> g;
  g.sr = sigmoid(r);
  const Vf<V> si = sigmoid(i);
  const Vf<V> y = k * g.sr;  // -z
  const Decay<V> d = decay_from(y);
  g.a = d.a;
  const Vf<V> ss = fma(d.em, d.a, d.em);
  Vf<V> rs;
#pragma unroll
  for (int v = 0; v < V; ++v) rs.v[v] = rsqrt_f(fmaxf(ss.v[v], 1.2e-38f));  // finite where the gate is closed: s, z 0
  g.x = ss * rs * si;
  g.add = g.x * x;
  g.i = g.add * rest_of(si);
  g.q = g.a * rs * (si * x);
  g.y = y * rest_of(g.sr);
  return g;
}
// Inputs of a step that leaves the state as it is: sigmoid(r) = 0, so a = 1 and s = 0.
template <int V>
__device__ __forceinline__ void shut(Vf<V>& x, Vf<V>& r, Vf<V>& i) {
  x = splat<V>(0.f);
  r = splat<V>(-1e30f);
  i = splat<V>(0.f);
}

template <int V>
struct Slope {
  Vf<V> a, x, r, i, l;
};
// at the state before the step, which moves on to h_t
template <int V>
__device__ __forceinline__ Slope<V> slope_of(const Gate<V>& g, Vf<V>& h) {
  const Vf<V> f = g.a * fma(h, splat<V>(-1.f), g.q);  // -(a h - (a^2 / s) sigmoid(i) x)
  h = fma(g.a, h, g.add);
  return Slope<V>{g.a, g.x, f * g.y, g.i, f * g.sr};
}

}  // namespace su
