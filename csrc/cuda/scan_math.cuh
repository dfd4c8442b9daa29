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
// small, so that a close to 1 (memories of thousands of steps) loses nothing:
// s = sqrt((1 - a)(1 + a)). Where s^2 is 0 or subnormal (a closed gate) 1 / s is held
// at its value for the smallest normal s^2: its product with z tends to 0.
#pragma once

#include "recurrence.h"
#include "vec_io.cuh"

namespace su {

// 1 - exp(z) for V values z <= 0. Taylor's series up to z^6 where |z| <= 0.25 (remainder below
// 0.25^6 / 7! = 5e-8 of the result), else the difference, which cancels at most two bits. A
// thread whose V values are all small, the rule for a memory of many steps, branches past
// the exponentials: the special-function unit is what bounds bf16 inputs.
template <int V>
__device__ __forceinline__ void one_minus_exp(const float (&z)[V], float (&em)[V]) {
  float least = z[0];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float t = fmaf(z[v], 1.f / 720.f, 1.f / 120.f);
    t = fmaf(z[v], t, 1.f / 24.f);
    t = fmaf(z[v], t, 1.f / 6.f);
    t = fmaf(z[v], t, 0.5f);
    t = fmaf(z[v], t, 1.f);
    em[v] = -z[v] * t;
    least = fminf(least, z[v]);
  }
  if (least < -0.25f) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float e = 1.f - ex2_f(kLog2e * z[v]);
      em[v] = z[v] < -0.25f ? e : em[v];
    }
  }
}

// -c softplus(decay)
__device__ __forceinline__ float decay_factor(float decay, float rate) {
  return -rate * (fmaxf(decay, 0.f) + log1pf(expf(-fabsf(decay))));
}

// What a step maps the state with: h -> a h + add.
struct Step {
  float a, add;
};
template <int V>
__device__ __forceinline__ void steps_of(const float (&x)[V], const float (&r)[V], const float (&i)[V],
                                         const float (&k)[V], Step (&g)[V]) {
  float z[V], em[V];
#pragma unroll
  for (int v = 0; v < V; ++v) z[v] = k[v] * sigmoid_f(r[v]);
  one_minus_exp(z, em);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    g[v].a = 1.f - em[v];
    g[v].add = sqrt_f(em[v] * (1.f + g[v].a)) * sigmoid_f(i[v]) * x[v];
  }
}
template <int V>
__device__ __forceinline__ void decays_of(const float (&r)[V], const float (&k)[V], float (&a)[V]) {
  float z[V], em[V];
#pragma unroll
  for (int v = 0; v < V; ++v) z[v] = k[v] * sigmoid_f(r[v]);
  one_minus_exp(z, em);
#pragma unroll
  for (int v = 0; v < V; ++v) a[v] = 1.f - em[v];
}

// One step's gradients are products with g, the gradient at h_t: dx = g x, dr = g r,
// di = g i, the share of ddecay's sum is g l and a g goes on to h_{t-1}. `Gate` is what the
// inputs alone give; the state before the step turns it into `Slope`. Each is evaluated once.
struct Gate {
  float a, x, i, add, q, z, sr;
};
template <int V>
__device__ __forceinline__ void gates_of(const float (&x)[V], const float (&r)[V], const float (&i)[V],
                                         const float (&k)[V], Gate (&g)[V]) {
  float z[V], em[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    g[v].sr = sigmoid_f(r[v]);
    z[v] = k[v] * g[v].sr;
  }
  one_minus_exp(z, em);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float si = sigmoid_f(i[v]);
    g[v].a = 1.f - em[v];
    const float ss = em[v] * (1.f + g[v].a);
    const float rs = rsqrt_f(fmaxf(ss, 1.2e-38f));  // finite where the gate is closed; s and z are 0 there
    g[v].x = ss * rs * si;
    g[v].add = g[v].x * x[v];
    g[v].i = fmaf(-g[v].add, si, g[v].add);
    g[v].q = g[v].a * rs * (si * x[v]);
    g[v].z = fmaf(-z[v], g[v].sr, z[v]);
  }
}
// Inputs of a step that leaves the state as it is: sigmoid(r) = 0, so a = 1 and s = 0.
__device__ __forceinline__ void shut(float& x, float& r, float& i) {
  x = 0.f;
  r = -1e30f;
  i = 0.f;
}

struct Slope {
  float a, x, r, i, l;
};
// at the state before the step, which moves on to h_t
__device__ __forceinline__ Slope slope_of(const Gate& g, float& h) {
  const float f = g.a * (h - g.q);
  h = fmaf(g.a, h, g.add);
  return Slope{g.a, g.x, f * g.z, g.i, f * g.sr};
}

}  // namespace su
