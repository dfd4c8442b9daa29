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

// 1 - exp(z) for z <= 0. Taylor's series up to z^6 where |z| <= 0.25 (remainder below
// 0.25^6 / 7! = 5e-8 of the result), else the difference, which cancels at most two bits.
// The exponential is issued only where some lane of the warp needs it.
__device__ __forceinline__ float one_minus_exp(float z) {
  float t = fmaf(z, 1.f / 720.f, 1.f / 120.f);
  t = fmaf(z, t, 1.f / 24.f);
  t = fmaf(z, t, 1.f / 6.f);
  t = fmaf(z, t, 0.5f);
  t = fmaf(z, t, 1.f);
  float em = -z * t;
  if (z < -0.25f) em = 1.f - ex2_f(kLog2e * z);
  return em;
}

// -c softplus(decay)
__device__ __forceinline__ float decay_factor(float decay, float rate) {
  return -rate * (fmaxf(decay, 0.f) + log1pf(expf(-fabsf(decay))));
}

// What a step maps the state with: h -> a h + add.
struct Step {
  float a, add;
};
__device__ __forceinline__ Step step_of(float x, float r, float i, float k) {
  const float em = one_minus_exp(k * sigmoid_f(r));
  Step g;
  g.a = 1.f - em;
  g.add = sqrt_f(em * (1.f + g.a)) * sigmoid_f(i) * x;
  return g;
}
__device__ __forceinline__ float decay_of(float r, float k) { return 1.f - one_minus_exp(k * sigmoid_f(r)); }

// One step's gradients are products with g, the gradient at h_t: dx = g x, dr = g r,
// di = g i, the share of ddecay's sum is g l and a g goes on to h_{t-1}. `Gate` is what the
// inputs alone give; the state before the step turns it into `Slope`. Each is evaluated once.
struct Gate {
  float a, x, i, add, q, z, sr;
};
__device__ __forceinline__ Gate gate_of(float x, float r, float i, float k) {
  Gate g;
  g.sr = sigmoid_f(r);
  const float si = sigmoid_f(i);
  const float z = k * g.sr;
  const float em = one_minus_exp(z);
  g.a = 1.f - em;
  const float ss = em * (1.f + g.a);
  const float rs = rsqrt_f(fmaxf(ss, 1.2e-38f));  // finite where the gate is closed; s and z are 0 there
  g.x = ss * rs * si;
  g.add = g.x * x;
  g.i = fmaf(-g.add, si, g.add);
  g.q = g.a * rs * (si * x);
  g.z = fmaf(-z, g.sr, z);
  return g;
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
