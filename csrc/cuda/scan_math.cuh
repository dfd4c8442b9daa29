// Arithmetic of one step of the gated linear recurrence (forward and gradients), shared
// by the kernels that walk whole sequences and those that split them into tiles.
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
// s = sqrt((1 - a)(1 + a)). Where s^2 is 0 or subnormal (a closed gate) s and
// a^2 / s are taken as 0: the first is below 1.1e-19, the second's product with z tends to 0.
#pragma once

#include "recurrence.h"
#include "vec_io.cuh"

namespace su {

__device__ __forceinline__ float approx_sqrt(float v) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float approx_rsqrt(float v) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// 1 - exp(z) for z <= 0. Taylor's series up to z^7 where |z| < 0.4 (remainder below
// 0.4^7 / 8! = 4e-8 of the result), else the difference, which cancels at most two bits.
__device__ __forceinline__ float one_minus_exp(float z) {
  float t = fmaf(z, 1.f / 5040.f, 1.f / 720.f);
  t = fmaf(z, t, 1.f / 120.f);
  t = fmaf(z, t, 1.f / 24.f);
  t = fmaf(z, t, 1.f / 6.f);
  t = fmaf(z, t, 0.5f);
  t = fmaf(z, t, 1.f);
  return z > -0.4f ? -z * t : 1.f - __expf(z);
}

// -c softplus(decay)
__device__ __forceinline__ float decay_factor(float decay, float rate) {
  return -rate * (fmaxf(decay, 0.f) + log1pf(expf(-fabsf(decay))));
}

struct Step {
  float sr, si, z, a, ss;  // sigmoids, log decay, decay, s^2
};
__device__ __forceinline__ Step step_of(float r, float i, float k) {
  Step g;
  g.sr = sigmoid_f(r);
  g.si = sigmoid_f(i);
  g.z = k * g.sr;
  const float em = one_minus_exp(g.z);
  g.a = 1.f - em;
  g.ss = em * (2.f - em);
  return g;
}

// Gradients of one step at the state before it; returns what goes on to h_{t-1} (a g).
__device__ __forceinline__ float step_grad(const Step& t, float x, float before, float g, float& dx, float& dr,
                                           float& di, float& dl) {
  const float rs = t.ss > 1.2e-38f ? approx_rsqrt(t.ss) : 0.f;  // rsqrt.ftz of a subnormal is infinite
  const float s = t.ss * rs;
  dx = g * s * t.si;
  di = dx * x * (1.f - t.si);
  const float dz = g * (t.a * before - t.a * t.a * rs * t.si * x);
  dr = dz * t.z * (1.f - t.sr);
  dl = fmaf(dz, t.sr, dl);
  return t.a * g;
}

// A thread's V channels: lanes of a row side by side, rows over threadIdx / lanes.
struct Lanes {
  int count;   // lanes that one row takes in a block
  int rows;    // rows side by side in a block
  int blocks;  // blocks over the channels
};

// Lanes of H channels at V per lane, at most `most` lanes a row and `threads` threads a block;
// with 8-bit codes every group of 32 channels gets its own aligned lanes, the last one's
// beyond H included.
inline Lanes lanes_of(int width, int V, bool codes, int most, int threads) {
  const int unit = codes ? kGroup8 / V : 1;
  const int all = codes ? (width + kGroup8 - 1) / kGroup8 * unit : (width + V - 1) / V;
  Lanes l;
  l.blocks = (all + most - 1) / most;
  l.count = (all + l.blocks - 1) / l.blocks;
  l.count = (l.count + unit - 1) / unit * unit;
  l.rows = threads / l.count;
  return l;
}

}  // namespace su
