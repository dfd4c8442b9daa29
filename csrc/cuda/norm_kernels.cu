// Norms before and after a block, fused with the block's gate and residual scale. Per row:
//
//   v = u rsqrt(mean u^2 + eps) w_post       t = scale sigmoid(gate)
//   y = x + t v                              n = y rsqrt(mean y^2 + eps) w_pre
//
// and backwards, with ru, ry the two rsqrt, uh = u ru, yh = y ry and q = dn w_pre:
//
//   dx = dy + ry (q - yh mean(q yh))         dw_pre = sum dn yh
//   dgate = dx scale v sigmoid'(gate)        dscale = sum dx sigmoid(gate) v
//   p = dx t w_post                          dw_post = sum dx t uh
//   du = ru (p - uh mean(p uh))
//
// A row belongs to one team of threads that keeps it in registers, so every input is read
// once and the statistics cost shuffles only. The backward pass recomputes y and both
// statistics from x, u and gate (or from their 8-bit codes) instead of reading y: the
// bytes are the same and nothing that was rounded to bf16 enters the gradients.
#include "kernels.h"
#include "recurrence.h"
#include "vec_io.cuh"

namespace su {
namespace {

// A team: `size` neighbouring threads (a power of two up to a warp, or the whole block).
struct Team {
  int size;
  int block;  // threads of a block
};

// Sums of N values over the team, the same on every thread, in a fixed order. For
// whole-block teams `box` alternates between two halves, so one barrier per call does.
template <int N>
__device__ __forceinline__ void team_sum(const Team& T, float (&v)[N], float (*box)[N][32], int& turn) {
  const int width = min(T.size, 32);
  for (int o = width / 2; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  if (T.size <= 32) return;
  const int warp = threadIdx.x / 32, warps = T.size / 32;
  float(*b)[32] = box[turn];
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) b[i][warp] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = 0.f;
    for (int w = 0; w < warps; ++w) s += b[i][w];
    v[i] = s;
  }
}

// Column of a thread's vector j: vectors of the team side by side, so a group of 32
// columns is held by 32 / V neighbouring lanes.
template <class T, int V, int NV, int MAXT, bool CODES>
__global__ void __launch_bounds__(MAXT) norm_fwd_kernel(const NormArgs A, const Team M) {
  __shared__ float box[2][1][32];
  int turn = 0;
  const int team = threadIdx.x / M.size, lane = threadIdx.x % M.size, teams = M.block / M.size;
  const int H = A.width;
  const int G = (H + kGroup8 - 1) / kGroup8;
  const float over = 1.f / static_cast<float>(H);
  float wp[NV][V], wn[NV][V], sc[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (j * M.size + lane) * V + v;
      wp[j][v] = (c < H && A.w_post != nullptr) ? param_at(A.w_post, A.post_bf16, c) : 1.f;
      wn[j][v] = (c < H && A.w_pre != nullptr) ? param_at(A.w_pre, A.pre_bf16, c) : 1.f;
      sc[j][v] = (c < H && A.scale != nullptr) ? param_at(A.scale, A.scale_bf16, c) : 1.f;
    }
  // every thread of a block makes the same number of rounds (shuffles and barriers inside)
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * teams; r0 < A.rows; r0 += static_cast<int64_t>(gridDim.x) * teams) {
    const int64_t row = r0 + team;
    const bool in = row < A.rows;
    float x[NV][V], u[NV][V], g[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * M.size + lane) * V;
      Pack<T, V> a, b, d;
      a.zero();
      b.zero();
      d.zero();
      if (in && c < H) {
        a.load(static_cast<const T*>(A.x) + row * A.x_ld + c);
        if (A.u != nullptr) b.load(static_cast<const T*>(A.u) + row * A.u_ld + c);
        if (A.gate != nullptr) d.load(static_cast<const T*>(A.gate) + row * A.gate_ld + c);
      }
      a.get(x[j]);
      b.get(u[j]);
      d.get(g[j]);
    }
    if constexpr (CODES) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * M.size + lane) * V;
        const bool live = in && c < H;
        Codes<V> q;
        int8_t* to = A.codes + row * H + c;
        float* ts = A.scales + row * G + c / kGroup8;
        const int64_t part = A.rows * H, spart = A.rows * G;
        const bool first = live && c % kGroup8 == 0;
        float s = encode8(x[j], q);
        if (live) q.store(to);
        if (first) ts[0] = s;
        if (A.u != nullptr) {
          s = encode8(u[j], q);
          if (live) q.store(to + part);
          if (first) ts[spart] = s;
        }
        if (A.gate != nullptr) {
          s = encode8(g[j], q);
          if (live) q.store(to + 2 * part);
          if (first) ts[2 * spart] = s;
        }
      }
    }
    if (A.u != nullptr) {
      float ru = 1.f;
      if (A.w_post != nullptr) {
        float q[1] = {0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int v = 0; v < V; ++v) q[0] = fmaf(u[j][v], u[j][v], q[0]);
        team_sum(M, q, box, turn);
        ru = rsqrtf(q[0] * over + A.eps);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * M.size + lane) * V;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float t = sc[j][v] * (A.gate != nullptr ? sigmoid_f(g[j][v]) : 1.f);
          x[j][v] = fmaf(t, u[j][v] * ru * wp[j][v], x[j][v]);
        }
        if (in && c < H && A.y != nullptr) {
          Pack<T, V> o;
          o.set(x[j]);
          o.store(static_cast<T*>(A.y) + row * H + c);
        }
      }
    }
    if (A.n != nullptr) {
      float q[1] = {0.f};
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) q[0] = fmaf(x[j][v], x[j][v], q[0]);
      team_sum(M, q, box, turn);
      const float ry = rsqrtf(q[0] * over + A.eps);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * M.size + lane) * V;
        if (in && c < H) {
          float f[V];
#pragma unroll
          for (int v = 0; v < V; ++v) f[v] = x[j][v] * ry * wn[j][v];
          Pack<T, V> o;
          o.set(f);
          o.store(static_cast<T*>(A.n) + row * H + c);
        }
      }
    }
  }
}

template <class T, int V, int NV, int MAXT, bool CODES>
__global__ void __launch_bounds__(MAXT) norm_bwd_kernel(const NormArgs A, const Team M) {
  __shared__ float box1[2][1][32];
  __shared__ float box2[2][2][32];
  extern __shared__ float sums[];  // [teams][size * NV * V] of one parameter at a time
  int turn1 = 0, turn2 = 0;
  const int team = threadIdx.x / M.size, lane = threadIdx.x % M.size, teams = M.block / M.size;
  const int H = A.width;
  const int G = (H + kGroup8 - 1) / kGroup8;
  const float over = 1.f / static_cast<float>(H);
  float wp[NV][V], wn[NV][V], sc[NV][V], gp[NV][V], gn[NV][V], gs[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (j * M.size + lane) * V + v;
      wp[j][v] = (c < H && A.w_post != nullptr) ? param_at(A.w_post, A.post_bf16, c) : 1.f;
      wn[j][v] = (c < H && A.w_pre != nullptr) ? param_at(A.w_pre, A.pre_bf16, c) : 1.f;
      sc[j][v] = (c < H && A.scale != nullptr) ? param_at(A.scale, A.scale_bf16, c) : 1.f;
      gp[j][v] = gn[j][v] = gs[j][v] = 0.f;
    }
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * teams; r0 < A.rows; r0 += static_cast<int64_t>(gridDim.x) * teams) {
    const int64_t row = r0 + team;
    const bool in = row < A.rows;
    float x[NV][V], u[NV][V], g[NV][V], dy[NV][V], dn[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * M.size + lane) * V;
#pragma unroll
      for (int v = 0; v < V; ++v) x[j][v] = u[j][v] = g[j][v] = dy[j][v] = dn[j][v] = 0.f;
      if (in && c < H) {
        Pack<T, V> a;
        if constexpr (CODES) {
          const int8_t* from = A.codes + row * H + c;
          const float* fs = A.scales + row * G + c / kGroup8;
          const int64_t part = A.rows * H, spart = A.rows * G;
          Codes<V> q;
          q.load(from);
          q.get(fs[0], x[j]);
          if (A.u != nullptr) {
            q.load(from + part);
            q.get(fs[spart], u[j]);
          }
          if (A.gate != nullptr) {
            q.load(from + 2 * part);
            q.get(fs[2 * spart], g[j]);
          }
        } else {
          a.load(static_cast<const T*>(A.x) + row * A.x_ld + c);
          a.get(x[j]);
          if (A.u != nullptr) {
            a.load(static_cast<const T*>(A.u) + row * A.u_ld + c);
            a.get(u[j]);
          }
          if (A.gate != nullptr) {
            a.load(static_cast<const T*>(A.gate) + row * A.gate_ld + c);
            a.get(g[j]);
          }
        }
        if (A.dy != nullptr) {
          a.load(static_cast<const T*>(A.dy) + row * A.dy_ld + c);
          a.get(dy[j]);
        }
        if (A.dn != nullptr) {
          a.load(static_cast<const T*>(A.dn) + row * A.dn_ld + c);
          a.get(dn[j]);
        }
      }
    }
    // y in the place of x, sigmoid(gate) in the place of gate
    float ru = 1.f;
    if (A.u != nullptr) {
      if (A.w_post != nullptr) {
        float q[1] = {0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int v = 0; v < V; ++v) q[0] = fmaf(u[j][v], u[j][v], q[0]);
        team_sum(M, q, box1, turn1);
        ru = rsqrtf(q[0] * over + A.eps);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          g[j][v] = A.gate != nullptr ? sigmoid_f(g[j][v]) : 1.f;
          u[j][v] *= ru;
          x[j][v] = fmaf(sc[j][v] * g[j][v], u[j][v] * wp[j][v], x[j][v]);
        }
    }
    if (A.dn != nullptr) {
      float q[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          q[0] = fmaf(x[j][v], x[j][v], q[0]);
          q[1] = fmaf(dn[j][v] * wn[j][v], x[j][v], q[1]);
        }
      team_sum(M, q, box2, turn2);
      const float ry = rsqrtf(q[0] * over + A.eps);
      const float m = q[1] * ry * over;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float yh = x[j][v] * ry;
          gn[j][v] = fmaf(dn[j][v], yh, gn[j][v]);
          dy[j][v] = fmaf(ry, fmaf(-yh, m, dn[j][v] * wn[j][v]), dy[j][v]);
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * M.size + lane) * V;
      if (in && c < H && A.dx != nullptr) {
        Pack<T, V> o;
        o.set(dy[j]);
        o.store(static_cast<T*>(A.dx) + row * H + c);
      }
    }
    if (A.u == nullptr) continue;
    float q[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * M.size + lane) * V;
      float dg[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float vv = u[j][v] * wp[j][v];
        const float ds = dy[j][v] * g[j][v];
        gs[j][v] = fmaf(ds, vv, gs[j][v]);
        dg[v] = ds * sc[j][v] * vv * (1.f - g[j][v]);
        const float dv = ds * sc[j][v];
        gp[j][v] = fmaf(dv, u[j][v], gp[j][v]);
        dn[j][v] = dv * wp[j][v];
        q[0] = fmaf(dn[j][v], u[j][v], q[0]);
      }
      if (in && c < H && A.dgate != nullptr) {
        Pack<T, V> o;
        o.set(dg);
        o.store(static_cast<T*>(A.dgate) + row * H + c);
      }
    }
    float m = 0.f;
    if (A.w_post != nullptr) {
      team_sum(M, q, box1, turn1);
      m = q[0] * over;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * M.size + lane) * V;
      if (in && c < H && A.du != nullptr) {
        float f[V];
#pragma unroll
        for (int v = 0; v < V; ++v) f[v] = ru * fmaf(-u[j][v], m, dn[j][v]);
        Pack<T, V> o;
        o.set(f);
        o.store(static_cast<T*>(A.du) + row * H + c);
      }
    }
  }
  // the block's share of the three column sums, its teams added up in order
  const int span = M.size * NV * V;
#pragma unroll
  for (int w = 0; w < 3; ++w) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v)
        sums[team * span + (j * M.size + lane) * V + v] = w == 0 ? gp[j][v] : w == 1 ? gn[j][v] : gs[j][v];
    __syncthreads();
    for (int c = threadIdx.x; c < min(span, H); c += blockDim.x) {
      float t = 0.f;
      for (int k = 0; k < teams; ++k) t += sums[k * span + c];
      A.partial[(static_cast<int64_t>(blockIdx.x) * 3 + w) * H + c] = t;
    }
  }
}

// partial [n, 3, H] added up in order: 32 columns x 32 shares per block
__global__ void norm_param_grad_kernel(const NormArgs A) {
  __shared__ float sum[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x, w = blockIdx.y;
  void* out = w == 0 ? A.dw_post : w == 1 ? A.dw_pre : A.dscale;
  if (out == nullptr) return;
  float t = 0.f;
  if (c < A.width)
    for (int k = threadIdx.y; k < A.n_partial; k += 32) t += A.partial[(static_cast<int64_t>(k) * 3 + w) * A.width + c];
  sum[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.y == 0 && c < A.width) {
    for (int k = 1; k < 32; ++k) t += sum[k][threadIdx.x];
    param_store(out, w == 0 ? A.post_bf16 : w == 1 ? A.pre_bf16 : A.scale_bf16, c, t);
  }
}

// Smallest team whose threads hold at most `nv` vectors each, at least a whole 8-bit group
// wide; blocks of up to 256 threads (more registers each) where `most` vectors a thread do.
struct Shape {
  Team team;
  int V, NV;
};
Shape shape_of(const NormArgs& a, int nv, int most) {
  Shape s;
  s.V = a.vec ? 4 : 1;
  const int vecs = (a.width + s.V - 1) / s.V;
  int size = kGroup8 / s.V;
  const int limit = vecs <= 256 * most ? 256 : 1024;
  while (size < limit && size * nv < vecs) size *= 2;
  s.team = {size, size <= 32 ? 256 : size};
  s.NV = 1;
  while (s.NV * size < vecs) s.NV *= 2;
  return s;
}
int norm_blocks(const NormArgs& a, const Shape& s, int sms) {
  const int teams = s.team.block / s.team.size;
  const int64_t want = (a.rows + teams - 1) / teams;
  const int64_t most = static_cast<int64_t>(sms) * (s.team.block <= 256 ? 8 : 2);
  return static_cast<int>(want < most ? want : most);
}
Shape fwd_shape(const NormArgs& a) { return shape_of(a, a.vec ? 2 : 4, a.vec ? 4 : 8); }
Shape bwd_shape(const NormArgs& a) { return shape_of(a, a.vec ? 2 : 4, a.vec ? 2 : 8); }

template <class T, int V, int NV, int MAXT, bool CODES>
void run_fwd(const NormArgs& a, const Shape& s, int sms, cudaStream_t st) {
  norm_fwd_kernel<T, V, NV, MAXT, CODES><<<norm_blocks(a, s, sms), s.team.block, 0, st>>>(a, s.team);
}
template <class T, int V, int NV, int MAXT, bool CODES>
void run_bwd(const NormArgs& a, const Shape& s, int sms, cudaStream_t st) {
  const size_t smem = static_cast<size_t>(s.team.block) * NV * V * sizeof(float);
  if (smem > 40 * 1024)
    cudaFuncSetAttribute(norm_bwd_kernel<T, V, NV, MAXT, CODES>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         static_cast<int>(smem));
  norm_bwd_kernel<T, V, NV, MAXT, CODES><<<norm_blocks(a, s, sms), s.team.block, smem, st>>>(a, s.team);
}

template <class T, bool CODES, bool BWD>
void run_norm(const NormArgs& a, int sms, cudaStream_t st) {
  const Shape s = BWD ? bwd_shape(a) : fwd_shape(a);
  const bool small = s.team.block <= 256;
#define SU_NORM_CASE(V_, NV_, MAXT_)                    \
  if (s.V == V_ && s.NV == NV_ && small == (MAXT_ == 256)) { \
    if constexpr (BWD)                                  \
      run_bwd<T, V_, NV_, MAXT_, CODES>(a, s, sms, st); \
    else                                                \
      run_fwd<T, V_, NV_, MAXT_, CODES>(a, s, sms, st); \
    return;                                             \
  }
  // a team is grown until 2 (vectors of 4) or 4 (single values) a thread are enough, or to its limit
  SU_NORM_CASE(4, 1, 256)
  SU_NORM_CASE(4, 2, 256)
  if constexpr (!BWD) {
    SU_NORM_CASE(4, 4, 256)
  }
  SU_NORM_CASE(4, 2, 1024)
  SU_NORM_CASE(4, 4, 1024)
  SU_NORM_CASE(1, 1, 256)
  SU_NORM_CASE(1, 2, 256)
  SU_NORM_CASE(1, 4, 256)
  SU_NORM_CASE(1, 8, 256)
  SU_NORM_CASE(1, 4, 1024)
  SU_NORM_CASE(1, 8, 1024)
  SU_NORM_CASE(1, 16, 1024)
#undef SU_NORM_CASE
}

}  // namespace

int norm_partials(const NormArgs& a, int sms) { return norm_blocks(a, bwd_shape(a), sms); }

void launch_norm_fwd(const NormArgs& a, int sms, cudaStream_t st) {
  count_launch();
  const bool codes = a.codes != nullptr;
  if (a.bf16)
    codes ? run_norm<__nv_bfloat16, true, false>(a, sms, st) : run_norm<__nv_bfloat16, false, false>(a, sms, st);
  else
    codes ? run_norm<float, true, false>(a, sms, st) : run_norm<float, false, false>(a, sms, st);
}

void launch_norm_bwd(const NormArgs& a, int sms, cudaStream_t st) {
  const bool codes = a.codes != nullptr;
  count_launch();
  if (a.bf16)
    codes ? run_norm<__nv_bfloat16, true, true>(a, sms, st) : run_norm<__nv_bfloat16, false, true>(a, sms, st);
  else
    codes ? run_norm<float, true, true>(a, sms, st) : run_norm<float, false, true>(a, sms, st);
  if (a.dw_post == nullptr && a.dw_pre == nullptr && a.dscale == nullptr) return;
  count_launch();
  norm_param_grad_kernel<<<dim3((a.width + 31) / 32, 3), dim3(32, 32), 0, st>>>(a);
}

}  // namespace su
