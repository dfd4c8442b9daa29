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
// once and the statistics cost shuffles only. AHEAD: while a row is worked on, the next one of
// the team is copied to slots of shared memory that belong to the thread (no barrier needed).
// The backward pass recomputes y and both statistics from x, u and gate (or from their
// 8-bit codes) instead of reading y: the bytes are the same and nothing that was rounded
// to bf16 enters the gradients.
//
// Bound by bytes where a row fits a team inside a warp: 1,600,000 x 64 fp32 331 us forward and
// 495 backward, 6.2 and 6.6 TB/s. Wider rows pay the block's sums and the issue of three columns'
// gradients: 16,384 x 2048 bf16 64 and 158 us, 5.2 and 3.4 TB/s; with codes the encoding and
// decoding: 400,000 x 172 fp32 352 and 407 us.
#include "kernels.h"
#include "recurrence.h"
#include "vec_io.cuh"

namespace su {
namespace {

// 8-bit codes to write: none, or of rows of at least one group of 32 or narrower ones, whose
// group is the team
enum { kNoCodes = 0, kWide = 1, kNarrow = 2 };

// A team: `size` neighbouring threads (4 to 32, a power of two, or the whole block).
struct Team {
  int size;
  int block;  // threads of a block
};

// Sums of N values over the team, the same on every thread, in a fixed order. For
// whole-block teams `box` (zero where no warp writes) alternates between two halves, so one
// barrier per call does.
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
    for (int w = 0; w < warps; w += 4) {
      const float4 q = *reinterpret_cast<const float4*>(&b[i][w]);
      s += (q.x + q.y) + (q.z + q.w);
    }
    v[i] = s;
  }
}

template <int N>
__device__ __forceinline__ void clear_box(float (*box)[N][32]) {
  for (int i = threadIdx.x; i < 2 * N * 32; i += blockDim.x) (&box[0][0][0])[i] = 0.f;
}

// One thread's vectors of a row on their way to registers: two rows' slots of W streams. Vector j
// of lane l is at column (j * size + l) * V: vectors of a team side by side, so a group of 32
// columns is held by 32 / V neighbouring lanes.
template <class Raw, int W, int NV>
struct Slots {
  Raw* at;  // [2][W][NV][threads], at this thread's place
  int ld;
  __device__ __forceinline__ Raw* slot(int buf, int w, int j) const { return at + ((buf * W + w) * NV + j) * ld; }
};

template <class T, int V, int NV, int MAXT, int CODES, bool AHEAD>
__global__ void __launch_bounds__(MAXT, MAXT > 256 ? 1 : NV * V <= 8 && !CODES ? 4 : 2)
    norm_fwd_kernel(const NormArgs A, const Team M) {
  constexpr bool kAsync = AHEAD;
  extern __shared__ uint4 smem[];
  __shared__ __align__(16) float box[2][1][32];
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
  const T* src[3] = {static_cast<const T*>(A.x), static_cast<const T*>(A.u), static_cast<const T*>(A.gate)};
  const int64_t ld[3] = {A.x_ld, A.u_ld, A.gate_ld};
  using Raw = typename Pack<T, V>::Raw;
  Slots<Raw, 3, NV> slots{reinterpret_cast<Raw*>(smem) + threadIdx.x, static_cast<int>(blockDim.x)};
  // this thread's vectors inside the row: the first n of them
  const int c0 = lane * V, step = M.size * V;
  const int n_live = c0 < H ? min(NV, (H - c0 + step - 1) / step) : 0;
  clear_box(box);
  if constexpr (kAsync) {  // what no copy writes reads as zero
#pragma unroll
    for (int w = 0; w < 3; ++w)
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (j >= n_live || src[w] == nullptr) *slots.slot(0, w, j) = *slots.slot(1, w, j) = Raw{};
  }
  __syncthreads();
  auto fetch = [&](int64_t row, int buf) {
    if constexpr (kAsync) {
      if (row < A.rows) {
#pragma unroll
        for (int w = 0; w < 3; ++w) {
          if (src[w] == nullptr) continue;
          const T* from = src[w] + row * ld[w] + c0;
#pragma unroll
          for (int j = 0; j < NV; ++j, from += step)
            if (j < n_live) copy_async<sizeof(Raw)>(slots.slot(buf, w, j), from);
        }
      }
      commit_copies();
    }
  };
  // every thread of a block makes the same number of rounds (shuffles and barriers inside)
  const int64_t stride = static_cast<int64_t>(gridDim.x) * teams;
  int buf = 0;
  fetch(static_cast<int64_t>(blockIdx.x) * teams + team, 0);
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * teams; r0 < A.rows; r0 += stride, buf ^= 1) {
    const int64_t row = r0 + team;
    const int n = row < A.rows ? n_live : 0;  // vectors to read and write
    fetch(row + stride, buf ^ 1);
    if constexpr (kAsync) wait_copies<1>();
    float f[3][NV][V];
#pragma unroll
    for (int w = 0; w < 3; ++w) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        Pack<T, V> a;
        if constexpr (kAsync) {
          a.raw = *slots.slot(buf, w, j);  // of an earlier row behind the last: nothing of it is written
        } else {
          const int c = (j * M.size + lane) * V;
          a.zero();
          if (row < A.rows && c < H && src[w] != nullptr) a.load(src[w] + row * ld[w] + c);
        }
        a.get(f[w][j]);
      }
    }
    float(&x)[NV][V] = f[0];
    float(&u)[NV][V] = f[1];
    float(&g)[NV][V] = f[2];
    if constexpr (CODES) {
#pragma unroll
      for (int w = 0; w < 3; ++w) {
        if (src[w] == nullptr) continue;
        int8_t* code = A.codes + (w * A.rows + row) * H + c0;
        float* scale = A.scales + (w * A.rows + row) * G + c0 / kGroup8;
#pragma unroll
        for (int j = 0; j < NV; ++j, code += step, scale += step / kGroup8) {
          Codes<V> q;
          const float s = encode8<CODES == kNarrow>(f[w][j], q, M.size);
          if (j < n) {
            q.store(code);
            if (c0 % kGroup8 == 0) *scale = s;  // a team is whole groups wide
          }
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
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float t = sc[j][v] * (A.gate != nullptr ? sigmoid_f(g[j][v]) : 1.f);
          x[j][v] = fmaf(t, u[j][v] * ru * wp[j][v], x[j][v]);
        }
        if (j < n) {
          Pack<T, V> o;
          o.set(x[j]);
          o.store(static_cast<T*>(A.y) + row * H + c0 + j * step);
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
        if (j < n) {
          float t[V];
#pragma unroll
          for (int v = 0; v < V; ++v) t[v] = x[j][v] * ry * wn[j][v];
          Pack<T, V> o;
          o.set(t);
          o.store(static_cast<T*>(A.n) + row * H + c0 + j * step);
        }
      }
    }
  }
}

template <class T, int V, int NV, int MAXT, bool CODES, bool AHEAD>
__global__ void __launch_bounds__(MAXT, MAXT > 256 || NV * V > 12 ? 1 : 2)
    norm_bwd_kernel(const NormArgs A, const Team M) {
  constexpr bool kAsync = AHEAD;
  using Raw = typename Pack<T, V>::Raw;
  // streams: dy, dn, and without codes x, u, gate; with them three words of codes and three scales
  constexpr int W = CODES ? 2 : 5;
  constexpr int kWords = CODES ? 6 : 0;
  __shared__ __align__(16) float box1[2][1][32];
  __shared__ __align__(16) float box2[2][2][32];
  extern __shared__ uint4 smem[];
  int turn1 = 0, turn2 = 0;
  const int team = threadIdx.x / M.size, lane = threadIdx.x % M.size, teams = M.block / M.size;
  const int H = A.width;
  const int G = (H + kGroup8 - 1) / kGroup8;
  const float over = 1.f / static_cast<float>(H);
  float gp[NV][V], gn[NV][V], gs[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int v = 0; v < V; ++v) gp[j][v] = gn[j][v] = gs[j][v] = 0.f;
  // The three vectors in shared memory, one copy a block: registers go to the row and its sums
  // (8-bit 400,000 x 172: 456 -> 407 us). Lanes of 8 columns would meet in the banks there and
  // keep theirs in registers (16,384 x 2048 bf16: 181 -> 158 us).
  constexpr bool kOwn = V == 8;
  const int span = M.size * NV * V;
  float* const vecs = reinterpret_cast<float*>(smem);
  float own[3][kOwn ? NV : 1][kOwn ? V : 1];
  auto param = [&](int w, int c) {
    const void* p = w == 0 ? A.w_post : w == 1 ? A.w_pre : A.scale;
    const int bf16 = w == 0 ? A.post_bf16 : w == 1 ? A.pre_bf16 : A.scale_bf16;
    return c < H && p != nullptr ? param_at(p, bf16, c) : 1.f;
  };
#pragma unroll
  for (int w = 0; w < 3; ++w) {
    if constexpr (kOwn) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) own[w][j][v] = param(w, (j * M.size + lane) * V + v);
    } else {
      for (int c = threadIdx.x; c < span; c += blockDim.x) vecs[w * span + c] = param(w, c);
    }
  }
  auto vec = [&](int w, int j, float (&f)[V]) {
    if constexpr (kOwn) {
#pragma unroll
      for (int v = 0; v < V; ++v) f[v] = own[w][j][v];
    } else {
      const float* p = vecs + w * span + (j * M.size + lane) * V;
      if constexpr (V == 1) {
        f[0] = *p;
      } else {
        const float4 q = *reinterpret_cast<const float4*>(p);
        f[0] = q.x;
        f[1] = q.y;
        f[2] = q.z;
        f[3] = q.w;
      }
    }
  };
  uint4* const rest = kOwn ? smem : smem + (3 * span + 3) / 4;
  const T* src[5] = {static_cast<const T*>(A.dy), static_cast<const T*>(A.dn), static_cast<const T*>(A.x),
                     static_cast<const T*>(A.u), static_cast<const T*>(A.gate)};
  const int64_t ld[5] = {A.dy_ld, A.dn_ld, A.x_ld, A.u_ld, A.gate_ld};
  Slots<Raw, W, NV> slots{reinterpret_cast<Raw*>(rest) + threadIdx.x, static_cast<int>(blockDim.x)};
  Slots<uint32_t, kWords, NV> words{
      reinterpret_cast<uint32_t*>(reinterpret_cast<Raw*>(rest) + 2 * W * NV * blockDim.x) + threadIdx.x,
      static_cast<int>(blockDim.x)};
  const int c0 = lane * V, step = M.size * V;
  const int n_live = c0 < H ? min(NV, (H - c0 + step - 1) / step) : 0;
  clear_box(box1);
  clear_box(box2);
  if constexpr (kAsync) {  // what no copy writes reads as zero
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int w = 0; w < W; ++w)
        if (j >= n_live || src[w] == nullptr) *slots.slot(0, w, j) = *slots.slot(1, w, j) = Raw{};
#pragma unroll
      for (int w = 0; w < kWords; ++w)
        if (j >= n_live || src[2 + w % 3] == nullptr) *words.slot(0, w, j) = *words.slot(1, w, j) = 0;
    }
  }
  __syncthreads();
  auto fetch = [&](int64_t row, int buf) {
    if constexpr (kAsync) {
      if (row < A.rows) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
          if (src[w] == nullptr) continue;
          const T* from = src[w] + row * ld[w] + c0;
#pragma unroll
          for (int j = 0; j < NV; ++j, from += step)
            if (j < n_live) copy_async<sizeof(Raw)>(slots.slot(buf, w, j), from);
        }
        if constexpr (CODES) {
#pragma unroll
          for (int w = 0; w < 3; ++w) {
            if (src[2 + w] == nullptr) continue;
            const int8_t* code = A.codes + (w * A.rows + row) * H + c0;
            const float* scale = A.scales + (w * A.rows + row) * G + c0 / kGroup8;
#pragma unroll
            for (int j = 0; j < NV; ++j, code += step, scale += step / kGroup8) {
              if (j < n_live) {
                copy_async<4>(words.slot(buf, w, j), code);
                copy_async<4>(words.slot(buf, 3 + w, j), scale);
              }
            }
          }
        }
      }
      commit_copies();
    }
  };
  const int64_t stride = static_cast<int64_t>(gridDim.x) * teams;
  int buf = 0;
  fetch(static_cast<int64_t>(blockIdx.x) * teams + team, 0);
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * teams; r0 < A.rows; r0 += stride, buf ^= 1) {
    const int64_t row = r0 + team;
    const int n = row < A.rows ? n_live : 0;  // vectors to read and write
    fetch(row + stride, buf ^ 1);
    if constexpr (kAsync) wait_copies<1>();
    float f[5][NV][V];
#pragma unroll
    for (int w = 0; w < 5; ++w) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if constexpr (CODES) {
          if (w >= 2) {
            Codes<V> q;
            float s = 0.f;
            if constexpr (kAsync) {
              q.raw = static_cast<typename RawOf<V>::type>(*words.slot(buf, w - 2, j));
              s = __uint_as_float(*words.slot(buf, w + 1, j));
            } else {
              q.zero();
              if (j < n && src[w] != nullptr) {
                q.load(A.codes + ((w - 2) * A.rows + row) * H + c0 + j * step);
                s = A.scales[((w - 2) * A.rows + row) * G + (c0 + j * step) / kGroup8];
              }
            }
            q.get(s, f[w][j]);
            continue;
          }
        }
        Pack<T, V> a;
        if constexpr (kAsync) {
          a.raw = *slots.slot(buf, w < W ? w : 0, j);
        } else {
          const int c = (j * M.size + lane) * V;
          a.zero();
          if (row < A.rows && c < H && src[w] != nullptr) a.load(src[w] + row * ld[w] + c);
        }
        a.get(f[w][j]);
      }
    }
    if (kAsync && row >= A.rows) {  // the slots hold an earlier row or nothing: the sums get zeros
#pragma unroll
      for (int w = 0; w < 5; ++w)
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int v = 0; v < V; ++v) f[w][j][v] = 0.f;
    }
    float(&dy)[NV][V] = f[0];
    float(&dn)[NV][V] = f[1];
    float(&x)[NV][V] = f[2];
    float(&u)[NV][V] = f[3];
    float(&g)[NV][V] = f[4];
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
      for (int j = 0; j < NV; ++j) {
        float wp[V], sc[V];
        vec(0, j, wp);
        vec(2, j, sc);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          g[j][v] = A.gate != nullptr ? sigmoid_f(g[j][v]) : 1.f;
          u[j][v] *= ru;
          x[j][v] = fmaf(sc[v] * g[j][v], u[j][v] * wp[v], x[j][v]);
        }
      }
    }
    if (A.dn != nullptr) {
      float q[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float wn[V];
        vec(1, j, wn);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          q[0] = fmaf(x[j][v], x[j][v], q[0]);
          q[1] = fmaf(dn[j][v] * wn[v], x[j][v], q[1]);
        }
      }
      team_sum(M, q, box2, turn2);
      const float ry = rsqrtf(q[0] * over + A.eps);
      const float m = q[1] * ry * over;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float wn[V];
        vec(1, j, wn);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float yh = x[j][v] * ry;
          gn[j][v] = fmaf(dn[j][v], yh, gn[j][v]);
          dy[j][v] = fmaf(ry, fmaf(-yh, m, dn[j][v] * wn[v]), dy[j][v]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j < n) {
        Pack<T, V> o;
        o.set(dy[j]);
        o.store(static_cast<T*>(A.dx) + row * H + c0 + j * step);
      }
    }
    if (A.u == nullptr) continue;
    float q[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float dg[V], wp[V], sc[V];
      vec(0, j, wp);
      vec(2, j, sc);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float vv = u[j][v] * wp[v];
        const float ds = dy[j][v] * g[j][v];
        gs[j][v] = fmaf(ds, vv, gs[j][v]);
        dg[v] = ds * sc[v] * vv * (1.f - g[j][v]);
        const float dv = ds * sc[v];
        gp[j][v] = fmaf(dv, u[j][v], gp[j][v]);
        dn[j][v] = dv * wp[v];
        q[0] = fmaf(dn[j][v], u[j][v], q[0]);
      }
      if (j < n && A.dgate != nullptr) {
        Pack<T, V> o;
        o.set(dg);
        o.store(static_cast<T*>(A.dgate) + row * H + c0 + j * step);
      }
    }
    float m = 0.f;
    if (A.w_post != nullptr) {
      team_sum(M, q, box1, turn1);
      m = q[0] * over;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j < n) {
        float t[V];
#pragma unroll
        for (int v = 0; v < V; ++v) t[v] = ru * fmaf(-u[j][v], m, dn[j][v]);
        Pack<T, V> o;
        o.set(t);
        o.store(static_cast<T*>(A.du) + row * H + c0 + j * step);
      }
    }
  }
  // the block's share of the three column sums, its teams added up in order
  float* sums = reinterpret_cast<float*>(smem);  // [teams][size * NV * V] of one vector at a time
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

// How a width is laid out over threads. Teams of 4 to 32 lanes (at least a whole 8-bit group
// wide) with up to `most` vectors each where that holds the row, whichever leaves the fewest
// vectors idle; else the whole block, with the fewest vectors a thread that fit.
struct Shape {
  Team team;
  int V, NV;
};
int round_nv(int nv, int V) {  // the counts that are compiled
  if (V > 1) return nv;
  for (int n : {1, 2, 3, 4, 6, 8})
    if (nv <= n) return n;
  return 16;
}
Shape shape_of(const NormArgs& a, int V, int least, int most) {
  Shape s;
  s.V = V;
  const int vecs = (a.width + V - 1) / V;
  const bool few = a.rows < 4096;  // one short round: the fewest vectors a lane
  int best = 1 << 30;
  // with codes a lane's group is a team's, or the team whole groups wide
  const int least_size = a.codes != nullptr ? group_lanes(a.width, V) : 1;
  const int from = vecs > 4 ? 8 : 4;
  for (int size = least_size > from ? least_size : from; size <= 32; size *= 2) {
    const int nv = round_nv((vecs + size - 1) / size, V);
    if (nv <= most && nv * size < best + few) {  // equal: fewer lanes, more loads each
      best = nv * size;
      s.team = {size, 256};
      s.NV = nv;
    }
  }
  if (best < 1 << 30) return s;
  for (int nv = least; nv <= 16; nv = V > 1 ? nv + 1 : nv * 2) {
    const int size = ((vecs + nv - 1) / nv + 31) / 32 * 32;
    if (size <= (nv < most ? 256 : 1024)) {
      s.team = {size, size};
      s.NV = nv;
      return s;
    }
  }
  return s;
}
// 16 bytes a vector; 8-bit codes go by words of four. Backward keeps 11 values of a column in
// registers (5 inputs, 3 parameters, 3 sums), forward 6.
int vec_of(const NormArgs& a) { return a.vec ? (a.bf16 && a.vec8 && a.codes == nullptr ? 8 : 4) : 1; }
Shape fwd_shape(const NormArgs& a) {
  const int V = vec_of(a);
  return shape_of(a, V, 2, V == 8 ? 2 : V == 4 ? 4 : 8);
}
Shape bwd_shape(const NormArgs& a) {
  const int V = vec_of(a);
  return shape_of(a, V, V == 1 ? 2 : 1, V == 8 ? 2 : V == 4 ? 3 : 8);
}
int64_t round_count(const NormArgs& a, const Shape& s) {
  const int teams = s.team.block / s.team.size;
  return (a.rows + teams - 1) / teams;
}

constexpr int kMostBlocks = 8;  // per SM
// Blocks that an SM takes, asked once per kernel and team: block size and shared memory go by the
// team (8-bit backward pass, fp32: 88 KB and two blocks with teams of 16 in blocks of 256, 123 KB and
// one block with a team of 256), and so must the grid, whose blocks are the vectors' partial sums.
struct Fits {
  int of[39] = {};  // teams of 4 to 32 lanes in larger blocks, then teams of 32 k that are blocks
  int& at(const Team& t) {
    if (t.size == t.block) return of[6 + t.size / 32];
    int k = 0;
    while (1 << k < t.size) ++k;
    return of[k];
  }
};
template <class K>
void run(K kernel, Fits& fits, uint64_t& allowed, const NormArgs& a, const Shape& s, size_t smem, int sms, cudaStream_t st,
         int* grid) {
  allow_smem(kernel, smem, allowed);
  int& per_sm = fits.at(s.team);
  if (per_sm == 0) {
    int n = 1;
    cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, s.team.block, smem);
    per_sm = n < 1 ? 1 : (n > kMostBlocks ? kMostBlocks : n);
  }
  const int64_t want = round_count(a, s), most = static_cast<int64_t>(sms) * per_sm;
  const int blocks = static_cast<int>(want < most ? want : most);
  if (grid != nullptr) *grid = blocks;
  kernel<<<blocks, s.team.block, smem, st>>>(a, s.team);
}

// The next row is fetched ahead where a block or a few warps with codes to decode would wait for
// it; teams inside a warp have enough other rows under way (1,600,000 rows of 64 fp32,
// backward: 495 us without, 588 us with it). Copies have 4 bytes at least, and two rows of
// blocks above 256 threads do not fit.
template <class T, int V, int NV, int MAXT, bool CODES, bool BWD, bool AHEAD>
void run_case(const NormArgs& a, const Shape& s, int sms, cudaStream_t st, int* grid) {
  static Fits fits;
  static uint64_t allowed = 0;
  const size_t threads = s.team.block;
  if constexpr (BWD) {
    const size_t vecs = V == 8 ? 0 : (3 * s.team.size * NV * V + 3) / 4 * 16;
    size_t smem = vecs + (AHEAD ? threads * 2 * NV * (CODES ? 2 * sizeof(T) * V + 24 : 5 * sizeof(T) * V) : 0);
    const size_t sums = threads * NV * V * sizeof(float);
    smem = smem > sums ? smem : sums;
    run(norm_bwd_kernel<T, V, NV, MAXT, CODES, AHEAD>, fits, allowed, a, s, smem, sms, st, grid);
  } else {
    const size_t smem = AHEAD ? threads * 2 * NV * 3 * sizeof(T) * V : 0;
    constexpr int kCodes = !CODES ? kNoCodes : kWide;
    if constexpr (CODES && NV == 1) {
      if (a.width < kGroup8) {
        static Fits narrow_fits;
        return run(norm_fwd_kernel<T, V, NV, MAXT, kNarrow, AHEAD>, narrow_fits, allowed, a, s, smem, sms, st, grid);
      }
    }
    run(norm_fwd_kernel<T, V, NV, MAXT, kCodes, AHEAD>, fits, allowed, a, s, smem, sms, st, grid);
  }
}
template <class T, int V, int NV, int MAXT, bool CODES, bool BWD>
void run_case(const NormArgs& a, const Shape& s, int sms, cudaStream_t st, int* grid) {
  if constexpr (MAXT == 256 && (CODES && BWD ? V == 4 : sizeof(T) * V >= 4)) {
    if (s.team.size > 32 || CODES) return run_case<T, V, NV, MAXT, CODES, BWD, true>(a, s, sms, st, grid);
  }
  run_case<T, V, NV, MAXT, CODES, BWD, false>(a, s, sms, st, grid);
}

template <class T, bool CODES, bool BWD>
void run_norm(const NormArgs& a, int sms, cudaStream_t st, int* grid) {
  const Shape s = BWD ? bwd_shape(a) : fwd_shape(a);
  const bool small = s.team.block <= 256;
#define SU_NORM_CASE(V_, NV_, MAXT_) \
  if (s.V == V_ && s.NV == NV_ && small == (MAXT_ == 256)) return run_case<T, V_, NV_, MAXT_, CODES, BWD>(a, s, sms, st, grid);
  if constexpr (sizeof(T) == 2 && !CODES) {
    SU_NORM_CASE(8, 1, 256)
    SU_NORM_CASE(8, 2, 256)
    SU_NORM_CASE(8, 2, 1024)
  }
  SU_NORM_CASE(4, 1, 256)
  SU_NORM_CASE(4, 2, 256)
  SU_NORM_CASE(4, 3, 256)
  if constexpr (!BWD) {
    SU_NORM_CASE(4, 4, 256)
  }
  if constexpr (BWD) {
    SU_NORM_CASE(4, 3, 1024)
  }
  SU_NORM_CASE(4, 4, 1024)
  SU_NORM_CASE(1, 1, 256)
  SU_NORM_CASE(1, 2, 256)
  SU_NORM_CASE(1, 3, 256)
  SU_NORM_CASE(1, 4, 256)
  SU_NORM_CASE(1, 6, 256)
  SU_NORM_CASE(1, 8, 256)
  SU_NORM_CASE(1, 8, 1024)
  SU_NORM_CASE(1, 16, 1024)
#undef SU_NORM_CASE
}

}  // namespace

int norm_partials(const NormArgs& a, int sms) {
  const int64_t want = round_count(a, bwd_shape(a)), most = static_cast<int64_t>(sms) * kMostBlocks;
  return static_cast<int>(want < most ? want : most);
}

void launch_norm_fwd(const NormArgs& a, int sms, cudaStream_t st) {
  count_launch();
  const bool codes = a.codes != nullptr;
  if (a.bf16)
    codes ? run_norm<__nv_bfloat16, true, false>(a, sms, st, nullptr)
          : run_norm<__nv_bfloat16, false, false>(a, sms, st, nullptr);
  else
    codes ? run_norm<float, true, false>(a, sms, st, nullptr) : run_norm<float, false, false>(a, sms, st, nullptr);
}

void launch_norm_bwd(const NormArgs& in, int sms, cudaStream_t st) {
  NormArgs a = in;
  const bool codes = a.codes != nullptr;
  count_launch();
  int* n = &a.n_partial;  // the blocks that ran
  if (a.bf16)
    codes ? run_norm<__nv_bfloat16, true, true>(in, sms, st, n) : run_norm<__nv_bfloat16, false, true>(in, sms, st, n);
  else
    codes ? run_norm<float, true, true>(in, sms, st, n) : run_norm<float, false, true>(in, sms, st, n);
  if (a.dw_post == nullptr && a.dw_pre == nullptr && a.dscale == nullptr) return;
  count_launch();
  norm_param_grad_kernel<<<dim3((a.width + 31) / 32, 3), dim3(32, 32), 0, st>>>(a);
}

}  // namespace su
