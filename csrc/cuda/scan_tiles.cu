// The gated linear recurrence split over its steps: for few or unequal sequences, whose
// channels alone do not fill the GPU. One pass over the data.
//
// A tile is kRun steps for each of `rows` neighbouring threads times 32 or fewer
// lanes of channels; it is loaded once and stays in registers. A run of steps maps the
// state before it to A h + B, and two runs compose to (A2 A1, A2 B1 + B2). A tile
// composes its threads' runs in shared memory, publishes (A, B), obtains the state before
// itself from the tiles before it and then writes its steps.
//
// The state before tile j comes from three levels, so that the serial chain is one hop per
// 256 tiles instead of one per tile: the tiles of its group of 16 so far, the groups of its
// block of 16 groups so far, and the state that the block before left. The last tile of a
// group publishes the group, the last tile of a block the state after it. What is
// composed, and in which order, depends on j alone, so results are the same every run.
// Tiles are handed out by a counter, earlier steps first: a tile waits only for tiles
// that run or are done. Every wait is bounded (kScanTimeout is recorded, the carry then
// counts as 0 and the tile goes on).
//
// Packed sequences are one long run with restarts: at a first step the state before it is
// that sequence's h0, so unequal lengths cost nothing. Backwards the same scheme runs from
// the last step to the first on E = a (dh + E), the gradient that reaches h_{t-1}.
#include "kernels.h"
#include "scan_math.cuh"

namespace su {
namespace {

constexpr int kRun = 8;                        // steps per thread; divides kStateEvery by 2
constexpr int kFan = 16;                       // tiles per group, groups per block
constexpr long long kCarryBudget = 400000000;  // cycles, ~0.2 s

struct TileShape {
  Lanes l;
  int64_t tiles;   // along the steps
  int64_t chains;  // batch * channel blocks
};

struct TileWork {
  unsigned long long* ticket;
  int* tile_flag;   // [chains, tiles]
  int* group_flag;  // [chains, groups]
  int* block_flag;  // [chains, blocks]
  float2* tile_map;   // [chains, tiles, lanes * V]
  float2* group_map;  // [chains, groups, lanes * V]
  float* block_state;  // [chains, blocks, lanes * V]
};

__device__ __forceinline__ void flag_set(int* f) {
  __threadfence();
  asm volatile("st.release.gpu.global.s32 [%0], 1;" ::"l"(f) : "memory");
}
__device__ __forceinline__ int flag_get(const int* f) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(f) : "memory");
  return v;
}
// One warp waits until f[0 .. n) are set (n <= 32). False when the budget ran out.
__device__ __forceinline__ bool flags_wait(const int* f, int n) {
  const int lane = threadIdx.x & 31;
  bool ok = lane >= n || flag_get(f + lane) != 0;
  if (!__all_sync(0xffffffffu, ok)) {
    const long long t0 = clock64();
    do {
      if (!ok) ok = flag_get(f + lane) != 0;
      if (__all_sync(0xffffffffu, ok)) break;
    } while (clock64() - t0 < kCarryBudget);
  }
  return __all_sync(0xffffffffu, ok) != 0;
}

// First warp: publishes tile j's map (A, B) and returns the state before it in c, which comes
// in as the state before the chain's first tile. Lanes without channels (`live` false) only wait.
template <int V>
__device__ __forceinline__ void carry_in(const TileShape& S, const TileWork& W, int64_t chain, int64_t j, int x,
                                         bool live, const float (&A)[V], const float (&B)[V], float (&c)[V],
                                         int* status) {
  const int lane = threadIdx.x & 31;
  const int width = S.l.count * V;
  const int64_t groups = (S.tiles + kFan - 1) / kFan, blocks = (groups + kFan - 1) / kFan;
  const int64_t g = j / kFan, b = g / kFan;
  const int m = static_cast<int>(j % kFan), mg = static_cast<int>(g % kFan);
  const bool more = j + 1 < S.tiles;
  bool ok = true;
  float2* tm = W.tile_map + (chain * S.tiles + g * kFan) * width + x * V;
  float2* gm = W.group_map + (chain * groups + b * kFan) * width + x * V;
  float* bs = W.block_state + (chain * blocks + b) * width + x * V;
  if (more && m != kFan - 1) {
    if (live) {
#pragma unroll
      for (int v = 0; v < V; ++v) __stcg(tm + static_cast<int64_t>(m) * width + v, make_float2(A[v], B[v]));
    }
    __syncwarp();
    if (lane == 0) flag_set(W.tile_flag + chain * S.tiles + j);
  }
  float ga[V], gb[V];  // the group's tiles before this one
#pragma unroll
  for (int v = 0; v < V; ++v) {
    ga[v] = 1.f;
    gb[v] = 0.f;
  }
  if (m > 0) {
    ok &= flags_wait(W.tile_flag + chain * S.tiles + g * kFan, m);
    if (live) {
#pragma unroll 5
      for (int k = 0; k < m; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float2 t = __ldcg(tm + static_cast<int64_t>(k) * width + v);
          ga[v] *= t.x;
          gb[v] = fmaf(t.x, gb[v], t.y);
        }
    }
  }
  if (more && m == kFan - 1 && mg != kFan - 1) {
    if (live) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        __stcg(gm + static_cast<int64_t>(mg) * width + v, make_float2(A[v] * ga[v], fmaf(A[v], gb[v], B[v])));
    }
    __syncwarp();
    if (lane == 0) flag_set(W.group_flag + chain * groups + g);
  }
  if (b > 0) {
    ok &= flags_wait(W.block_flag + chain * blocks + b, 1);
    if (live) {
#pragma unroll
      for (int v = 0; v < V; ++v) c[v] = __ldcg(bs + v);
    }
  }
  if (mg > 0) {
    ok &= flags_wait(W.group_flag + chain * groups + b * kFan, mg);
    if (live) {
#pragma unroll 5
      for (int k = 0; k < mg; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float2 t = __ldcg(gm + static_cast<int64_t>(k) * width + v);
          c[v] = fmaf(t.x, c[v], t.y);
        }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) c[v] = ok ? fmaf(ga[v], c[v], gb[v]) : 0.f;
  if (more && m == kFan - 1 && mg == kFan - 1) {
    if (live) {
#pragma unroll
      for (int v = 0; v < V; ++v) __stcg(bs + width + v, fmaf(A[v], c[v], B[v]));
    }
    __syncwarp();
    if (lane == 0) flag_set(W.block_flag + chain * blocks + b + 1);
  }
  if (!ok && lane == 0) record_status(status, kScanTimeout);
}

// First and last steps of the packed sequences inside [t0, t0 + n): first[t - t0] and
// last[t - t0] are the sequence, or -1. The whole block calls; empty sequences have neither.
__device__ __forceinline__ void mark_sequences(const ScanArgs& A, int64_t t0, int n, int* first, int* last) {
  for (int k = threadIdx.x; k < n; k += blockDim.x) first[k] = last[k] = -1;
  // a 32-way search of the first sequence that begins at t0 or later, every warp by itself
  const int lane = threadIdx.x & 31;
  int64_t lo = 0, hi = A.batch;  // offsets[lo - 1] < t0 <= offsets[hi], with offsets[batch] = steps >= t0
  const bool whole = blockDim.x >= 32 && threadIdx.x / 32 < blockDim.x / 32;  // a full warp
  if (whole) {
    while (hi - lo > 0) {
      const int64_t step = (hi - lo + 31) / 32;
      const int64_t at = lo + lane * step;
      const bool below = at < hi && A.offsets[at] < t0;
      const int cnt = __popc(__ballot_sync(0xffffffffu, below));
      const int64_t nlo = cnt == 0 ? lo : lo + static_cast<int64_t>(cnt - 1) * step + 1;
      const int64_t nhi = cnt == 32 ? hi : min(hi, lo + static_cast<int64_t>(cnt) * step);
      lo = nlo;
      hi = nhi;
    }
  } else {
    while (hi - lo > 0) {
      const int64_t mid = lo + (hi - lo) / 2;
      if (A.offsets[mid] < t0)
        lo = mid + 1;
      else
        hi = mid;
    }
  }
  __syncthreads();
  // the sequence before may end here
  for (int64_t s = (lo > 0 ? lo - 1 : 0) + threadIdx.x; s < A.batch; s += blockDim.x) {
    const int64_t a = A.offsets[s], b = A.offsets[s + 1];
    if (a < 0 || b < a || b > A.steps) {
      record_status(A.status, kBadIndex);
      continue;
    }
    if (a >= t0 + n) break;
    if (b == a) continue;
    if (a >= t0) first[a - t0] = static_cast<int>(s);
    if (b - 1 >= t0 && b - 1 < t0 + n) last[b - 1 - t0] = static_cast<int>(s);
  }
  // rows outside every sequence are a caller's mistake
  if (threadIdx.x == 0 && t0 == 0 && (A.offsets[0] != 0 || A.offsets[A.batch] != A.steps))
    record_status(A.status, kBadIndex);
  __syncthreads();
}

struct Place {
  int64_t j, chain, b;  // tile along the walk, chain, batch index
  int x, y, c;
  bool live;
};
template <int V>
__device__ __forceinline__ Place place_of(const TileShape& S, const TileWork& W, int width) {
  __shared__ unsigned long long ticket;
  if (threadIdx.x == 0) ticket = atomicAdd(W.ticket, 1ull);
  __syncthreads();
  Place p;
  p.j = static_cast<int64_t>(ticket / static_cast<unsigned long long>(S.chains));
  p.chain = static_cast<int64_t>(ticket % static_cast<unsigned long long>(S.chains));
  p.b = p.chain / S.l.blocks;
  p.x = threadIdx.x % S.l.count;
  p.y = threadIdx.x / S.l.count;
  p.c = (static_cast<int>(p.chain % S.l.blocks) * S.l.count + p.x) * V;
  p.live = p.c < width;
  return p;
}

// The state before each thread's run: composes the runs of a tile (maps in shared memory),
// asks for the state before the tile and walks it through the runs. [rows][lanes * V] each.
template <int V>
__device__ __forceinline__ void tile_carry(const TileShape& S, const TileWork& W, const Place& p, const float (&A)[V],
                                           const float (&B)[V], const float (&init)[V], float2* maps, float (&h)[V],
                                           int* status) {
  const int width = S.l.count * V;
#pragma unroll
  for (int v = 0; v < V; ++v) maps[p.y * width + p.x * V + v] = make_float2(A[v], B[v]);
  __syncthreads();
  if (threadIdx.x < 32) {
    const bool live = p.y == 0 && p.live;
    float ta[V], tb[V], c[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      ta[v] = 1.f;
      tb[v] = 0.f;
      c[v] = init[v];
    }
    if (live) {
      for (int k = 0; k < S.l.rows; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float2 t = maps[k * width + p.x * V + v];
          ta[v] *= t.x;
          tb[v] = fmaf(t.x, tb[v], t.y);
        }
    }
    carry_in<V>(S, W, p.chain, p.j, p.x, live, ta, tb, c, status);
    if (live) {
      for (int k = 0; k < S.l.rows; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float2& t = maps[k * width + p.x * V + v];
          const float in = c[v];
          c[v] = fmaf(t.x, c[v], t.y);
          t.x = in;
        }
    }
  }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = maps[p.y * width + p.x * V + v].x;
}

template <class T, int V, bool CODES, bool PACKED, bool MASK>
__global__ void __launch_bounds__(256, V == 1 ? 4 : 3)
    scan_tiles_fwd_kernel(const ScanArgs A, const TileShape S, const TileWork W) {
  constexpr int K = kRun;
  extern __shared__ float2 smem[];
  float2* maps = smem;
  int* first = reinterpret_cast<int*>(maps + S.l.rows * S.l.count * V);
  int* last = first + S.l.rows * K;
  const int H = A.width;
  const int G = (H + kGroup8 - 1) / kGroup8;
  const Place p = place_of<V>(S, W, H);
  const int64_t tile0 = p.j * S.l.rows * K;
  const int64_t t0 = tile0 + p.y * K;
  const int n = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(K), A.steps - t0)));
  Pack<T, V> x[K], r[K], i[K];
  unsigned on = 0;
  {
    const T* in = static_cast<const T*>(A.p) + p.b * A.p_sb + t0 * A.p_st + p.c;
    const uint8_t* valid = MASK ? A.mask + p.b * A.m_sb + t0 * A.m_st : nullptr;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      x[k].zero();
      r[k].zero();
      i[k].zero();
      if (k < n && p.live && (!MASK || *valid != 0)) {
        on |= 1u << k;
        x[k].load(in);
        r[k].load(in + H);
        i[k].load(in + 2 * H);
      }
      in += A.p_st;
      if (MASK) valid += A.m_st;
    }
  }
  if (PACKED) mark_sequences(A, tile0, S.l.rows * K, first, last);
  float kd[V], init[V], a[K][V], add[K][V], ra[V], rb[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    kd[v] = p.live ? decay_factor(param_at(A.decay, A.decay_bf16, p.c + v), A.rate) : 0.f;
    init[v] = (!PACKED && p.live && A.h0 != nullptr) ? A.h0[p.b * H + p.c + v] : 0.f;
    ra[v] = 1.f;
    rb[v] = 0.f;
  }
  const int64_t row0 = p.b * A.row_sb + t0 * A.row_st;
  int8_t* code = CODES ? A.codes + row0 * 3 * H + p.c : nullptr;
  float* scale = CODES ? A.scales + row0 * 3 * G + p.c / kGroup8 : nullptr;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float fx[V], fr[V], fi[V];
    x[k].get(fx);
    r[k].get(fr);
    i[k].get(fi);
    if constexpr (CODES) {
      if (k < n) {  // the same for all lanes of a group
        Codes<V> q0, q1, q2;
        const float s0 = encode8(fx, q0), s1 = encode8(fr, q1), s2 = encode8(fi, q2);
        if (p.live) {
          q0.store(code);
          q1.store(code + H);
          q2.store(code + 2 * H);
          if (p.c % kGroup8 == 0) {
            scale[0] = s0;
            scale[G] = s1;
            scale[2 * G] = s2;
          }
        }
      }
      code += A.row_st * 3 * H;
      scale += A.row_st * 3 * G;
    }
    const int from = PACKED ? first[p.y * K + k] : -1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      a[k][v] = 1.f;
      add[k][v] = 0.f;
      if (on >> k & 1) {
        const Step g = step_of(fx[v], fr[v], fi[v], kd[v]);
        a[k][v] = g.a;
        add[k][v] = g.add;
      }
      if (PACKED && from >= 0) {
        ra[v] = 0.f;
        rb[v] = (p.live && A.h0 != nullptr) ? A.h0[static_cast<int64_t>(from) * H + p.c + v] : 0.f;
      }
      ra[v] *= a[k][v];
      rb[v] = fmaf(a[k][v], rb[v], add[k][v]);
    }
  }
  float h[V];
  tile_carry<V>(S, W, p, ra, rb, init, maps, h, A.status);
  if (!p.live) return;
  if (A.states != nullptr && t0 > 0 && t0 % kStateEvery == 0 && n > 0) {
    float* to = A.states + (p.b * A.n_states + t0 / kStateEvery - 1) * H + p.c;
#pragma unroll
    for (int v = 0; v < V; ++v) to[v] = h[v];
  }
  T* out = static_cast<T*>(A.h) + row0 * H + p.c;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (k < n) {
      const int from = PACKED ? first[p.y * K + k] : -1;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (PACKED && from >= 0) h[v] = A.h0 != nullptr ? A.h0[static_cast<int64_t>(from) * H + p.c + v] : 0.f;
        h[v] = fmaf(a[k][v], h[v], add[k][v]);
      }
      Pack<T, V> o;
      o.set(h);
      o.store(out);
      const int64_t done = PACKED ? last[p.y * K + k] : (t0 + k == A.steps - 1 ? p.b : -1);
      if (done >= 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) A.last[done * H + p.c + v] = h[v];
      }
    }
    out += A.row_st * H;
  }
}

// Walks from the last step to the first: run y of tile j covers the steps that end
// (j * rows + y) * K before the end of the last tile. One channel per thread: the factors of
// its steps' gradients, evaluated once, stay in registers.
template <class T, bool CODES, bool PACKED, bool MASK>
__global__ void __launch_bounds__(256, 2) scan_tiles_bwd_kernel(const ScanArgs A, const TileShape S, const TileWork W) {
  constexpr int K = kRun;
  extern __shared__ float2 smem[];
  float2* maps = smem;
  int* first = reinterpret_cast<int*>(maps + S.l.rows * S.l.count);
  int* last = first + S.l.rows * K;
  const int H = A.width;
  const int G = (H + kGroup8 - 1) / kGroup8;
  const Place p = place_of<1>(S, W, H);
  const int64_t tile = S.tiles - 1 - p.j;
  const int64_t tile0 = tile * S.l.rows * K;
  const int at0 = (S.l.rows - 1 - p.y) * K;  // inside the tile
  const int64_t t0 = tile0 + at0;
  const int n = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(K), A.steps - t0)));
  const int64_t row0 = p.b * A.row_sb + t0 * A.row_st;
  float x[K], r[K], i[K], d[K];
  unsigned on = 0;
  {
    const T* in = CODES ? nullptr : static_cast<const T*>(A.p) + p.b * A.p_sb + t0 * A.p_st + p.c;
    const int8_t* code = CODES ? A.codes + row0 * 3 * H + p.c : nullptr;
    const float* scale = CODES ? A.scales + row0 * 3 * G + p.c / kGroup8 : nullptr;
    const T* dh = static_cast<const T*>(A.dh) + (A.dh != nullptr ? p.b * A.dh_sb + t0 * A.dh_st + p.c : 0);
    const uint8_t* valid = MASK ? A.mask + p.b * A.m_sb + t0 * A.m_st : nullptr;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      x[k] = r[k] = i[k] = d[k] = 0.f;
      if (k < n && p.live) {
        if (!MASK || *valid != 0) {
          on |= 1u << k;
          if constexpr (CODES) {
            Codes<1> q[3];
            q[0].load(code);
            q[1].load(code + H);
            q[2].load(code + 2 * H);
            float f[3][1];
            q[0].get(scale[0], f[0]);
            q[1].get(scale[G], f[1]);
            q[2].get(scale[2 * G], f[2]);
            x[k] = f[0][0];
            r[k] = f[1][0];
            i[k] = f[2][0];
          } else {
            x[k] = to_f32(__ldcs(in));
            r[k] = to_f32(__ldcs(in + H));
            i[k] = to_f32(__ldcs(in + 2 * H));
          }
        }
        if (A.dh != nullptr) d[k] = to_f32(__ldcs(dh));
      }
      if (CODES) {
        code += A.row_st * 3 * H;
        scale += A.row_st * 3 * G;
      } else {
        in += A.p_st;
      }
      dh += A.dh_st;
      if (MASK) valid += A.m_st;
    }
  }
  // the state before the run: kept at every second run, handed on by the run before at the others
  const bool kept = t0 % kStateEvery == 0;
  float h = 0.f;
  if (p.live && n > 0 && kept) {
    if (t0 > 0)
      h = A.states[(p.b * A.n_states + t0 / kStateEvery - 1) * H + p.c];
    else if (!PACKED && A.h0 != nullptr)
      h = A.h0[p.b * H + p.c];
  }
  if (PACKED) mark_sequences(A, tile0, S.l.rows * K, first, last);
  const float kd = p.live ? decay_factor(param_at(A.decay, A.decay_bf16, p.c), A.rate) : 0.f;
  Gate g[K];
#pragma unroll
  for (int k = 0; k < K; ++k) g[k] = on >> k & 1 ? gate_of(x[k], r[k], i[k], kd) : gate_shut();
  Slope f[K];
  auto walk = [&]() {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int from = PACKED ? first[at0 + k] : -1;
      if (PACKED && from >= 0) h = (p.live && A.h0 != nullptr) ? A.h0[static_cast<int64_t>(from) * H + p.c] : 0.f;
      f[k] = slope_of(g[k], h);
    }
  };
  float* handed = &maps[p.y * S.l.count + p.x].x;
  if (kept) {
    walk();
    if (p.y > 0) handed[-2 * S.l.count] = h;  // the place of the run that follows in time
  }
  __syncthreads();
  if (!kept) {
    h = *handed;
    walk();
  }
  float ra[1] = {1.f}, rb[1] = {0.f}, E[1];
  const float init[1] = {(!PACKED && p.live && A.dlast != nullptr) ? A.dlast[p.b * H + p.c] : 0.f};
#pragma unroll
  for (int k = K - 1; k >= 0; --k) {
    const int to = PACKED ? last[at0 + k] : -1;
    if (PACKED && to >= 0) {
      ra[0] = 0.f;
      rb[0] = (p.live && A.dlast != nullptr) ? A.dlast[static_cast<int64_t>(to) * H + p.c] : 0.f;
    }
    ra[0] *= f[k].a;  // steps beyond the last: a = 1, d = 0
    rb[0] = f[k].a * (rb[0] + d[k]);
  }
  tile_carry<1>(S, W, p, ra, rb, init, maps, E, A.status);
  float dl = 0.f;
  if (p.live) {
    T* out = static_cast<T*>(A.dp) + (row0 + K * A.row_st) * 3 * H + p.c;
#pragma unroll
    for (int k = K - 1; k >= 0; --k) {
      out -= A.row_st * 3 * H;
      if (k >= n) continue;
      const int to = PACKED ? last[at0 + k] : -1;
      if (PACKED && to >= 0) E[0] = A.dlast != nullptr ? A.dlast[static_cast<int64_t>(to) * H + p.c] : 0.f;
      const float e = d[k] + E[0];
      __stcs(out, from_f32<T>(e * f[k].x));
      __stcs(out + H, from_f32<T>(e * f[k].r));
      __stcs(out + 2 * H, from_f32<T>(e * f[k].i));
      dl = fmaf(e, f[k].l, dl);
      E[0] = e * f[k].a;
      const int64_t begin = PACKED ? first[at0 + k] : (t0 + k == 0 ? p.b : -1);
      if (begin >= 0 && A.dh0 != nullptr) A.dh0[begin * H + p.c] = E[0];
    }
  }
  // the tile's share of sum dz sigmoid(r), its runs added up in order
  float* sum = reinterpret_cast<float*>(maps);
  __syncthreads();
  sum[p.y * S.l.count + p.x] = dl;
  __syncthreads();
  if (p.y == 0 && p.live) {
    float t = 0.f;
    for (int k = 0; k < S.l.rows; ++k) t += sum[k * S.l.count + p.x];
    A.partial[(p.b * S.tiles + tile) * H + p.c] = t;
  }
}

// channels per thread: forward 4 bytes of them, backward one, whose 7 factors of 8 steps
// have to fit its registers
int vec_of(const ScanArgs& a, bool bwd) { return !bwd && a.bf16 && a.vec ? 2 : 1; }

TileShape shape_of(const ScanArgs& a, bool bwd) {
  TileShape s;
  s.l = lanes_of(a.width, vec_of(a, bwd), a.codes != nullptr && !bwd, 32, 256);
  if (s.l.rows > 32) s.l.rows = 32;
  s.l.rows &= ~1;  // whole pairs of runs: a kept state for each
  const int64_t steps = static_cast<int64_t>(s.l.rows) * kRun;
  s.tiles = (a.steps + steps - 1) / steps;
  s.chains = (a.offsets != nullptr ? 1 : a.batch) * s.l.blocks;
  return s;
}

// workspace: ticket and flags (zeroed), then the maps
struct WorkLayout {
  int64_t groups, blocks, width, head, bytes;
};
WorkLayout layout_of(const ScanArgs& a, const TileShape& s, bool bwd) {
  WorkLayout w;
  w.groups = (s.tiles + kFan - 1) / kFan;
  w.blocks = (w.groups + kFan - 1) / kFan;
  w.width = s.l.count * vec_of(a, bwd);
  w.head = (8 + 4 * s.chains * (s.tiles + w.groups + w.blocks) + 15) / 16 * 16;
  w.bytes = w.head + s.chains * w.width * ((s.tiles + w.groups) * 8 + w.blocks * 4);
  return w;
}

TileWork work_of(const TileShape& s, const WorkLayout& l, void* buf) {
  TileWork w;
  w.ticket = static_cast<unsigned long long*>(buf);
  w.tile_flag = reinterpret_cast<int*>(w.ticket + 1);
  w.group_flag = w.tile_flag + s.chains * s.tiles;
  w.block_flag = w.group_flag + s.chains * l.groups;
  w.tile_map = reinterpret_cast<float2*>(static_cast<char*>(buf) + l.head);
  w.group_map = w.tile_map + s.chains * s.tiles * l.width;
  w.block_state = reinterpret_cast<float*>(w.group_map + s.chains * l.groups * l.width);
  return w;
}

template <class T, bool CODES, bool PACKED, bool MASK>
void run_tiles(const ScanArgs& a, const TileShape& s, const TileWork& w, bool bwd, cudaStream_t st) {
  const unsigned blocks = static_cast<unsigned>(s.tiles * s.chains);
  const int threads = s.l.rows * s.l.count;
  const size_t smem = static_cast<size_t>(threads) * vec_of(a, bwd) * sizeof(float2) +
                      (PACKED ? static_cast<size_t>(s.l.rows) * kRun * 2 * sizeof(int) : 0);
  if (bwd) {
    scan_tiles_bwd_kernel<T, CODES, PACKED, MASK><<<blocks, threads, smem, st>>>(a, s, w);
    return;
  }
  if constexpr (sizeof(T) == 2) {
    if (vec_of(a, bwd) == 2) {
      scan_tiles_fwd_kernel<T, 2, CODES, PACKED, MASK><<<blocks, threads, smem, st>>>(a, s, w);
      return;
    }
  }
  scan_tiles_fwd_kernel<T, 1, CODES, PACKED, MASK><<<blocks, threads, smem, st>>>(a, s, w);
}

template <class T, bool CODES>
void run_tiles(const ScanArgs& a, const TileShape& s, const TileWork& w, bool bwd, cudaStream_t st) {
  const bool mask = a.mask != nullptr;
  if (a.offsets != nullptr)
    mask ? run_tiles<T, CODES, true, true>(a, s, w, bwd, st) : run_tiles<T, CODES, true, false>(a, s, w, bwd, st);
  else
    mask ? run_tiles<T, CODES, false, true>(a, s, w, bwd, st) : run_tiles<T, CODES, false, false>(a, s, w, bwd, st);
}

}  // namespace

int64_t scan_tiles_partials(const ScanArgs& a) {
  return (a.offsets != nullptr ? 1 : a.batch) * shape_of(a, true).tiles;
}

size_t scan_tiles_workspace(const ScanArgs& a, bool bwd) {
  return static_cast<size_t>(layout_of(a, shape_of(a, bwd), bwd).bytes);
}

void launch_scan_tiles(const ScanArgs& a, bool bwd, void* workspace, cudaStream_t st) {
  const TileShape s = shape_of(a, bwd);
  if (a.offsets != nullptr) {
    // what an empty sequence returns: its first state, or the gradient of its last
    float* to = bwd ? a.dh0 : a.last;
    const float* from = bwd ? a.dlast : a.h0;
    const size_t bytes = static_cast<size_t>(a.batch) * a.width * sizeof(float);
    if (to != nullptr) {
      if (from != nullptr)
        cudaMemcpyAsync(to, from, bytes, cudaMemcpyDeviceToDevice, st);
      else
        cudaMemsetAsync(to, 0, bytes, st);
    }
  }
  if (s.tiles == 0) return;
  const WorkLayout l = layout_of(a, s, bwd);
  cudaMemsetAsync(workspace, 0, l.head, st);
  const TileWork w = work_of(s, l, workspace);
  count_launch();
  const bool codes = a.codes != nullptr;
  if (a.bf16)
    codes ? run_tiles<__nv_bfloat16, true>(a, s, w, bwd, st) : run_tiles<__nv_bfloat16, false>(a, s, w, bwd, st);
  else
    codes ? run_tiles<float, true>(a, s, w, bwd, st) : run_tiles<float, false>(a, s, w, bwd, st);
}

}  // namespace su
