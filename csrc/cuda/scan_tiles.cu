// The gated linear recurrence split over its steps: for few or unequal sequences, whose
// channels alone do not fill the GPU. One pass over the data.
//
// A tile is kStateEvery steps for each of `rows` neighbouring threads times 32 or fewer
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

template <class T, int V, bool CODES>
__global__ void __launch_bounds__(256, 2) scan_tiles_fwd_kernel(const ScanArgs A, const TileShape S, const TileWork W) {
  constexpr int K = kStateEvery;
  extern __shared__ float2 smem[];
  float2* maps = smem;
  int* first = reinterpret_cast<int*>(maps + S.l.rows * S.l.count * V);
  int* last = first + S.l.rows * K;
  const int H = A.width;
  const int G = (H + kGroup8 - 1) / kGroup8;
  const Place p = place_of<V>(S, W, H);
  const int64_t tile0 = p.j * S.l.rows * K;
  const int64_t t0 = tile0 + p.y * K;
  const bool packed = A.offsets != nullptr;
  Pack<T, V> x[K], r[K], i[K];
  unsigned on = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t t = t0 + k;
    x[k].zero();
    r[k].zero();
    i[k].zero();
    if (t < A.steps && p.live && (A.mask == nullptr || A.mask[p.b * A.m_sb + t * A.m_st] != 0)) {
      on |= 1u << k;
      const T* row = static_cast<const T*>(A.p) + p.b * A.p_sb + t * A.p_st + p.c;
      x[k].load(row);
      r[k].load(row + H);
      i[k].load(row + 2 * H);
    }
  }
  if (packed) mark_sequences(A, tile0, S.l.rows * K, first, last);
  float kd[V], init[V], a[K][V], add[K][V], ra[V], rb[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    kd[v] = p.live ? decay_factor(param_at(A.decay, A.decay_bf16, p.c + v), A.rate) : 0.f;
    init[v] = (!packed && p.live && A.h0 != nullptr) ? A.h0[p.b * H + p.c + v] : 0.f;
    ra[v] = 1.f;
    rb[v] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t t = t0 + k;
    float fx[V], fr[V], fi[V];
    x[k].get(fx);
    r[k].get(fr);
    i[k].get(fi);
    if constexpr (CODES) {
      if (t < A.steps) {  // the same for all lanes of a group
        const int64_t row = p.b * A.row_sb + t * A.row_st;
        int8_t code[V];
        int8_t* to = A.codes + row * 3 * H + p.c;
        float* sc = A.scales + row * 3 * G + p.c / kGroup8;
        const bool head = p.live && p.c % kGroup8 == 0;
        const float s0 = encode8(fx, code);
        if (p.live) store_codes(to, code);
        const float s1 = encode8(fr, code);
        if (p.live) store_codes(to + H, code);
        const float s2 = encode8(fi, code);
        if (p.live) store_codes(to + 2 * H, code);
        if (head) {
          sc[0] = s0;
          sc[G] = s1;
          sc[2 * G] = s2;
        }
      }
    }
    const int from = packed && t < A.steps ? first[p.y * K + k] : -1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      a[k][v] = 1.f;
      add[k][v] = 0.f;
      if (on >> k & 1) {
        const Step g = step_of(fr[v], fi[v], kd[v]);
        a[k][v] = g.a;
        add[k][v] = approx_sqrt(g.ss) * g.si * fx[v];
      }
      if (from >= 0) {
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
  if (A.states != nullptr && t0 > 0 && t0 < A.steps) {
    float* to = A.states + (p.b * A.n_states + t0 / K - 1) * H + p.c;
#pragma unroll
    for (int v = 0; v < V; ++v) to[v] = h[v];
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t t = t0 + k;
    if (t < A.steps) {
      const int from = packed ? first[p.y * K + k] : -1;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (from >= 0) h[v] = A.h0 != nullptr ? A.h0[static_cast<int64_t>(from) * H + p.c + v] : 0.f;
        h[v] = fmaf(a[k][v], h[v], add[k][v]);
      }
      Pack<T, V> o;
      o.set(h);
      o.store(static_cast<T*>(A.h) + (p.b * A.row_sb + t * A.row_st) * H + p.c);
      const int64_t done = packed ? last[p.y * K + k] : (t == A.steps - 1 ? p.b : -1);
      if (done >= 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) A.last[done * H + p.c + v] = h[v];
      }
    }
  }
}

// Walks from the last step to the first: run y of tile j covers the steps that end
// (j * rows + y) * K before the end of the last tile.
template <class T, int V, bool CODES>
__global__ void __launch_bounds__(256, 1) scan_tiles_bwd_kernel(const ScanArgs A, const TileShape S, const TileWork W) {
  constexpr int K = kStateEvery;
  extern __shared__ float2 smem[];
  float2* maps = smem;
  int* first = reinterpret_cast<int*>(maps + S.l.rows * S.l.count * V);
  int* last = first + S.l.rows * K;
  const int H = A.width;
  const int G = (H + kGroup8 - 1) / kGroup8;
  const Place p = place_of<V>(S, W, H);
  const int64_t tile = S.tiles - 1 - p.j;
  const int64_t tile0 = tile * S.l.rows * K;
  const int at0 = (S.l.rows - 1 - p.y) * K;  // inside the tile
  const int64_t t0 = tile0 + at0;
  const bool packed = A.offsets != nullptr;
  float x[K][V], r[K][V], i[K][V], d[K][V];
  unsigned on = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t t = t0 + k;
#pragma unroll
    for (int v = 0; v < V; ++v) x[k][v] = r[k][v] = i[k][v] = d[k][v] = 0.f;
    if (t < A.steps && p.live) {
      if (A.mask == nullptr || A.mask[p.b * A.m_sb + t * A.m_st] != 0) {
        on |= 1u << k;
        if constexpr (CODES) {
          const int64_t row = p.b * A.row_sb + t * A.row_st;
          const int8_t* from = A.codes + row * 3 * H + p.c;
          const float* sc = A.scales + row * 3 * G + p.c / kGroup8;
          load_codes(from, sc[0], x[k]);
          load_codes(from + H, sc[G], r[k]);
          load_codes(from + 2 * H, sc[2 * G], i[k]);
        } else {
          const T* row = static_cast<const T*>(A.p) + p.b * A.p_sb + t * A.p_st + p.c;
          Pack<T, V> w;
          w.load(row);
          w.get(x[k]);
          w.load(row + H);
          w.get(r[k]);
          w.load(row + 2 * H);
          w.get(i[k]);
        }
      }
      if (A.dh != nullptr) {
        Pack<T, V> w;
        w.load(static_cast<const T*>(A.dh) + p.b * A.dh_sb + t * A.dh_st + p.c);
        w.get(d[k]);
      }
    }
  }
  float h[V];  // the state before the run
#pragma unroll
  for (int v = 0; v < V; ++v) {
    h[v] = 0.f;
    if (p.live && t0 < A.steps) {
      if (t0 > 0)
        h[v] = A.states[(p.b * A.n_states + t0 / K - 1) * H + p.c + v];
      else if (!packed && A.h0 != nullptr)
        h[v] = A.h0[p.b * H + p.c + v];
    }
  }
  if (packed) mark_sequences(A, tile0, S.l.rows * K, first, last);
  float kd[V], init[V], ra[V], rb[V], dl[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    kd[v] = p.live ? decay_factor(param_at(A.decay, A.decay_bf16, p.c + v), A.rate) : 0.f;
    init[v] = (!packed && p.live && A.dlast != nullptr) ? A.dlast[p.b * H + p.c + v] : 0.f;
    ra[v] = 1.f;
    rb[v] = 0.f;
    dl[v] = 0.f;
  }
#pragma unroll
  for (int k = K - 1; k >= 0; --k) {
    if (t0 + k >= A.steps) continue;
    const int to = packed ? last[at0 + k] : -1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (to >= 0) {
        ra[v] = 0.f;
        rb[v] = (p.live && A.dlast != nullptr) ? A.dlast[static_cast<int64_t>(to) * H + p.c + v] : 0.f;
      }
      rb[v] += d[k][v];
      if (on >> k & 1) {
        const float a = 1.f - one_minus_exp(kd[v] * sigmoid_f(r[k][v]));
        ra[v] *= a;
        rb[v] *= a;
      }
    }
  }
  float E[V];
  tile_carry<V>(S, W, p, ra, rb, init, maps, E, A.status);
  float before[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (t0 + k >= A.steps) continue;
    const int from = packed ? first[at0 + k] : -1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (from >= 0) h[v] = (p.live && A.h0 != nullptr) ? A.h0[static_cast<int64_t>(from) * H + p.c + v] : 0.f;
      before[k][v] = h[v];
      if (on >> k & 1) {
        const Step g = step_of(r[k][v], i[k][v], kd[v]);
        h[v] = fmaf(g.a, h[v], approx_sqrt(g.ss) * g.si * x[k][v]);
      }
    }
  }
#pragma unroll
  for (int k = K - 1; k >= 0; --k) {
    const int64_t t = t0 + k;
    if (t >= A.steps || !p.live) continue;
    const int to = packed ? last[at0 + k] : -1;
    float dx[V], dr[V], di[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (to >= 0) E[v] = A.dlast != nullptr ? A.dlast[static_cast<int64_t>(to) * H + p.c + v] : 0.f;
      const float g = d[k][v] + E[v];
      if (on >> k & 1) {
        E[v] = step_grad(step_of(r[k][v], i[k][v], kd[v]), x[k][v], before[k][v], g, dx[v], dr[v], di[v], dl[v]);
      } else {
        E[v] = g;
        dx[v] = dr[v] = di[v] = 0.f;
      }
    }
    T* out = static_cast<T*>(A.dp) + (p.b * A.row_sb + t * A.row_st) * 3 * H + p.c;
    Pack<T, V> o;
    o.set(dx);
    o.store(out);
    o.set(dr);
    o.store(out + H);
    o.set(di);
    o.store(out + 2 * H);
    const int64_t begin = packed ? first[at0 + k] : (t == 0 ? p.b : -1);
    if (begin >= 0 && A.dh0 != nullptr) {
#pragma unroll
      for (int v = 0; v < V; ++v) A.dh0[begin * H + p.c + v] = E[v];
    }
  }
  // the tile's share of sum dz sigmoid(r), its runs added up in order
  float* sum = reinterpret_cast<float*>(maps);
  const int width = S.l.count * V;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) sum[p.y * width + p.x * V + v] = dl[v];
  __syncthreads();
  if (p.y == 0 && p.live) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float t = 0.f;
      for (int k = 0; k < S.l.rows; ++k) t += sum[k * width + p.x * V + v];
      A.partial[(p.b * S.tiles + tile) * H + p.c + v] = t;
    }
  }
}

// 4 bytes of channels per thread and step: 16 steps of three inputs, decays and additions
// have to fit its registers
int vec_of(const ScanArgs& a) { return a.bf16 && a.vec ? 2 : 1; }

TileShape shape_of(const ScanArgs& a, bool codes) {
  TileShape s;
  s.l = lanes_of(a.width, vec_of(a), codes, 32, 256);
  if (s.l.rows > 32) s.l.rows = 32;
  const int64_t steps = static_cast<int64_t>(s.l.rows) * kStateEvery;
  s.tiles = (a.steps + steps - 1) / steps;
  s.chains = (a.offsets != nullptr ? 1 : a.batch) * s.l.blocks;
  return s;
}

int64_t flag_count(const TileShape& s) {
  const int64_t groups = (s.tiles + kFan - 1) / kFan, blocks = (groups + kFan - 1) / kFan;
  return s.chains * (s.tiles + groups + blocks);
}

size_t smem_of(const ScanArgs& a, const TileShape& s) {
  size_t b = static_cast<size_t>(s.l.rows) * s.l.count * vec_of(a) * sizeof(float2);
  if (a.offsets != nullptr) b += static_cast<size_t>(s.l.rows) * kStateEvery * 2 * sizeof(int);
  return b;
}

TileWork work_of(const ScanArgs& a, const TileShape& s, void* buf) {
  const int64_t groups = (s.tiles + kFan - 1) / kFan, blocks = (groups + kFan - 1) / kFan;
  const int64_t width = s.l.count * vec_of(a);
  TileWork w;
  w.ticket = static_cast<unsigned long long*>(buf);
  w.tile_flag = reinterpret_cast<int*>(w.ticket + 1);
  w.group_flag = w.tile_flag + s.chains * s.tiles;
  w.block_flag = w.group_flag + s.chains * groups;
  const int64_t head = (8 + 4 * flag_count(s) + 15) / 16 * 16;
  w.tile_map = reinterpret_cast<float2*>(static_cast<char*>(buf) + head);
  w.group_map = w.tile_map + s.chains * s.tiles * width;
  w.block_state = reinterpret_cast<float*>(w.group_map + s.chains * groups * width);
  (void)blocks;
  return w;
}

template <class T, bool CODES>
void run_tiles(const ScanArgs& a, const TileShape& s, const TileWork& w, bool bwd, cudaStream_t st) {
  const unsigned blocks = static_cast<unsigned>(s.tiles * s.chains);
  const int threads = s.l.rows * s.l.count;
  const size_t smem = smem_of(a, s);
  if constexpr (sizeof(T) == 2) {
    if (vec_of(a) == 2) {
      if (bwd)
        scan_tiles_bwd_kernel<T, 2, CODES><<<blocks, threads, smem, st>>>(a, s, w);
      else
        scan_tiles_fwd_kernel<T, 2, CODES><<<blocks, threads, smem, st>>>(a, s, w);
      return;
    }
  }
  if (bwd)
    scan_tiles_bwd_kernel<T, 1, CODES><<<blocks, threads, smem, st>>>(a, s, w);
  else
    scan_tiles_fwd_kernel<T, 1, CODES><<<blocks, threads, smem, st>>>(a, s, w);
}

}  // namespace

int64_t scan_tiles_partials(const ScanArgs& a) {
  return (a.offsets != nullptr ? 1 : a.batch) * shape_of(a, a.codes != nullptr).tiles;
}

size_t scan_tiles_workspace(const ScanArgs& a) {
  const TileShape s = shape_of(a, a.codes != nullptr);
  const int64_t groups = (s.tiles + kFan - 1) / kFan, blocks = (groups + kFan - 1) / kFan;
  const int64_t width = s.l.count * vec_of(a);
  return (8 + 4 * flag_count(s) + 15) / 16 * 16 + s.chains * width * ((s.tiles + groups) * 8 + blocks * 4);
}

void launch_scan_tiles(const ScanArgs& a, bool bwd, void* workspace, cudaStream_t st) {
  const TileShape s = shape_of(a, a.codes != nullptr);
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
  cudaMemsetAsync(workspace, 0, 8 + 4 * flag_count(s), st);
  const TileWork w = work_of(a, s, workspace);
  count_launch();
  const bool codes = a.codes != nullptr;
  if (a.bf16)
    codes ? run_tiles<__nv_bfloat16, true>(a, s, w, bwd, st) : run_tiles<__nv_bfloat16, false>(a, s, w, bwd, st);
  else
    codes ? run_tiles<float, true>(a, s, w, bwd, st) : run_tiles<float, false>(a, s, w, bwd, st);
}

}  // namespace su
