// Gated linear recurrence over node histories (formulas in scan_math.cuh): a thread walks
// its channels of one sequence after another. Bound by bytes: forward reads the three
// input rows and writes h, backward reads the three and dh and writes three.
#include "kernels.h"
#include "scan_math.cuh"

namespace su {
namespace {

// ---------------------------------------------------------------------------
// A thread walks its V channels of one sequence after another.
// ---------------------------------------------------------------------------
template <class T, int V, int U, bool CODES>
__global__ void __launch_bounds__(256) scan_rows_fwd_kernel(const ScanArgs A, const Lanes L) {
  const int y = threadIdx.x / L.count;
  const int c = (blockIdx.y * L.count + threadIdx.x % L.count) * V;
  const bool live = c < A.width;
  if (!CODES && !live) return;
  const int H = A.width;
  const int G = (H + kGroup8 - 1) / kGroup8;
  float k[V];
#pragma unroll
  for (int v = 0; v < V; ++v) k[v] = live ? decay_factor(param_at(A.decay, A.decay_bf16, c + v), A.rate) : 0.f;
  const T* P = static_cast<const T*>(A.p) + c;
  T* Hout = static_cast<T*>(A.h) + c;
  for (int64_t s = static_cast<int64_t>(blockIdx.x) * L.rows + y; s < A.batch;
       s += static_cast<int64_t>(gridDim.x) * L.rows) {
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = (live && A.h0 != nullptr) ? A.h0[s * H + c + v] : 0.f;
    for (int64_t t0 = 0; t0 < A.steps; t0 += U) {
      Pack<T, V> x[U], r[U], i[U];
      bool on[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int64_t t = t0 + j;
        on[j] = t < A.steps && (A.mask == nullptr || A.mask[s * A.m_sb + t * A.m_st] != 0);
        x[j].zero();
        r[j].zero();
        i[j].zero();
        if (on[j] && live) {
          const T* row = P + s * A.p_sb + t * A.p_st;
          x[j].load(row);
          r[j].load(row + H);
          i[j].load(row + 2 * H);
        }
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int64_t t = t0 + j;
        if (t >= A.steps) break;
        if (A.states != nullptr && live && t > 0 && t % kStateEvery == 0) {
          float* to = A.states + (s * A.n_states + t / kStateEvery - 1) * H + c;
#pragma unroll
          for (int v = 0; v < V; ++v) to[v] = h[v];
        }
        float fx[V], fr[V], fi[V];
        x[j].get(fx);
        r[j].get(fr);
        i[j].get(fi);
        const int64_t row = s * A.row_sb + t * A.row_st;
        if constexpr (CODES) {
          int8_t code[V];
          int8_t* to = A.codes + row * 3 * H + c;
          float* sc = A.scales + (row * 3) * G + c / kGroup8;
          const bool first = (c % kGroup8) == 0 && live;
          const float s0 = encode8(fx, code);
          if (live) store_codes(to, code);
          const float s1 = encode8(fr, code);
          if (live) store_codes(to + H, code);
          const float s2 = encode8(fi, code);
          if (live) store_codes(to + 2 * H, code);
          if (first) {
            sc[0] = s0;
            sc[G] = s1;
            sc[2 * G] = s2;
          }
        }
        if (on[j]) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const Step g = step_of(fr[v], fi[v], k[v]);
            h[v] = fmaf(g.a, h[v], approx_sqrt(g.ss) * g.si * fx[v]);
          }
        }
        if (live) {
          Pack<T, V> o;
          o.set(h);
          o.store(Hout + row * H);
        }
      }
    }
    if (live) {
#pragma unroll
      for (int v = 0; v < V; ++v) A.last[s * H + c + v] = h[v];
    }
  }
}

// Backwards by chunks of CH steps (kStateEvery, or fewer where the sequence has no more):
// the states inside a chunk are recomputed from the state before it and kept in registers.
template <class T, int V, int CH, bool CODES>
__global__ void __launch_bounds__(256) scan_rows_bwd_kernel(const ScanArgs A, const Lanes L) {
  const int y = threadIdx.x / L.count;
  const int lane_c = threadIdx.x % L.count;
  const int c = (blockIdx.y * L.count + lane_c) * V;
  const bool live = c < A.width;
  const int H = A.width;
  const int G = (H + kGroup8 - 1) / kGroup8;
  float k[V], dl[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    k[v] = live ? decay_factor(param_at(A.decay, A.decay_bf16, c + v), A.rate) : 0.f;
    dl[v] = 0.f;
  }
  if (live) {
    for (int64_t s = static_cast<int64_t>(blockIdx.x) * L.rows + y; s < A.batch;
         s += static_cast<int64_t>(gridDim.x) * L.rows) {
      float E[V];
#pragma unroll
      for (int v = 0; v < V; ++v) E[v] = A.dlast != nullptr ? A.dlast[s * H + c + v] : 0.f;
      for (int64_t tc = (A.steps + CH - 1) / CH * CH - CH; tc >= 0; tc -= CH) {
        float x[CH][V], r[CH][V], i[CH][V], d[CH][V], before[CH][V];
        bool in[CH], on[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          const int64_t t = tc + j;
          in[j] = t < A.steps;
          on[j] = in[j] && (A.mask == nullptr || A.mask[s * A.m_sb + t * A.m_st] != 0);
#pragma unroll
          for (int v = 0; v < V; ++v) x[j][v] = r[j][v] = i[j][v] = d[j][v] = 0.f;
          if (on[j]) {
            if constexpr (CODES) {
              const int64_t row = s * A.row_sb + t * A.row_st;
              const int8_t* from = A.codes + row * 3 * H + c;
              const float* sc = A.scales + row * 3 * G + c / kGroup8;
              load_codes(from, sc[0], x[j]);
              load_codes(from + H, sc[G], r[j]);
              load_codes(from + 2 * H, sc[2 * G], i[j]);
            } else {
              const T* row = static_cast<const T*>(A.p) + s * A.p_sb + t * A.p_st + c;
              Pack<T, V> w;
              w.load(row);
              w.get(x[j]);
              w.load(row + H);
              w.get(r[j]);
              w.load(row + 2 * H);
              w.get(i[j]);
            }
          }
          if (in[j] && A.dh != nullptr) {
            Pack<T, V> w;
            w.load(static_cast<const T*>(A.dh) + s * A.dh_sb + t * A.dh_st + c);
            w.get(d[j]);
          }
        }
        float h[V];
        if (tc > 0) {
          const float* from = A.states + (s * A.n_states + tc / kStateEvery - 1) * H + c;
#pragma unroll
          for (int v = 0; v < V; ++v) h[v] = from[v];
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v) h[v] = A.h0 != nullptr ? A.h0[s * H + c + v] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < CH; ++j) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            before[j][v] = h[v];
            if (on[j]) {
              const Step g = step_of(r[j][v], i[j][v], k[v]);
              h[v] = fmaf(g.a, h[v], approx_sqrt(g.ss) * g.si * x[j][v]);
            }
          }
        }
#pragma unroll
        for (int j = CH - 1; j >= 0; --j) {
          if (!in[j]) continue;
          const int64_t row = s * A.row_sb + (tc + j) * A.row_st;
          float dx[V], dr[V], di[V];
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float g = d[j][v] + E[v];
            if (on[j]) {
              E[v] = step_grad(step_of(r[j][v], i[j][v], k[v]), x[j][v], before[j][v], g, dx[v], dr[v], di[v], dl[v]);
            } else {
              E[v] = g;
              dx[v] = dr[v] = di[v] = 0.f;
            }
          }
          T* to = static_cast<T*>(A.dp) + row * 3 * H + c;
          Pack<T, V> o;
          o.set(dx);
          o.store(to);
          o.set(dr);
          o.store(to + H);
          o.set(di);
          o.store(to + 2 * H);
        }
      }
      if (A.dh0 != nullptr) {
#pragma unroll
        for (int v = 0; v < V; ++v) A.dh0[s * H + c + v] = E[v];
      }
    }
  }
  // the block's share of sum dz sigmoid(r), added up over its rows in order
  __shared__ float sum[256 * V];
#pragma unroll
  for (int v = 0; v < V; ++v) sum[threadIdx.x * V + v] = dl[v];
  __syncthreads();
  if (y == 0 && live) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float t = 0.f;
      for (int w = 0; w < L.rows; ++w) t += sum[(w * L.count + lane_c) * V + v];
      A.partial[static_cast<int64_t>(blockIdx.x) * H + c + v] = t;
    }
  }
}

// Rows k, k + m, k + 2m, ... of partial [n, H] added up in order into row k of out [m, H]:
// 32 channels x 32 shares per block. `last`: out is ddecay, -c sigmoid(decay) times the sum.
__global__ void scan_decay_grad_kernel(const float* __restrict__ partial, int64_t n, int H, bool last, const void* decay,
                                       int decay_bf16, float rate, void* out) {
  __shared__ float sum[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float t = 0.f;
  if (c < H) {
#pragma unroll 4
    for (int64_t w = blockIdx.y + static_cast<int64_t>(threadIdx.y) * gridDim.y; w < n; w += 32ll * gridDim.y)
      t += partial[w * H + c];
  }
  sum[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.y == 0 && c < H) {
    for (int w = 1; w < 32; ++w) t += sum[w][threadIdx.x];
    if (last)
      param_store(out, decay_bf16, c, -rate * sigmoid_f(param_at(decay, decay_bf16, c)) * t);
    else
      static_cast<float*>(out)[static_cast<int64_t>(blockIdx.y) * H + c] = t;
  }
}

// One new token per row: thread per channel, states read and written in place.
template <class T>
__global__ void __launch_bounds__(256) scan_step_kernel(const ScanStepArgs A) {
  const int64_t n = A.rows * A.width;
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (e >= n) return;
  const int64_t row = e / A.width;
  const int c = static_cast<int>(e - row * A.width);
  const T* p = static_cast<const T*>(A.p) + row * A.p_sb + c;
  const float x = to_f32(p[0]), r = to_f32(p[A.width]), i = to_f32(p[2 * static_cast<int64_t>(A.width)]);
  const float k = decay_factor(param_at(A.decay, A.decay_bf16, c), A.rate);
  const int64_t at = A.index != nullptr ? A.index[row] : row;
  float h = 0.f;
  if (at < 0 || at >= A.table_rows) {
    record_status(A.status, kBadIndex);  // the row is left out
  } else {
    float* to = A.state + at * A.state_sb + c;
    const Step g = step_of(r, i, k);
    h = fmaf(g.a, *to, approx_sqrt(g.ss) * g.si * x);
    *to = h;
  }
  static_cast<T*>(A.h)[e] = from_f32<T>(h);
}

// blocks over the sequences: every SM filled a few times, so that per-block sums stay few
int row_blocks(const ScanArgs& a, const Lanes& l, int sms) {
  const int64_t want = (a.batch + l.rows - 1) / l.rows;
  const int64_t most = (static_cast<int64_t>(sms) * 8 + l.blocks - 1) / l.blocks;
  return static_cast<int>(want < most ? want : most);
}

struct BwdShape {
  int V, CH;
};
// 16 bytes of a channel per thread and step where the whole sequence is one short chunk,
// 4 bytes where 16 steps of inputs and states have to stay in registers
BwdShape bwd_shape(const ScanArgs& a) {
  if (a.steps <= 4) return {a.vec ? 4 : 1, 4};
  if (a.steps <= 8) return {a.vec ? 2 : 1, 8};
  return {a.vec && a.bf16 ? 2 : 1, kStateEvery};
}

template <class T, bool CODES>
void rows_fwd(const ScanArgs& a, int sms, cudaStream_t st) {
  const Lanes l = lanes_of(a.width, a.vec ? 4 : 1, CODES, 256, 256);
  const dim3 grid(row_blocks(a, l, sms), l.blocks);
  const int threads = l.count * l.rows;
  if (a.vec)
    scan_rows_fwd_kernel<T, 4, 4, CODES><<<grid, threads, 0, st>>>(a, l);
  else
    scan_rows_fwd_kernel<T, 1, 8, CODES><<<grid, threads, 0, st>>>(a, l);
}

template <class T, bool CODES>
void rows_bwd(const ScanArgs& a, int sms, cudaStream_t st) {
  const BwdShape b = bwd_shape(a);
  const Lanes l = lanes_of(a.width, b.V, false, 256, 256);
  const dim3 grid(row_blocks(a, l, sms), l.blocks);
  const int threads = l.count * l.rows;
  if (b.CH == 4) {
    if (b.V == 4)
      scan_rows_bwd_kernel<T, 4, 4, CODES><<<grid, threads, 0, st>>>(a, l);
    else
      scan_rows_bwd_kernel<T, 1, 4, CODES><<<grid, threads, 0, st>>>(a, l);
  } else if (b.CH == 8) {
    if (b.V == 2)
      scan_rows_bwd_kernel<T, 2, 8, CODES><<<grid, threads, 0, st>>>(a, l);
    else
      scan_rows_bwd_kernel<T, 1, 8, CODES><<<grid, threads, 0, st>>>(a, l);
  } else {
    if (b.V == 2)
      scan_rows_bwd_kernel<T, 2, kStateEvery, CODES><<<grid, threads, 0, st>>>(a, l);
    else
      scan_rows_bwd_kernel<T, 1, kStateEvery, CODES><<<grid, threads, 0, st>>>(a, l);
  }
}

// Tiles for packed sequences, and where a thread per sequence and 4 channels leaves the SMs
// short of threads; a sequence of one chunk has nothing to split.
bool in_tiles(const ScanArgs& a, int sms) {
  if (a.offsets != nullptr) return true;
  if (a.steps <= kStateEvery) return false;
  return a.batch * ((a.width + (a.vec ? 3 : 0)) / (a.vec ? 4 : 1)) < static_cast<int64_t>(sms) * 512;
}

constexpr int64_t kSumRows = 64;  // above it the partial sums are added up in two launches
int64_t partial_rows(const ScanArgs& a, int sms) {
  return in_tiles(a, sms) ? scan_tiles_partials(a)
                          : row_blocks(a, lanes_of(a.width, bwd_shape(a).V, false, 256, 256), sms);
}

}  // namespace

size_t scan_workspace(const ScanArgs& a, int sms) { return in_tiles(a, sms) ? scan_tiles_workspace(a) : 0; }

int64_t scan_partials(const ScanArgs& a, int sms) {
  const int64_t n = partial_rows(a, sms);
  return n > 8 * kSumRows ? n + kSumRows : n;
}

void launch_scan_fwd(const ScanArgs& a, int sms, void* workspace, cudaStream_t st) {
  if (in_tiles(a, sms)) return launch_scan_tiles(a, false, workspace, st);
  count_launch();
  const bool codes = a.codes != nullptr;
  if (a.bf16)
    codes ? rows_fwd<__nv_bfloat16, true>(a, sms, st) : rows_fwd<__nv_bfloat16, false>(a, sms, st);
  else
    codes ? rows_fwd<float, true>(a, sms, st) : rows_fwd<float, false>(a, sms, st);
}

void launch_scan_bwd(const ScanArgs& a, int sms, void* workspace, void* ddecay, cudaStream_t st) {
  const bool codes = a.codes != nullptr;
  if (in_tiles(a, sms)) {
    launch_scan_tiles(a, true, workspace, st);
  } else {
    count_launch();
    if (a.bf16)
      codes ? rows_bwd<__nv_bfloat16, true>(a, sms, st) : rows_bwd<__nv_bfloat16, false>(a, sms, st);
    else
      codes ? rows_bwd<float, true>(a, sms, st) : rows_bwd<float, false>(a, sms, st);
  }
  int64_t n = partial_rows(a, sms);
  const float* from = a.partial;
  const int cols = (a.width + 31) / 32;
  const dim3 threads(32, 32);
  if (n > 8 * kSumRows) {
    float* to = a.partial + n * a.width;
    count_launch();
    scan_decay_grad_kernel<<<dim3(cols, kSumRows), threads, 0, st>>>(from, n, a.width, false, a.decay, a.decay_bf16,
                                                                     a.rate, to);
    from = to;
    n = kSumRows;
  }
  count_launch();
  scan_decay_grad_kernel<<<cols, threads, 0, st>>>(from, n, a.width, true, a.decay, a.decay_bf16, a.rate, ddecay);
}

void launch_scan_step(const ScanStepArgs& a, cudaStream_t st) {
  count_launch();
  const int64_t n = a.rows * a.width;
  const unsigned blocks = static_cast<unsigned>((n + 255) / 256);
  if (a.bf16)
    scan_step_kernel<__nv_bfloat16><<<blocks, 256, 0, st>>>(a);
  else
    scan_step_kernel<float><<<blocks, 256, 0, st>>>(a);
}

}  // namespace su
