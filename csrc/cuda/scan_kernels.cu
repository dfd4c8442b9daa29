// Gated linear recurrence over node histories (formulas in scan_math.cuh): a thread walks
// its channels of one sequence after another. Bound by bytes: forward reads the three
// input rows and writes h, backward reads the three and dh and writes three.
#include "kernels.h"
#include "scan_math.cuh"

namespace su {
namespace {

// Forward by U steps: their inputs are loaded together, so that U x 3 loads of 4 V (fp32)
// bytes are under way per thread.
template <class T, int V, int U, bool CODES, bool MASK>
__global__ void __launch_bounds__(256) scan_rows_fwd_kernel(const ScanArgs A, const Lanes L) {
  const int y = threadIdx.x / L.count;
  const int c = (blockIdx.y * L.count + threadIdx.x % L.count) * V;
  const bool live = c < A.width;
  if (!CODES && !live) return;
  const int H = A.width;
  const int G = (H + kGroup8 - 1) / kGroup8;
  const int steps = static_cast<int>(A.steps);
  float k[V];
#pragma unroll
  for (int v = 0; v < V; ++v) k[v] = live ? decay_factor(param_at(A.decay, A.decay_bf16, c + v), A.rate) : 0.f;
  for (int64_t s = static_cast<int64_t>(blockIdx.x) * L.rows + y; s < A.batch;
       s += static_cast<int64_t>(gridDim.x) * L.rows) {
    const T* in = static_cast<const T*>(A.p) + s * A.p_sb + c;
    const uint8_t* valid = MASK ? A.mask + s * A.m_sb : nullptr;
    T* out = static_cast<T*>(A.h) + s * A.row_sb * H + c;
    int8_t* code = CODES ? A.codes + s * A.row_sb * 3 * H + c : nullptr;
    float* scale = CODES ? A.scales + s * A.row_sb * 3 * G + c / kGroup8 : nullptr;
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = (live && A.h0 != nullptr) ? A.h0[s * H + c + v] : 0.f;
    for (int t0 = 0; t0 < steps; t0 += U) {
      Pack<T, V> x[U], r[U], i[U];
      bool on[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        on[j] = t0 + j < steps && (!MASK || *valid != 0);
        x[j].zero();
        r[j].zero();
        i[j].zero();
        if (on[j] && live) {
          x[j].load(in);
          r[j].load(in + H);
          i[j].load(in + 2 * H);
        }
        in += A.p_st;
        if (MASK && t0 + j + 1 < steps) valid += A.m_st;
      }
      if (A.states != nullptr && live && t0 > 0 && t0 % kStateEvery == 0) {  // U divides kStateEvery
        float* to = A.states + (s * A.n_states + t0 / kStateEvery - 1) * H + c;
#pragma unroll
        for (int v = 0; v < V; ++v) to[v] = h[v];
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (t0 + j >= steps) break;
        float fx[V], fr[V], fi[V];
        x[j].get(fx);
        r[j].get(fr);
        i[j].get(fi);
        if constexpr (CODES) {
          Codes<V> q[3];
          const float s0 = encode8(fx, q[0]), s1 = encode8(fr, q[1]), s2 = encode8(fi, q[2]);
          if (live) {
            q[0].store(code);
            q[1].store(code + H);
            q[2].store(code + 2 * H);
            if (c % kGroup8 == 0) {
              scale[0] = s0;
              scale[G] = s1;
              scale[2 * G] = s2;
            }
          }
          code += A.row_st * 3 * H;
          scale += A.row_st * 3 * G;
        }
        if (!MASK || on[j]) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const Step g = step_of(fx[v], fr[v], fi[v], k[v]);
            h[v] = fmaf(g.a, h[v], g.add);
          }
        }
        if (live) {
          Pack<T, V> o;
          o.set(h);
          o.store(out);
        }
        out += A.row_st * H;
      }
    }
    if (live) {
#pragma unroll
      for (int v = 0; v < V; ++v) A.last[s * H + c + v] = h[v];
    }
  }
}

// Backwards by chunks of CH steps (kStateEvery, or fewer where the sequence has no more).
// Every gradient of a step is g times a factor that the inputs and the state before the
// step give: the chunk is walked forwards from its first state for the factors, which stay
// in registers, and then backwards for g. The gates are evaluated once.
template <class T, int V, int CH, bool CODES, bool MASK>
__global__ void __launch_bounds__(256, 2) scan_rows_bwd_kernel(const ScanArgs A, const Lanes L) {
  const int y = threadIdx.x / L.count;
  const int lane_c = threadIdx.x % L.count;
  const int c = (blockIdx.y * L.count + lane_c) * V;
  const bool live = c < A.width;
  const int H = A.width;
  const int G = (H + kGroup8 - 1) / kGroup8;
  const int steps = static_cast<int>(A.steps);
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
      for (int tc = (steps + CH - 1) / CH * CH - CH; tc >= 0; tc -= CH) {
        const int64_t row = s * A.row_sb + tc * A.row_st;
        Pack<T, V> x[CH], r[CH], i[CH], d[CH];
        Codes<V> qx[CH], qr[CH], qi[CH];
        float sx[CH], sr[CH], si[CH];
        bool on[CH];
        const T* in = CODES ? nullptr : static_cast<const T*>(A.p) + s * A.p_sb + tc * A.p_st + c;
        const T* dh = static_cast<const T*>(A.dh) + (A.dh != nullptr ? s * A.dh_sb + tc * A.dh_st + c : 0);
        const int8_t* code = CODES ? A.codes + row * 3 * H + c : nullptr;
        const float* scale = CODES ? A.scales + row * 3 * G + c / kGroup8 : nullptr;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          const bool inside = tc + j < steps;
          on[j] = inside && (!MASK || A.mask[s * A.m_sb + (tc + j) * A.m_st] != 0);
          d[j].zero();
          if constexpr (CODES) {
            qx[j].zero();
            qr[j].zero();
            qi[j].zero();
            sx[j] = sr[j] = si[j] = 0.f;
            if (on[j]) {
              qx[j].load(code);
              qr[j].load(code + H);
              qi[j].load(code + 2 * H);
              sx[j] = scale[0];
              sr[j] = scale[G];
              si[j] = scale[2 * G];
            }
            code += A.row_st * 3 * H;
            scale += A.row_st * 3 * G;
          } else {
            x[j].zero();
            r[j].zero();
            i[j].zero();
            if (on[j]) {
              x[j].load(in);
              r[j].load(in + H);
              i[j].load(in + 2 * H);
            }
            in += A.p_st;
          }
          if (inside && A.dh != nullptr) d[j].load(dh);
          dh += A.dh_st;
        }
        float h[V];
        const float* from = tc > 0 ? A.states + (s * A.n_states + tc / kStateEvery - 1) * H + c
                                   : (A.h0 != nullptr ? A.h0 + s * H + c : nullptr);
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = from != nullptr ? from[v] : 0.f;
        Slope f[CH][V];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          float fx[V], fr[V], fi[V];
          if constexpr (CODES) {
            qx[j].get(sx[j], fx);
            qr[j].get(sr[j], fr);
            qi[j].get(si[j], fi);
          } else {
            x[j].get(fx);
            r[j].get(fr);
            i[j].get(fi);
          }
#pragma unroll
          for (int v = 0; v < V; ++v) {
            f[j][v] = slope_of(on[j] ? gate_of(fx[v], fr[v], fi[v], k[v]) : gate_shut(), h[v]);
          }
        }
        T* out = static_cast<T*>(A.dp) + (row + CH * A.row_st) * 3 * H + c;
#pragma unroll
        for (int j = CH - 1; j >= 0; --j) {
          out -= A.row_st * 3 * H;
          if (tc + j >= steps) continue;
          float dy[V], dx[V], dr[V], di[V];
          d[j].get(dy);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float g = dy[v] + E[v];
            dx[v] = g * f[j][v].x;
            dr[v] = g * f[j][v].r;
            di[v] = g * f[j][v].i;
            dl[v] = fmaf(g, f[j][v].l, dl[v]);
            E[v] = g * f[j][v].a;
          }
          Pack<T, V> o;
          o.set(dx);
          o.store(out);
          o.set(dr);
          o.store(out + H);
          o.set(di);
          o.store(out + 2 * H);
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
    const Step g = step_of(x, r, i, k);
    h = fmaf(g.a, *to, g.add);
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
// 16 steps' factors of one channel fit the registers, so do 8 of two and 4 of four
BwdShape bwd_shape(const ScanArgs& a) {
  if (a.steps <= 4) return {a.vec ? 4 : 1, 4};
  if (a.steps <= 8) return {a.vec ? 2 : 1, 8};
  return {1, kStateEvery};
}

template <class T, bool CODES, bool MASK>
void rows_fwd(const ScanArgs& a, int sms, cudaStream_t st) {
  const Lanes l = lanes_of(a.width, a.vec ? 4 : 1, CODES, 256, 256);
  const dim3 grid(row_blocks(a, l, sms), l.blocks);
  const int threads = l.count * l.rows;
  if (a.vec)
    scan_rows_fwd_kernel<T, 4, 4, CODES, MASK><<<grid, threads, 0, st>>>(a, l);
  else
    scan_rows_fwd_kernel<T, 1, 8, CODES, MASK><<<grid, threads, 0, st>>>(a, l);
}

template <class T, bool CODES, bool MASK>
void rows_bwd(const ScanArgs& a, int sms, cudaStream_t st) {
  const BwdShape b = bwd_shape(a);
  const Lanes l = lanes_of(a.width, b.V, false, 256, 256);
  const dim3 grid(row_blocks(a, l, sms), l.blocks);
  const int threads = l.count * l.rows;
  if (b.CH == 4) {
    if (b.V == 4)
      scan_rows_bwd_kernel<T, 4, 4, CODES, MASK><<<grid, threads, 0, st>>>(a, l);
    else
      scan_rows_bwd_kernel<T, 1, 4, CODES, MASK><<<grid, threads, 0, st>>>(a, l);
  } else if (b.CH == 8) {
    if (b.V == 2)
      scan_rows_bwd_kernel<T, 2, 8, CODES, MASK><<<grid, threads, 0, st>>>(a, l);
    else
      scan_rows_bwd_kernel<T, 1, 8, CODES, MASK><<<grid, threads, 0, st>>>(a, l);
  } else {
    scan_rows_bwd_kernel<T, 1, kStateEvery, CODES, MASK><<<grid, threads, 0, st>>>(a, l);
  }
}

template <class T, bool CODES>
void rows_run(const ScanArgs& a, bool bwd, int sms, cudaStream_t st) {
  if (a.mask != nullptr)
    bwd ? rows_bwd<T, CODES, true>(a, sms, st) : rows_fwd<T, CODES, true>(a, sms, st);
  else
    bwd ? rows_bwd<T, CODES, false>(a, sms, st) : rows_fwd<T, CODES, false>(a, sms, st);
}
void rows_launch(const ScanArgs& a, bool bwd, int sms, cudaStream_t st) {
  count_launch();
  const bool codes = a.codes != nullptr;
  if (a.bf16)
    codes ? rows_run<__nv_bfloat16, true>(a, bwd, sms, st) : rows_run<__nv_bfloat16, false>(a, bwd, sms, st);
  else
    codes ? rows_run<float, true>(a, bwd, sms, st) : rows_run<float, false>(a, bwd, sms, st);
}

// Tiles for packed sequences, and where a thread per sequence and 4 channels leaves the SMs
// short of threads; a sequence of one chunk has nothing to split.
bool in_tiles(const ScanArgs& a, int sms) {
  if (a.offsets != nullptr || a.steps > (1 << 30)) return true;
  if (a.steps <= kStateEvery) return false;
  return a.batch * ((a.width + (a.vec ? 3 : 0)) / (a.vec ? 4 : 1)) < static_cast<int64_t>(sms) * 512;
}

constexpr int64_t kSumRows = 64;  // above 8 times it the partial sums are added up in two launches
int64_t partial_rows(const ScanArgs& a, int sms) {
  return in_tiles(a, sms) ? scan_tiles_partials(a)
                          : row_blocks(a, lanes_of(a.width, bwd_shape(a).V, false, 256, 256), sms);
}

}  // namespace

size_t scan_workspace(const ScanArgs& a, bool bwd, int sms) {
  return in_tiles(a, sms) ? scan_tiles_workspace(a, bwd) : 0;
}

int64_t scan_partials(const ScanArgs& a, int sms) {
  const int64_t n = partial_rows(a, sms);
  return n > 8 * kSumRows ? n + kSumRows : n;
}

void launch_scan_fwd(const ScanArgs& a, int sms, void* workspace, cudaStream_t st) {
  if (in_tiles(a, sms))
    launch_scan_tiles(a, false, workspace, st);
  else
    rows_launch(a, false, sms, st);
}

void launch_scan_bwd(const ScanArgs& a, int sms, void* workspace, void* ddecay, cudaStream_t st) {
  if (in_tiles(a, sms))
    launch_scan_tiles(a, true, workspace, st);
  else
    rows_launch(a, true, sms, st);
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
