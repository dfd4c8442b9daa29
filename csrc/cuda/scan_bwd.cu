// Gated linear recurrence, backward (formulas in scan_math.cuh): a thread walks its channels
// through one segment of one sequence, last step to first.
#include "scan_shape.cuh"

namespace su {
namespace {

// V values of each of x, r and i of one step: the inputs, or their 8-bit codes and scales.
template <class T, int V, bool CODES>
struct Inputs;
template <class T, int V>
struct Inputs<T, V, false> {
  Pack<T, V> v[3];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int w = 0; w < 3; ++w) v[w].zero();
  }
  __device__ __forceinline__ void load(const T* p, const float*, int H, int) {
#pragma unroll
    for (int w = 0; w < 3; ++w) v[w].load(p + w * static_cast<int64_t>(H));
  }
  __device__ __forceinline__ void get(int w, float (&f)[V]) const { v[w].get(f); }
};
template <class T, int V>
struct Inputs<T, V, true> {
  Codes<V> v[3];
  float scale[3];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int w = 0; w < 3; ++w) {
      v[w].zero();
      scale[w] = 0.f;
    }
  }
  __device__ __forceinline__ void load(const int8_t* p, const float* s, int H, int G) {
#pragma unroll
    for (int w = 0; w < 3; ++w) {
      v[w].load(p + w * static_cast<int64_t>(H));
      scale[w] = s[w * static_cast<int64_t>(G)];
    }
  }
  __device__ __forceinline__ void get(int w, float (&f)[V]) const { v[w].get(scale[w], f); }
};

// Chunks of CH steps (kStateEvery, or fewer where the sequence has no more). Every gradient
// of a step is g times a factor that the inputs and the state before the step give: the
// chunk is walked forwards from its first state for the factors, which stay in registers,
// and then backwards for g. The gates are evaluated once.
template <class T, int V, int CH, bool CODES, int KIND>
__global__ void __launch_bounds__(256, 2) scan_bwd_kernel(const ScanArgs A, const ScanPlan P, const Lanes L) {
  const int y = threadIdx.x / L.count;
  const int lane_c = threadIdx.x % L.count;
  const int c = (blockIdx.y * L.count + lane_c) * V;
  const bool live = c < A.width;
  const int H = A.width;
  const int G = (H + kGroup8 - 1) / kGroup8;
  const int64_t batch = KIND == kPacked ? 1 : A.batch;
  const int64_t rows = live ? batch * P.seg.n : 0;
  float k[V], dl[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    k[v] = live ? decay_factor(param_at(A.decay, A.decay_bf16, c + v), A.rate) : 0.f;
    dl[v] = 0.f;
  }
  for (int64_t rr = static_cast<int64_t>(blockIdx.x) * L.rows + y; rr < rows;
       rr += static_cast<int64_t>(gridDim.x) * L.rows) {
    const SegRow s = seg_row(rr, batch, P.seg, false);
    const int64_t begin = s.q * P.seg.len;
    const int steps = static_cast<int>(min(P.seg.len, A.steps - begin));
    float E[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      E[v] = 0.f;
      if (P.seg.n > 1)
        E[v] = P.carry[(s.q * batch + s.b) * H + c + v];
      else if (KIND != kPacked && A.dlast != nullptr)
        E[v] = A.dlast[s.b * H + c + v];
    }
    for (int tc = (steps + CH - 1) / CH * CH - CH; tc >= 0; tc -= CH) {
      const int64_t t0 = begin + tc;
      const int64_t row = s.b * A.row_sb + t0 * A.row_st;
      Inputs<T, V, CODES> w[CH];
      Pack<T, V> d[CH];
      unsigned on = 0, firsts = 0, lasts = 0;
      {
        const auto* in = [&] {
          if constexpr (CODES)
            return A.codes + row * 3 * H + c;
          else
            return static_cast<const T*>(A.p) + s.b * A.p_sb + t0 * A.p_st + c;
        }();
        const int64_t in_st = CODES ? A.row_st * 3 * H : A.p_st;
        const float* scale = CODES ? A.scales + row * 3 * G + c / kGroup8 : nullptr;
        const T* dh = static_cast<const T*>(A.dh) + (A.dh != nullptr ? s.b * A.dh_sb + t0 * A.dh_st + c : 0);
        const uint8_t* valid = A.mask != nullptr ? A.mask + s.b * A.m_sb + t0 * A.m_st : nullptr;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          const bool inside = tc + j < steps;
          bool step = inside;
          if (KIND == kMasked || (KIND == kPacked && valid != nullptr)) {
            if (inside) step = *valid != 0;
            valid += A.m_st;
          }
          if (KIND == kPacked) {
            const int mk = inside ? A.marks[t0 + j] : -1;
            if (mk >= 0) {
              firsts |= static_cast<unsigned>(mk & kMarkFirst) << j;
              lasts |= static_cast<unsigned>((mk & kMarkLast) >> 1) << j;
            }
          }
          if (step) on |= 1u << j;
          w[j].zero();
          if (step) w[j].load(in, scale, H, G);
          in += in_st;
          if (CODES) scale += A.row_st * 3 * G;
          d[j].zero();
          if (inside && A.dh != nullptr) d[j].load(dh);
          dh += A.dh_st;
        }
      }
      float h[V];
      const float* from = t0 > 0 ? A.states + (s.b * A.n_states + t0 / kStateEvery - 1) * H + c
                                 : (KIND != kPacked && A.h0 != nullptr ? A.h0 + s.b * H + c : nullptr);
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = from != nullptr ? from[v] : 0.f;
      Slope f[CH][V];
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        if (KIND == kPacked && (firsts >> j & 1)) {
          const int64_t q = A.marks[t0 + j] >> 2;
#pragma unroll
          for (int v = 0; v < V; ++v) h[v] = A.h0 != nullptr ? A.h0[q * H + c + v] : 0.f;
        }
        float fx[V], fr[V], fi[V];
        w[j].get(0, fx);
        w[j].get(1, fr);
        w[j].get(2, fi);
#pragma unroll
        for (int v = 0; v < V; ++v)
          f[j][v] = slope_of(on >> j & 1 ? gate_of(fx[v], fr[v], fi[v], k[v]) : gate_shut(), h[v]);
      }
      T* out = static_cast<T*>(A.dp) + (row + CH * A.row_st) * 3 * H + c;
#pragma unroll
      for (int j = CH - 1; j >= 0; --j) {
        out -= A.row_st * 3 * H;
        if (tc + j >= steps) continue;
        if (KIND == kPacked && (lasts >> j & 1)) {
          const int64_t q = A.marks[t0 + j] >> 2;
#pragma unroll
          for (int v = 0; v < V; ++v) E[v] = A.dlast != nullptr ? A.dlast[q * H + c + v] : 0.f;
        }
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
        if (KIND == kPacked && (firsts >> j & 1) && A.dh0 != nullptr) {
          const int64_t q = A.marks[t0 + j] >> 2;
#pragma unroll
          for (int v = 0; v < V; ++v) A.dh0[q * H + c + v] = E[v];
        }
      }
    }
    if (KIND != kPacked && s.q == 0 && A.dh0 != nullptr) {
#pragma unroll
      for (int v = 0; v < V; ++v) A.dh0[s.b * H + c + v] = E[v];
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

// The map of E = a (dh + E) over a segment, last step to first: only r and dh are read.
template <class T, int V, int U, bool CODES, int KIND>
__global__ void __launch_bounds__(256) scan_bwd_maps_kernel(const ScanArgs A, const ScanPlan P, const Lanes L) {
  const int y = threadIdx.x / L.count;
  const int c = (blockIdx.y * L.count + threadIdx.x % L.count) * V;
  if (c >= A.width) return;
  const int H = A.width;
  const int G = (H + kGroup8 - 1) / kGroup8;
  const int64_t batch = KIND == kPacked ? 1 : A.batch;
  const int64_t rows = batch * P.seg.n;
  float k[V];
#pragma unroll
  for (int v = 0; v < V; ++v) k[v] = decay_factor(param_at(A.decay, A.decay_bf16, c + v), A.rate);
  for (int64_t rr = static_cast<int64_t>(blockIdx.x) * L.rows + y; rr < rows;
       rr += static_cast<int64_t>(gridDim.x) * L.rows) {
    // the first segments last: the pass that follows begins with them
    const SegRow s = seg_row(rr, batch, P.seg, true);
    const int64_t begin = s.q * P.seg.len;
    const int steps = static_cast<int>(min(P.seg.len, A.steps - begin));
    float m[V], E[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      m[v] = 1.f;
      E[v] = 0.f;
    }
    for (int tc = (steps + U - 1) / U * U - U; tc >= 0; tc -= U) {
      const int64_t t0 = begin + tc;
      Pack<T, V> r[U], d[U];
      Codes<V> q[U];
      float scale[U];
      bool on[U];
      int mk[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int64_t t = t0 + j;
        const bool inside = tc + j < steps;
        on[j] = inside;
        if (KIND == kMasked || (KIND == kPacked && A.mask != nullptr))
          on[j] = inside && A.mask[s.b * A.m_sb + t * A.m_st] != 0;
        mk[j] = -1;
        if (KIND == kPacked) {
          if (inside) mk[j] = A.marks[t];
        }
        r[j].zero();
        q[j].zero();
        scale[j] = 0.f;
        if (on[j]) {
          if constexpr (CODES) {
            const int64_t row = s.b * A.row_sb + t * A.row_st;
            q[j].load(A.codes + row * 3 * H + H + c);
            scale[j] = A.scales[row * 3 * G + G + c / kGroup8];
          } else {
            r[j].load_keep(static_cast<const T*>(A.p) + s.b * A.p_sb + t * A.p_st + H + c);
          }
        }
        d[j].zero();
        if (inside && A.dh != nullptr) d[j].load_keep(static_cast<const T*>(A.dh) + s.b * A.dh_sb + t * A.dh_st + c);
      }
#pragma unroll
      for (int j = U - 1; j >= 0; --j) {
        if (KIND == kPacked && mk[j] >= 0 && (mk[j] & kMarkLast)) {
          const float* from = A.dlast != nullptr ? A.dlast + static_cast<int64_t>(mk[j] >> 2) * H + c : nullptr;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            E[v] = from != nullptr ? from[v] : 0.f;
            m[v] = 0.f;
          }
        }
        float fr[V], fd[V];
        d[j].get(fd);
        if constexpr (CODES)
          q[j].get(scale[j], fr);
        else
          r[j].get(fr);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          E[v] += fd[v];
          if (on[j]) {
            const float a = decay_of(fr[v], k[v]);
            E[v] *= a;
            m[v] *= a;
          }
        }
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) P.maps[(s.q * batch + s.b) * H + c + v] = make_float2(m[v], E[v]);
  }
}

struct BwdShape {
  int V, CH;
};
// 16 steps' factors of one channel fit the registers, so do 8 of two and 4 of four
BwdShape bwd_shape(const ScanArgs& a) {
  if (a.offsets == nullptr && a.steps <= 4) return {a.vec ? 4 : 1, 4};
  if (a.offsets == nullptr && a.steps <= 8) return {a.vec ? 2 : 1, 8};
  return {1, kStateEvery};
}

template <class T, bool CODES, int KIND>
void run(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) {
  const BwdShape b = bwd_shape(a);
  const Lanes l = lanes_of(a.width, b.V, false);
  const dim3 grid(scan_bwd_blocks(a, p, sms), l.blocks);
  const int threads = l.count * l.rows;
  if constexpr (KIND != kPacked) {
    if (b.CH == 4) {
      if (b.V == 4)
        scan_bwd_kernel<T, 4, 4, CODES, KIND><<<grid, threads, 0, st>>>(a, p, l);
      else
        scan_bwd_kernel<T, 1, 4, CODES, KIND><<<grid, threads, 0, st>>>(a, p, l);
      return;
    }
    if (b.CH == 8) {
      if (b.V == 2)
        scan_bwd_kernel<T, 2, 8, CODES, KIND><<<grid, threads, 0, st>>>(a, p, l);
      else
        scan_bwd_kernel<T, 1, 8, CODES, KIND><<<grid, threads, 0, st>>>(a, p, l);
      return;
    }
  }
  scan_bwd_kernel<T, 1, kStateEvery, CODES, KIND><<<grid, threads, 0, st>>>(a, p, l);
}

template <class T, bool CODES, int KIND>
void run_maps(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) {
  const Lanes l = lanes_of(a.width, a.vec ? 4 : 1, false);
  const int64_t rows = (a.offsets != nullptr ? 1 : a.batch) * p.seg.n;
  const dim3 grid(row_blocks(rows, l, sms), l.blocks);
  const int threads = l.count * l.rows;
  if (a.vec)
    scan_bwd_maps_kernel<T, 4, 4, CODES, KIND><<<grid, threads, 0, st>>>(a, p, l);
  else
    scan_bwd_maps_kernel<T, 1, 8, CODES, KIND><<<grid, threads, 0, st>>>(a, p, l);
}

template <class T, bool CODES>
void run(const ScanArgs& a, const ScanPlan& p, bool maps, int sms, cudaStream_t st) {
  count_launch();
  switch (kind_of(a)) {
    case kPlain:
      return maps ? run_maps<T, CODES, kPlain>(a, p, sms, st) : run<T, CODES, kPlain>(a, p, sms, st);
    case kMasked:
      return maps ? run_maps<T, CODES, kMasked>(a, p, sms, st) : run<T, CODES, kMasked>(a, p, sms, st);
    default:
      return maps ? run_maps<T, CODES, kPacked>(a, p, sms, st) : run<T, CODES, kPacked>(a, p, sms, st);
  }
}

void run(const ScanArgs& a, const ScanPlan& p, bool maps, int sms, cudaStream_t st) {
  if (a.codes != nullptr)
    a.bf16 ? run<__nv_bfloat16, true>(a, p, maps, sms, st) : run<float, true>(a, p, maps, sms, st);
  else
    a.bf16 ? run<__nv_bfloat16, false>(a, p, maps, sms, st) : run<float, false>(a, p, maps, sms, st);
}

}  // namespace

int scan_bwd_blocks(const ScanArgs& a, const ScanPlan& p, int sms) {
  return row_blocks((a.offsets != nullptr ? 1 : a.batch) * p.seg.n, lanes_of(a.width, bwd_shape(a).V, false), sms);
}
void scan_bwd_maps(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) { run(a, p, true, sms, st); }
void scan_bwd_rows(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) { run(a, p, false, sms, st); }

}  // namespace su
