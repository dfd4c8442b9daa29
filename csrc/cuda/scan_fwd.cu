// Gated linear recurrence, forward (formulas in scan_math.cuh): a thread walks its channels
// through one segment of one sequence.
#include "scan_shape.cuh"

namespace su {
namespace {

template <class T, int V>
struct Inputs {
  Pack<T, V> x, r, i;
  __device__ __forceinline__ void zero() {
    x.zero();
    r.zero();
    i.zero();
  }
  template <bool KEEP>
  __device__ __forceinline__ void load(const T* p, int H) {
    if (KEEP) {
      x.load_keep(p);
      r.load_keep(p + H);
      i.load_keep(p + 2 * H);
    } else {
      x.load(p);
      r.load(p + H);
      i.load(p + 2 * H);
    }
  }
};

// MAPS: composes the segment's steps into h -> A h + B and writes nothing else. Otherwise
// walks the states from the one before the segment.
// Steps are taken U at a time: their inputs are loaded together, U x 3 loads of V values
// under way per thread.
template <class T, int V, int U, bool MAPS, bool CODES, int KIND>
__global__ void __launch_bounds__(256, 3) scan_fwd_kernel(const ScanArgs A, const ScanPlan P, const Lanes L) {
  const int y = threadIdx.x / L.count;
  const int c = (blockIdx.y * L.count + threadIdx.x % L.count) * V;
  const bool live = c < A.width;
  if (!CODES && !live) return;
  const int H = A.width;
  const int G = (H + kGroup8 - 1) / kGroup8;
  const int64_t batch = KIND == kPacked ? 1 : A.batch;
  const int64_t rows = batch * P.seg.n;
  float k[V];
#pragma unroll
  for (int v = 0; v < V; ++v) k[v] = live ? decay_factor(param_at(A.decay, A.decay_bf16, c + v), A.rate) : 0.f;
  for (int64_t rr = static_cast<int64_t>(blockIdx.x) * L.rows + y; rr < rows;
       rr += static_cast<int64_t>(gridDim.x) * L.rows) {
    // after the maps were made first to last, the last segments are the ones still in L2
    const SegRow s = seg_row(rr, batch, P.seg, !MAPS && P.seg.n > 1);
    const int64_t begin = s.q * P.seg.len;
    const int steps = static_cast<int>(min(P.seg.len, A.steps - begin));
    const int64_t row = s.b * A.row_sb + begin * A.row_st;
    const int64_t at = (s.q * batch + s.b) * H + c;
    const T* in = static_cast<const T*>(A.p) + s.b * A.p_sb + begin * A.p_st + c;
    const uint8_t* valid = A.mask != nullptr ? A.mask + s.b * A.m_sb + begin * A.m_st : nullptr;
    const int* mark = KIND == kPacked ? A.marks + begin : nullptr;
    T* out = MAPS ? nullptr : static_cast<T*>(A.h) + row * H + c;
    int8_t* code = CODES ? A.codes + row * 3 * H + c : nullptr;
    float* scale = CODES ? A.scales + row * 3 * G + c / kGroup8 : nullptr;
    float h[V], m[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      m[v] = 1.f;
      h[v] = 0.f;
      if (!MAPS && live) {
        if (P.seg.n > 1)
          h[v] = P.carry[at + v];
        else if (KIND != kPacked && A.h0 != nullptr)
          h[v] = A.h0[s.b * H + c + v];
      }
    }
    for (int t0 = 0; t0 < steps; t0 += U) {
      Inputs<T, V> w[U];
      int mk[U];
      bool on[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const bool inside = t0 + j < steps;
        on[j] = inside && live;
        if (KIND == kMasked || (KIND == kPacked && valid != nullptr)) {
          if (inside) on[j] = on[j] && *valid != 0;
          valid += A.m_st;
        }
        mk[j] = -1;
        if (KIND == kPacked) {
          if (inside) mk[j] = mark[j];
        }
        w[j].zero();
        if (on[j]) w[j].template load<MAPS>(in, H);
        in += A.p_st;
      }
      if (KIND == kPacked) mark += U;
      if (!MAPS && A.states != nullptr && live && begin + t0 > 0 && t0 % A.state_every == 0) {  // U divides it
        float* to = A.states + (s.b * A.n_states + (begin + t0) / A.state_every - 1) * H + c;
#pragma unroll
        for (int v = 0; v < V; ++v) to[v] = h[v];
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (t0 + j >= steps) break;
        float fx[V], fr[V], fi[V];
        w[j].x.get(fx);
        w[j].r.get(fr);
        w[j].i.get(fi);
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
        if (KIND == kPacked && mk[j] >= 0 && (mk[j] & kMarkFirst) && live) {
          const float* from = A.h0 != nullptr ? A.h0 + static_cast<int64_t>(mk[j] >> 2) * H + c : nullptr;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            h[v] = from != nullptr ? from[v] : 0.f;
            m[v] = 0.f;
          }
        }
        if (KIND != kPlain && !on[j]) {
#pragma unroll
          for (int v = 0; v < V; ++v) shut(fx[v], fr[v], fi[v]);
        }
        Step g[V];
        steps_of(fx, fr, fi, k, g);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          h[v] = fmaf(g[v].a, h[v], g[v].add);
          if (MAPS) m[v] *= g[v].a;
        }
        if (!MAPS) {
          if (live) {
            Pack<T, V> o;
            o.set(h);
            o.store(out);
          }
          out += A.row_st * H;
          if (KIND == kPacked && mk[j] >= 0 && (mk[j] & kMarkLast) && live) {
            float* to = A.last + static_cast<int64_t>(mk[j] >> 2) * H + c;
#pragma unroll
            for (int v = 0; v < V; ++v) to[v] = h[v];
          }
        }
      }
    }
    if (!live) continue;
    if (MAPS) {
#pragma unroll
      for (int v = 0; v < V; ++v) P.maps[at + v] = make_float2(m[v], h[v]);
    } else if (KIND != kPacked && s.q == P.seg.n - 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) A.last[s.b * H + c + v] = h[v];
    }
  }
}

template <class T, bool MAPS, bool CODES, int KIND>
void run(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) {
  const Lanes l = lanes_of(a.width, a.vec ? 4 : 1, CODES, 256);
  const int64_t rows = (a.offsets != nullptr ? 1 : a.batch) * p.seg.n;
  const dim3 grid(row_blocks(rows, l, sms), l.blocks);
  const int threads = l.count * l.rows;
  if (a.vec)
    scan_fwd_kernel<T, 4, 4, MAPS, CODES, KIND><<<grid, threads, 0, st>>>(a, p, l);
  else
    scan_fwd_kernel<T, 1, 8, MAPS, CODES, KIND><<<grid, threads, 0, st>>>(a, p, l);
}

template <class T, bool MAPS, bool CODES>
void run(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) {
  count_launch();
  switch (kind_of(a)) {
    case kPlain:
      return run<T, MAPS, CODES, kPlain>(a, p, sms, st);
    case kMasked:
      return run<T, MAPS, CODES, kMasked>(a, p, sms, st);
    default:
      return run<T, MAPS, CODES, kPacked>(a, p, sms, st);
  }
}

}  // namespace

void scan_fwd_maps(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) {
  a.bf16 ? run<__nv_bfloat16, true, false>(a, p, sms, st) : run<float, true, false>(a, p, sms, st);
}

void scan_fwd_rows(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) {
  if (a.codes != nullptr)
    a.bf16 ? run<__nv_bfloat16, false, true>(a, p, sms, st) : run<float, false, true>(a, p, sms, st);
  else
    a.bf16 ? run<__nv_bfloat16, false, false>(a, p, sms, st) : run<float, false, false>(a, p, sms, st);
}

}  // namespace su
