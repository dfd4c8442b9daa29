// Gated linear recurrence, backward (formulas in scan_math.cuh): a thread walks its channels
// through one segment of one sequence, last step to first.
#include <type_traits>

#include "scan_shape.cuh"

namespace su {
namespace {

// Where a unit of work (one chunk of one segment) lies.
struct Unit {
  int64_t q, b, begin;  // segment, sequence, the segment's first step
  int steps, tc;        // of the segment; the chunk's first step inside it
};

// A chunk's x, r, i (or their codes and scales), dh and marks on their way to registers. In
// flight they are copies into slots of shared memory that belong to the thread, so the
// next chunk's loads are under way while this one is worked on and no barrier is needed.
template <class T, int V, int CH, bool CODES, bool MARKS>
struct Slots {
  using Raw = typename RawOf<sizeof(T) * V>::type;
  static constexpr int kRows = CODES ? 1 : 4;                      // of Raw: dh, and without codes x, r, i
  static constexpr int kWords = (CODES ? 6 : 0) + (MARKS ? 1 : 0);  // codes, scales, marks
  static constexpr int kBytes = 2 * CH * (kRows * static_cast<int>(sizeof(Raw)) + kWords * 4);  // of a thread
  Raw* rows;        // [2][CH][kRows][threads], at this thread's place
  uint32_t* words;  // [2][CH][kWords][threads]
  int ld;           // threads

  __device__ __forceinline__ void init(void* smem) {
    ld = blockDim.x;
    rows = static_cast<Raw*>(smem) + threadIdx.x;
    words = reinterpret_cast<uint32_t*>(static_cast<Raw*>(smem) + 2 * CH * kRows * ld) + threadIdx.x;
  }
  __device__ __forceinline__ Raw* row(int buf, int j, int w) const { return rows + ((buf * CH + j) * kRows + w) * ld; }
  __device__ __forceinline__ uint32_t* word(int buf, int j, int w) const {
    return words + ((buf * CH + j) * kWords + w) * ld;
  }
  __device__ __forceinline__ void fetch(const ScanArgs& A, const Unit& u, int c, int buf) const {
    const int64_t H = A.width, G = (A.width + kGroup8 - 1) / kGroup8;
    const int64_t t0 = u.begin + u.tc;
    const int64_t at = u.b * A.row_sb + t0 * A.row_st;
    const T* in = CODES ? nullptr : static_cast<const T*>(A.p) + u.b * A.p_sb + t0 * A.p_st + c;
    // the aligned word that holds this lane's codes (rows of codes are multiples of 4)
    const int8_t* code = CODES ? A.codes + at * 3 * H + (c & ~3) : nullptr;
    const float* scale = CODES ? A.scales + at * 3 * G + c / kGroup8 : nullptr;
    const T* dh = static_cast<const T*>(A.dh) + (A.dh != nullptr ? u.b * A.dh_sb + t0 * A.dh_st + c : 0);
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      if (u.tc + j < u.steps) {
        if constexpr (CODES) {
#pragma unroll
          for (int w = 0; w < 3; ++w) {
            copy_async<4>(word(buf, j, w), code + w * H);
            copy_async<4>(word(buf, j, 3 + w), scale + w * G);
          }
        } else {
#pragma unroll
          for (int w = 0; w < 3; ++w) copy_async<sizeof(Raw)>(row(buf, j, 1 + w), in + w * H);
        }
        if (A.dh != nullptr) copy_async<sizeof(Raw)>(row(buf, j, 0), dh);
        if constexpr (MARKS) copy_async<4>(word(buf, j, kWords - 1), A.marks + t0 + j);
      }
      if (CODES) {
        code += A.row_st * 3 * H;
        scale += A.row_st * 3 * G;
      } else {
        in += A.p_st;
      }
      dh += A.dh_st;
    }
  }
  __device__ __forceinline__ void get(int buf, int j, int w, int c, float (&f)[V]) const {
    if constexpr (CODES) {
      Codes<V> q;
      q.raw = static_cast<typename RawOf<V>::type>(*word(buf, j, w) >> (V == 4 ? 0 : 8 * (c & 3)));
      q.get(__uint_as_float(*word(buf, j, 3 + w)), f);
    } else {
      Pack<T, V> p;
      p.raw = *row(buf, j, 1 + w);
      p.get(f);
    }
  }
  __device__ __forceinline__ void get_dh(int buf, int j, float (&f)[V]) const {
    Pack<T, V> p;
    p.raw = *row(buf, j, 0);
    p.get(f);
  }
  __device__ __forceinline__ int mark(int buf, int j) const { return static_cast<int>(*word(buf, j, kWords - 1)); }
};

// The same values in registers, where a lane's are less than the 4 bytes that a copy has: single
// bf16 values, and single codes (whose 16 steps of words would take too much shared memory).
template <class T, int V, int CH, bool CODES>
struct Held {
  Pack<T, V> v[CODES ? 1 : CH][3], d[CH];
  Codes<V> q[CODES ? CH : 1][3];
  float scale[CODES ? CH : 1][3];

  __device__ __forceinline__ void fetch(const ScanArgs& A, const Unit& u, int c, unsigned on) {
    const int H = A.width, G = (H + kGroup8 - 1) / kGroup8;
    const int64_t t0 = u.begin + u.tc;
    const int64_t row = u.b * A.row_sb + t0 * A.row_st;
    const T* in = CODES ? nullptr : static_cast<const T*>(A.p) + u.b * A.p_sb + t0 * A.p_st + c;
    const int8_t* code = CODES ? A.codes + row * 3 * H + c : nullptr;
    const float* sc = CODES ? A.scales + row * 3 * G + c / kGroup8 : nullptr;
    const T* dh = static_cast<const T*>(A.dh) + (A.dh != nullptr ? u.b * A.dh_sb + t0 * A.dh_st + c : 0);
#pragma unroll
    for (int j = 0; j < CH; ++j) {
#pragma unroll
      for (int w = 0; w < 3; ++w) {
        if constexpr (CODES) {
          q[j][w].zero();
          scale[j][w] = 0.f;
          if (on >> j & 1) {
            q[j][w].load(code + w * static_cast<int64_t>(H));
            scale[j][w] = sc[w * static_cast<int64_t>(G)];
          }
        } else {
          v[j][w].zero();
          if (on >> j & 1) v[j][w].load(in + w * static_cast<int64_t>(H));
        }
      }
      d[j].zero();
      if (u.tc + j < u.steps && A.dh != nullptr) d[j].load(dh);
      if (CODES) {
        code += A.row_st * 3 * H;
        sc += A.row_st * 3 * G;
      } else {
        in += A.p_st;
      }
      dh += A.dh_st;
    }
  }
  __device__ __forceinline__ void get(int j, int w, float (&f)[V]) const {
    if constexpr (CODES)
      q[j][w].get(scale[j][w], f);
    else
      v[j][w].get(f);
  }
};

// Chunks of CH steps (those between kept states, or the whole of a short sequence). Every
// gradient of a step is g times a factor that the inputs and the state before the step give:
// the chunk is walked forwards from its first state for the factors, which stay in
// registers, and then backwards for g. The gates are evaluated once.
//
// Bound by the loads under way: three blocks of 128 threads fit an SM with their factors and
// slots (74 KB a block with packed fp32). 200,000 x 8 x 64 fp32 567 us, 5.1 TB/s; 2 x 65,537 x 256
// bf16 128 us, where the gates' special functions and issue bound it; 1,000,000 x 100 packed
// fp32 704 us, 4.1 TB/s, the marks' branches on top; 400,000 x 4 x 128 from 8-bit codes 802 us.
constexpr int kBwdThreads = 128;
template <class T, int V, int CH, bool CODES, int KIND>
__global__ void __launch_bounds__(kBwdThreads, 3) scan_bwd_kernel(const ScanArgs A, const ScanPlan P, const Lanes L) {
  constexpr bool kAsync = CODES ? V > 1 : sizeof(T) * V >= 4;
  extern __shared__ uint4 smem[];
  const int y = threadIdx.x / L.count;
  const int lane_c = threadIdx.x % L.count;
  const int c = (blockIdx.y * L.count + lane_c) * V;
  const bool live = c < A.width;
  const int H = A.width;
  const int64_t batch = KIND == kPacked ? 1 : A.batch;
  const int64_t rows = live ? batch * P.seg.n : 0;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * L.rows;
  Vf<V> k, dl, E;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    k[v] = live ? decay_factor(param_at(A.decay, A.decay_bf16, c + v), A.rate) : 0.f;
    dl[v] = E[v] = 0.f;
  }
  // units in the order of work: a row's chunks from the last to the first, then the next row;
  // false behind the last one. Rows without steps have one empty chunk.
  auto place = [&](int64_t rr, Unit& u) {
    if (rr >= rows) return false;
    const SegRow s = seg_row(rr, batch, P.seg, false);
    u.q = s.q;
    u.b = s.b;
    u.begin = s.q * P.seg.len;
    u.steps = static_cast<int>(min(P.seg.len, A.steps - u.begin));
    u.tc = u.steps > 0 ? (u.steps - 1) / CH * CH : 0;
    return true;
  };
  int64_t rr = static_cast<int64_t>(blockIdx.x) * L.rows + y;
  Unit u;
  bool more = place(rr, u);
  Slots<T, V, CH, CODES, KIND == kPacked> slots;
  if constexpr (kAsync) {
    slots.init(smem);
    if (more) slots.fetch(A, u, c, 0);
    commit_copies();
  }
  bool fresh = true;
  int buf = 0;
  while (more) {
    Unit next = u;
    bool more_next;
    if (u.tc > 0) {
      next.tc -= CH;
      more_next = true;
    } else {
      rr += stride;
      more_next = place(rr, next);
    }
    const int64_t t0 = u.begin + u.tc;
    const int64_t row = u.b * A.row_sb + t0 * A.row_st;
    const int64_t at = (u.q * batch + u.b) * H + c;
    if (fresh) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        E[v] = 0.f;
        if (P.seg.n > 1)
          E[v] = P.carry[at + v];
        else if (KIND != kPacked && A.dlast != nullptr)
          E[v] = A.dlast[u.b * H + c + v];
      }
    }
    Vf<V> h;
    const float* from = t0 > 0 ? A.states + (u.b * A.n_states + t0 / A.state_every - 1) * H + c
                               : (KIND != kPacked && A.h0 != nullptr ? A.h0 + u.b * H + c : nullptr);
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = from != nullptr ? from[v] : 0.f;
    if constexpr (kAsync) {
      if (more_next) slots.fetch(A, next, c, buf ^ 1);
      commit_copies();
      wait_copies<1>();
    }
    unsigned on = 0, firsts = 0, lasts = 0;
    if (KIND == kPlain) {
      const int n = u.steps - u.tc;
      on = n >= CH ? (1u << CH) - 1u : (1u << n) - 1u;
    } else {
      const uint8_t* valid = A.mask != nullptr ? A.mask + u.b * A.m_sb + t0 * A.m_st : nullptr;
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        if (u.tc + j >= u.steps) continue;
        if (valid == nullptr || valid[j * A.m_st] != 0) on |= 1u << j;
        if constexpr (KIND == kPacked) {
          int mk;
          if constexpr (kAsync)
            mk = slots.mark(buf, j);
          else
            mk = A.marks[t0 + j];
          if (mk >= 0) {
            firsts |= static_cast<unsigned>(mk & kMarkFirst) << j;
            lasts |= static_cast<unsigned>((mk & kMarkLast) >> 1) << j;
          }
        }
      }
    }
    Held<T, V, CH, CODES> held;
    if constexpr (!kAsync) held.fetch(A, u, c, on);
    // WHOLE: every step of the chunk is inside the sequence and counts
    auto work = [&](auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
      Slope<V> f[CH];
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        if (KIND == kPacked && (firsts >> j & 1)) {
          const int64_t q = A.marks[t0 + j] >> 2;
#pragma unroll
          for (int v = 0; v < V; ++v) h[v] = A.h0 != nullptr ? A.h0[q * H + c + v] : 0.f;
        }
        Vf<V> fx, fr, fi;
        if constexpr (kAsync) {
          slots.get(buf, j, 0, c, fx.v);
          slots.get(buf, j, 1, c, fr.v);
          slots.get(buf, j, 2, c, fi.v);
        } else {
          held.get(j, 0, fx.v);
          held.get(j, 1, fr.v);
          held.get(j, 2, fi.v);
        }
        if (!WHOLE && !(on >> j & 1)) shut(fx, fr, fi);
        f[j] = slope_of(gate_of(fx, fr, fi, k), h);
      }
      T* out = static_cast<T*>(A.dp) + (row + CH * A.row_st) * 3 * H + c;
#pragma unroll
      for (int j = CH - 1; j >= 0; --j) {
        out -= A.row_st * 3 * H;
        if (!WHOLE && u.tc + j >= u.steps) continue;
        if (KIND == kPacked && (lasts >> j & 1)) {
          const int64_t q = A.marks[t0 + j] >> 2;
#pragma unroll
          for (int v = 0; v < V; ++v) E[v] = A.dlast != nullptr ? A.dlast[q * H + c + v] : 0.f;
        }
        Vf<V> dy;
        if constexpr (kAsync) {
          slots.get_dh(buf, j, dy.v);
          if (A.dh == nullptr) {
#pragma unroll
            for (int v = 0; v < V; ++v) dy[v] = 0.f;
          }
        } else {
          held.d[j].get(dy.v);
        }
        const Vf<V> g = dy + E;
        Vf<V> dx = g * f[j].x, dr = g * f[j].r, di = g * f[j].i;
        if (WHOLE || (on >> j & 1)) {
          dl = fma(g, f[j].l, dl);
          E = g * f[j].a;
        } else {  // the factors are 0 times the state, and g need not be finite either
          dx = dr = di = splat<V>(0.f);
          E = g;
        }
        Pack<T, V> o;
        o.set(dx.v);
        o.store(out);
        o.set(dr.v);
        o.store(out + H);
        o.set(di.v);
        o.store(out + 2 * H);
        if (KIND == kPacked && (firsts >> j & 1) && A.dh0 != nullptr) {
          const int64_t q = A.marks[t0 + j] >> 2;
#pragma unroll
          for (int v = 0; v < V; ++v) A.dh0[q * H + c + v] = E[v];
        }
      }
    };
    if (on == (1u << CH) - 1u)
      work(std::true_type{});
    else
      work(std::false_type{});
    fresh = u.tc == 0;
    if (KIND != kPacked && fresh && u.q == 0 && A.dh0 != nullptr) {
#pragma unroll
      for (int v = 0; v < V; ++v) A.dh0[u.b * H + c + v] = E[v];
    }
    u = next;
    more = more_next;
    buf ^= 1;
  }
  // the block's share of -sum dz sigmoid(r), added up over its rows in order
  __shared__ float sum[kBwdThreads * V];
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
  Vf<V> k;
#pragma unroll
  for (int v = 0; v < V; ++v) k[v] = decay_factor(param_at(A.decay, A.decay_bf16, c + v), A.rate);
  for (int64_t rr = static_cast<int64_t>(blockIdx.x) * L.rows + y; rr < rows;
       rr += static_cast<int64_t>(gridDim.x) * L.rows) {
    // the first segments last: the pass that follows begins with them
    const SegRow s = seg_row(rr, batch, P.seg, true);
    const int64_t begin = s.q * P.seg.len;
    int steps = static_cast<int>(min(P.seg.len, A.steps - begin));
    if (KIND == kPacked) steps = min(steps, static_cast<int>(P.seg.len) - max(0, P.reach[s.q]));
    Vf<V> m, E;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      m[v] = 1.f;
      E[v] = 0.f;
    }
    int tc = (steps + U - 1) / U * U;
    const int64_t end = s.b * A.row_sb + (begin + tc) * A.row_st;
    const T* in = CODES ? nullptr : static_cast<const T*>(A.p) + s.b * A.p_sb + (begin + tc) * A.p_st + H + c;
    const int8_t* code = CODES ? A.codes + end * 3 * H + H + c : nullptr;
    const float* sc = CODES ? A.scales + end * 3 * G + G + c / kGroup8 : nullptr;
    const T* dh = static_cast<const T*>(A.dh) + (A.dh != nullptr ? s.b * A.dh_sb + (begin + tc) * A.dh_st + c : 0);
    const uint8_t* valid = A.mask != nullptr ? A.mask + s.b * A.m_sb + (begin + tc) * A.m_st : nullptr;
    while (tc > 0) {
      tc -= U;
      Pack<T, V> r[U], d[U];
      Codes<V> q[U];
      float scale[U];
      bool on[U];
      int mk[U];
#pragma unroll
      for (int j = U - 1; j >= 0; --j) {
        const bool inside = tc + j < steps;
        on[j] = inside;
        if (KIND == kMasked || (KIND == kPacked && A.mask != nullptr)) {
          valid -= A.m_st;
          if (inside) on[j] = *valid != 0;
        }
        mk[j] = -1;
        if (KIND == kPacked) {
          if (inside) mk[j] = A.marks[begin + tc + j];
        }
        r[j].zero();
        q[j].zero();
        scale[j] = 0.f;
        if constexpr (CODES) {
          code -= A.row_st * 3 * H;
          sc -= A.row_st * 3 * G;
          if (on[j]) {
            q[j].load(code);
            scale[j] = *sc;
          }
        } else {
          in -= A.p_st;
          if (on[j]) r[j].load_keep(in);
        }
        d[j].zero();
        dh -= A.dh_st;
        if (inside && A.dh != nullptr) d[j].load_keep(dh);
      }
#pragma unroll
      for (int j = U - 1; j >= 0; --j) {
        if (KIND == kPacked && mk[j] >= 0 && (mk[j] & kMarkLast)) {
          const float* from = A.dlast != nullptr ? A.dlast + static_cast<int64_t>(mk[j] >> 2) * H + c : nullptr;
#pragma unroll
          for (int v = 0; v < V; ++v) E[v] = from != nullptr ? from[v] : 0.f;
        }
        Vf<V> fr, fd;
        d[j].get(fd.v);
        if constexpr (CODES)
          q[j].get(scale[j], fr.v);
        else
          r[j].get(fr.v);
        if (!on[j]) fr = splat<V>(-1e30f);  // a = 1; dh is 0 beyond the last step
        const Vf<V> a = decay_of(fr, k);
        E = a * (E + fd);
        m = m * a;
      }
    }
    const bool anew = KIND == kPacked && P.reach[s.q] >= 0;
#pragma unroll
    for (int v = 0; v < V; ++v) P.maps[(s.q * batch + s.b) * H + c + v] = make_float2(anew ? kAnew : m[v], E[v]);
  }
}

struct BwdShape {
  int V, CH;
};
// 16 steps' factors of one channel fit the registers, so do 8 of two and 4 of four
BwdShape bwd_shape(const ScanArgs& a) {
  const int vec = a.codes != nullptr && a.vec != 4 ? 1 : a.vec;  // codes go by words of four
  if (a.offsets == nullptr && a.steps <= 4 && vec != 2) return {vec, 4};
  if (a.state_every == kStateShort || (a.offsets == nullptr && a.steps <= 8)) return {vec > 1 ? 2 : 1, 8};
  return {1, kStateEvery};
}
Lanes bwd_lanes(const ScanArgs& a) { return lanes_of(a.width, bwd_shape(a).V, false, kBwdThreads); }

template <class T, int V, int CH, bool CODES, int KIND>
void run(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) {
  const Lanes l = bwd_lanes(a);
  const dim3 grid(scan_bwd_blocks(a, p, sms), l.blocks);
  const int threads = l.count * l.rows;
  const bool async = CODES ? V > 1 : sizeof(T) * V >= 4;
  const size_t smem = async ? static_cast<size_t>(threads) * Slots<T, V, CH, CODES, KIND == kPacked>::kBytes : 0;
  auto kernel = scan_bwd_kernel<T, V, CH, CODES, KIND>;
  static uint64_t allowed = 0;
  allow_smem(kernel, smem, allowed);
  kernel<<<grid, threads, smem, st>>>(a, p, l);
}

template <class T, bool CODES, int KIND>
void run(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) {
  const BwdShape b = bwd_shape(a);
  if (b.CH == 4) {
    if constexpr (KIND != kPacked)
      b.V == 4 ? run<T, 4, 4, CODES, KIND>(a, p, sms, st) : run<T, 1, 4, CODES, KIND>(a, p, sms, st);
  } else if (b.CH == 8) {
    if constexpr (KIND != kPacked || !CODES)
      b.V == 2 ? run<T, 2, 8, CODES, KIND>(a, p, sms, st) : run<T, 1, 8, CODES, KIND>(a, p, sms, st);
  } else {
    if constexpr (CODES) run<T, 1, kStateEvery, CODES, KIND>(a, p, sms, st);
  }
}

template <class T, bool CODES, int KIND>
void run_maps(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) {
  const Lanes l = lanes_of(a.width, a.codes != nullptr && a.vec != 4 ? 1 : a.vec, false, 256);
  const int64_t rows = (a.offsets != nullptr ? 1 : a.batch) * p.seg.n;
  const dim3 grid(row_blocks(rows, l, sms), l.blocks);
  const int threads = l.count * l.rows;
  if (a.vec == 4) {
    scan_bwd_maps_kernel<T, 4, 4, CODES, KIND><<<grid, threads, 0, st>>>(a, p, l);
    return;
  }
  if constexpr (!CODES) {
    if (a.vec == 2) {
      scan_bwd_maps_kernel<T, 2, 8, CODES, KIND><<<grid, threads, 0, st>>>(a, p, l);
      return;
    }
  }
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
  return row_blocks((a.offsets != nullptr ? 1 : a.batch) * p.seg.n, bwd_lanes(a), sms);
}
void scan_bwd_maps(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) { run(a, p, true, sms, st); }
void scan_bwd_rows(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) { run(a, p, false, sms, st); }

}  // namespace su
