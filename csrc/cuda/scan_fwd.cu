// Gated linear recurrence, forward (formulas in scan_math.cuh): a thread walks its channels
// through one segment of one sequence.
#include "scan_shape.cuh"

namespace su {
namespace {

// 8-bit codes to write: none, or with rows of at least one group of 32 or narrower ones
enum { kNoCodes = 0, kWide = 1, kNarrow = 2 };

// U steps of one segment: a unit of work.
struct Unit {
  int64_t q, b, begin;  // segment, sequence, the segment's first step
  int steps, t;         // of the segment; the unit's first step inside it
};

// MAPS: composes the segment's steps into h -> A h + B and writes nothing else. Otherwise
// walks the states from the one before the segment.
//
// ASYNC, threads of four channels: while a unit is worked on the inputs of the next one (of the
// next segment behind the last) are copied into slots of shared memory that belong to the
// thread, so loads are always under way, no barrier is needed and the registers hold one step's
// inputs. Otherwise the unit's inputs are loaded together into registers: threads of fewer
// channels, and bf16 with marks or a mask, where the copies' instructions cost more than they
// hide. Copies against registers: 200,000 x 8 x 64 bf16 166 and 180 us, 200,000 x 4 x 128 bf16
// to 8-bit codes 370 and 451; packed 404,952 x 100 bf16 113 and 103, masked 68 x 9,528 x 30
// fp32 (two channels) 68 and 63.
//
// Bound by bytes at fp32: 200,000 x 8 x 64 takes 262 us, 6.3 TB/s. With codes the encoding's
// instructions bound it (400,000 x 4 x 128 fp32: 693 us), in bf16 the gates' as well.
template <class T, int V, int KIND>
constexpr bool kAsyncOf = V == 4 && (sizeof(T) == 4 || KIND == kPlain);

template <class T, int V, int U, bool MAPS, int CODES, int KIND>
__global__ void __launch_bounds__(256, !CODES && kAsyncOf<T, V, KIND> ? 4 : 3)
    scan_fwd_kernel(const ScanArgs A, const ScanPlan P, const Lanes L) {
  constexpr bool kAsync = kAsyncOf<T, V, KIND>;
  using Raw = typename Pack<T, V>::Raw;
  extern __shared__ uint4 smem[];
  const int y = threadIdx.x / L.count;
  const int c = (blockIdx.y * L.count + threadIdx.x % L.count) * V;
  const bool live = c < A.width;
  if (!CODES && !live) return;
  const int H = A.width;
  const int G = (H + kGroup8 - 1) / kGroup8;
  const int64_t batch = KIND == kPacked ? 1 : A.batch;
  const int64_t rows = batch * P.seg.n;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * L.rows;
  const int group = CODES ? group_lanes(H, V) : 1;
  const bool masked = KIND == kMasked || (KIND == kPacked && A.mask != nullptr);
  Vf<V> k, h, m;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    k[v] = live ? decay_factor(param_at(A.decay, A.decay_bf16, c + v), A.rate) : 0.f;
    h[v] = m[v] = 0.f;
  }
  auto place = [&](int64_t rr, Unit& u) {
    if (rr >= rows) return false;
    // after the maps were made first to last, the last segments are the ones still in L2
    const SegRow s = seg_row(rr, batch, P.seg, !MAPS && P.seg.n > 1);
    u.q = s.q;
    u.b = s.b;
    u.begin = s.q * P.seg.len;
    u.steps = static_cast<int>(min(P.seg.len, A.steps - u.begin));
    u.t = 0;
    if (MAPS && KIND == kPacked) u.t = max(0, P.reach[u.q]);  // that step's mark starts h
    return true;
  };
  Raw* const slots = reinterpret_cast<Raw*>(smem) + threadIdx.x;
  const int ld = blockDim.x;
  auto slot = [&](int buf, int j, int w) { return slots + ((buf * U + j) * 3 + w) * ld; };
  auto input = [&](const Unit& u, int j) {
    return static_cast<const T*>(A.p) + u.b * A.p_sb + (u.begin + u.t + j) * A.p_st + c;
  };
  auto fetch = [&](const Unit& u, int buf) {
    if constexpr (kAsync) {
      const T* in = input(u, 0);
#pragma unroll
      for (int j = 0; j < U; ++j, in += A.p_st) {
        if (u.t + j < u.steps && live) {
          copy_async<sizeof(Raw)>(slot(buf, j, 0), in);
          copy_async<sizeof(Raw)>(slot(buf, j, 1), in + H);
          copy_async<sizeof(Raw)>(slot(buf, j, 2), in + 2 * static_cast<int64_t>(H));
        }
      }
    }
  };
  // marks and mask of a unit, a unit ahead of their use
  auto peek = [&](const Unit& u, int (&mk)[U], bool (&on)[U]) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const bool inside = u.t + j < u.steps;
      mk[j] = -1;
      on[j] = inside;
      if (KIND == kPacked && inside) mk[j] = A.marks[u.begin + u.t + j];
      if (masked && inside) on[j] = A.mask[u.b * A.m_sb + (u.begin + u.t + j) * A.m_st] != 0;
    }
  };
  int64_t rr = static_cast<int64_t>(blockIdx.x) * L.rows + y;
  Unit u;
  bool more = place(rr, u);
  int mk[U];
  bool on[U];
  if (more) {
    fetch(u, 0);
    peek(u, mk, on);
  }
  commit_copies();
  T* out = nullptr;
  int8_t* code = nullptr;
  float* scale = nullptr;
  int buf = 0;
  while (more) {
    Unit next = u;
    bool more_next = true;
    if (u.t + U < u.steps) {
      next.t += U;
    } else {
      rr += stride;
      more_next = place(rr, next);
    }
    int mk_next[U];
    bool on_next[U];
    if (more_next) {
      fetch(next, buf ^ 1);
      peek(next, mk_next, on_next);
    }
    commit_copies();
    const int64_t at = (u.q * batch + u.b) * H + c;
    if (u.t == 0) {
      const int64_t row = u.b * A.row_sb + u.begin * A.row_st;
      out = MAPS ? nullptr : static_cast<T*>(A.h) + row * H + c;
      if (CODES) {
        code = A.codes + row * 3 * H + c;
        scale = A.scales + row * 3 * G + c / kGroup8;
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        m[v] = 1.f;
        h[v] = 0.f;
        if (!MAPS && live) {
          if (P.seg.n > 1)
            h[v] = P.carry[at + v];
          else if (KIND != kPacked && A.h0 != nullptr)
            h[v] = A.h0[u.b * H + c + v];
        }
      }
    }
    if (!MAPS && A.states != nullptr && live && u.begin + u.t > 0 && u.t % A.state_every == 0 && u.steps > 0) {
      // U divides state_every
      float* to = A.states + (u.b * A.n_states + (u.begin + u.t) / A.state_every - 1) * H + c;
#pragma unroll
      for (int v = 0; v < V; ++v) to[v] = h[v];
    }
    if constexpr (kAsync) wait_copies<1>();
    Pack<T, V> w[kAsync ? 1 : U][3];
    if constexpr (!kAsync) {
      const T* in = input(u, 0);
#pragma unroll
      for (int j = 0; j < U; ++j, in += A.p_st)
#pragma unroll
        for (int s = 0; s < 3; ++s) {
          w[j][s].zero();
          if (on[j] && live) {
            if (MAPS)
              w[j][s].load_keep(in + s * static_cast<int64_t>(H));
            else
              w[j][s].load(in + s * static_cast<int64_t>(H));
          }
        }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (u.t + j >= u.steps) break;
      constexpr int kAt = kAsync ? 0 : 1;
      if constexpr (kAsync) {
#pragma unroll
        for (int s = 0; s < 3; ++s) {
          w[0][s].zero();
          if (live && (KIND == kPlain || on[j])) w[0][s].raw = *slot(buf, j, s);
        }
      }
      Vf<V> fx, fr, fi;
      w[kAt * j][0].get(fx.v);
      w[kAt * j][1].get(fr.v);
      w[kAt * j][2].get(fi.v);
      if constexpr (CODES) {
        Codes<V> q[3];
        const float s0 = encode8<CODES == kNarrow>(fx.v, q[0], group), s1 = encode8<CODES == kNarrow>(fr.v, q[1], group),
                    s2 = encode8<CODES == kNarrow>(fi.v, q[2], group);
        if (live) {
          q[0].store(code);
          q[1].store(code + H);
          q[2].store(code + 2 * static_cast<int64_t>(H));
          if (c % kGroup8 == 0) {
            scale[0] = s0;
            scale[G] = s1;
            scale[2 * static_cast<int64_t>(G)] = s2;
          }
        }
        code += A.row_st * 3 * H;
        scale += A.row_st * 3 * G;
      }
      if (KIND == kPacked && mk[j] >= 0 && (mk[j] & kMarkFirst) && live) {
        const float* from = A.h0 != nullptr ? A.h0 + static_cast<int64_t>(mk[j] >> 2) * H + c : nullptr;
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = from != nullptr ? from[v] : 0.f;
      }
      if (KIND != kPlain && !on[j]) shut(fx, fr, fi);
      const Step<V> g = step_of(fx, fr, fi, k);
      h = fma(g.a, h, g.add);
      if (MAPS) m = m * g.a;
      if (!MAPS) {
        if (live) {
          Pack<T, V> o;
          o.set(h.v);
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
    if (u.t + U >= u.steps && live) {
      if (MAPS) {
        const bool anew = KIND == kPacked && P.reach[u.q] >= 0;
#pragma unroll
        for (int v = 0; v < V; ++v) P.maps[at + v] = make_float2(anew ? kAnew : m[v], h[v]);
      } else if (KIND != kPacked && u.q == P.seg.n - 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) A.last[u.b * H + c + v] = h[v];
      }
    }
    u = next;
    more = more_next;
    buf ^= 1;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      mk[j] = mk_next[j];
      on[j] = on_next[j];
    }
  }
}

template <class T, int V, int U, bool MAPS, int CODES, int KIND>
void run(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) {
  const Lanes l = lanes_of(a.width, V, CODES, 256);
  const int64_t rows = (a.offsets != nullptr ? 1 : a.batch) * p.seg.n;
  const dim3 grid(row_blocks(rows, l, sms), l.blocks);
  const int threads = l.count * l.rows;
  const size_t smem = kAsyncOf<T, V, KIND> ? static_cast<size_t>(threads) * 2 * U * 3 * sizeof(T) * V : 0;
  auto kernel = scan_fwd_kernel<T, V, U, MAPS, CODES, KIND>;
  static uint64_t allowed = 0;
  allow_smem(kernel, smem, allowed);
  kernel<<<grid, threads, smem, st>>>(a, p, l);
}

// four channels: 192 bytes of slots a thread, four blocks an SM
template <class T, bool MAPS, int CODES, int KIND>
void run(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) {
  if (a.vec == 2) return run<T, 2, 4, MAPS, CODES, KIND>(a, p, sms, st);
  a.vec == 4 ? run<T, 4, 8 / static_cast<int>(sizeof(T)), MAPS, CODES, KIND>(a, p, sms, st) : run<T, 1, 8, MAPS, CODES, KIND>(a, p, sms, st);
}

template <class T, bool MAPS, int CODES>
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
  a.bf16 ? run<__nv_bfloat16, true, kNoCodes>(a, p, sms, st) : run<float, true, kNoCodes>(a, p, sms, st);
}

void scan_fwd_rows(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st) {
  if (a.codes == nullptr)
    a.bf16 ? run<__nv_bfloat16, false, kNoCodes>(a, p, sms, st) : run<float, false, kNoCodes>(a, p, sms, st);
  else if (a.width >= kGroup8)
    a.bf16 ? run<__nv_bfloat16, false, kWide>(a, p, sms, st) : run<float, false, kWide>(a, p, sms, st);
  else
    a.bf16 ? run<__nv_bfloat16, false, kNarrow>(a, p, sms, st) : run<float, false, kNarrow>(a, p, sms, st);
}

}  // namespace su
