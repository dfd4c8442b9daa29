// The gated recurrence's launches: segments, the states between them, packed sequences'
// marks, the decay's gradient, and the form for one new token per row.
//
// Where the sequences and channels alone leave the SMs short of threads, the steps are cut
// into segments that threads walk side by side. A run of steps maps the state before it to
// A h + B, and two runs compose to (A2 A1, A2 B1 + B2): one pass over the inputs makes the
// segments' maps, a short kernel walks the states through them, and the second pass starts
// every segment from its state. The inputs are read twice (backwards only r and dh are),
// which costs 7/4 of the bytes forward and 9/7 backward (packed sequences less: the maps need
// not go behind a sequence's start); nothing waits for another block.
// Handing the states on inside one pass instead (each tile publishing its map and gathering
// those before it) reads once. Tried in tiles of 8 and 16 steps a thread, no larger ones, it was
// slower at every size: 10 to 17 us a tile went by in the exchange, 1.44 against 0.83 ms forward for 1,000,000 packed rows of 100 fp32 with the
// same arithmetic in both (0.56 ms now).
// Every sum and composition has a fixed order: results are the same every run.
#include "scan_shape.cuh"

namespace su {
namespace {

// A warp per packed sequence: marks its first and last rows (marks != nullptr, -1 before), reports
// offsets that do not rise from 0 to `rows`, and copies what an empty sequence returns, its
// first state or the gradient of its last (`from`, nullptr: zeros). reach (see ScanPlan, -1
// before): maxima of integers, in whatever order they come.
__global__ void __launch_bounds__(256) scan_sequences_kernel(const int64_t* __restrict__ offsets, int64_t batch,
                                                             int64_t rows, int H, int* marks,
                                                             const float* __restrict__ from, float* __restrict__ to,
                                                             int* reach, int64_t len, bool bwd, int* status) {
  const int lane = threadIdx.x & 31;
  for (int64_t s = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32; s < batch;
       s += static_cast<int64_t>(gridDim.x) * 8) {
    const int64_t lo = offsets[s], hi = offsets[s + 1];
    if (lo < 0 || hi < lo || hi > rows || (s == 0 && lo != 0) || (s == batch - 1 && hi != rows)) {
      if (lane == 0) record_status(status, kBadIndex);
      continue;
    }
    if (hi == lo) {
      if (to != nullptr)
        for (int c = lane; c < H; c += 32) to[s * H + c] = from != nullptr ? from[s * H + c] : 0.f;
    } else if (lane == 0) {
      if (reach != nullptr) {
        const int64_t at = bwd ? hi - 1 : lo, q = at / len;
        atomicMax(reach + q, static_cast<int>(bwd ? len - 1 - (at - q * len) : at - q * len));
      }
      if (marks == nullptr) continue;
      const int id = static_cast<int>(s) * 4;
      if (hi - lo == 1) {
        marks[lo] = id + kMarkFirst + kMarkLast;
      } else {
        marks[lo] = id + kMarkFirst;
        marks[hi - 1] = id + kMarkLast;
      }
    }
  }
}

void launch_sequences(const ScanArgs& a, const ScanPlan& p, bool bwd, cudaStream_t st) {
  int* const marks = bwd ? nullptr : a.marks;
  float* const to = bwd ? a.dh0 : a.last;
  int* const reach = p.seg.n > 1 ? p.reach : nullptr;
  if (marks != nullptr && a.steps > 0) cudaMemsetAsync(marks, 0xff, static_cast<size_t>(a.steps) * sizeof(int), st);
  if (reach != nullptr) cudaMemsetAsync(reach, 0xff, static_cast<size_t>(p.seg.n) * sizeof(int), st);
  if (marks == nullptr && to == nullptr && reach == nullptr) return;
  count_launch();
  const int64_t blocks = (a.batch + 7) / 8;
  scan_sequences_kernel<<<static_cast<unsigned>(blocks < 8192 ? blocks : 8192), 256, 0, st>>>(
      a.offsets, a.batch, a.steps, a.width, marks, bwd ? a.dlast : a.h0, to, reach, p.seg.len, bwd, a.status);
}

// carry[q] = the state before segment q (backwards: the gradient after it), from `start` through
// the maps of the segments before it (after it). A block has 8 channels of one sequence (64
// bytes of maps, two sectors); each of its rows of threads (a quarter of the segments' number, up
// to 128) composes a share of the segments, the shares meet in order, and the row walks its
// share again from the state it gets.
constexpr int kShares = 128, kShareCols = 8;
__global__ void __launch_bounds__(kShareCols * kShares) scan_carry_kernel(const float2* __restrict__ maps, const float* start,
                                                                  int64_t n, int64_t batch, int H, bool bwd,
                                                                  float* __restrict__ carry) {
  __shared__ float2 part[kShares][kShareCols];
  const int c = blockIdx.y * kShareCols + threadIdx.x;
  const int64_t b = blockIdx.x;
  const bool live = c < H;
  const int64_t share = (n + blockDim.y - 1) / blockDim.y;
  const int64_t lo = min(n, threadIdx.y * share), hi = min(n, lo + share);
  const int64_t step = (bwd ? -1 : 1) * batch * H;
  const int64_t at = ((bwd ? n - 1 - lo : lo) * batch + b) * H + c;
  float2 all = make_float2(1.f, 0.f);
  if (live) {
    const float2* m = maps + at;
#pragma unroll 8
    for (int64_t q = lo; q < hi; ++q, m += step) all = compose(all, *m);
  }
  part[threadIdx.y][threadIdx.x] = all;
  __syncthreads();
  if (!live) return;
  float h = start != nullptr ? start[b * H + c] : 0.f;
#pragma unroll 8
  for (int k = 0; k < static_cast<int>(threadIdx.y); ++k) h = through(part[k][threadIdx.x], h);
  const float2* m = maps + at;
  float* to = carry + at;
#pragma unroll 8
  for (int64_t q = lo; q < hi; ++q, m += step, to += step) {
    *to = h;
    h = through(*m, h);
  }
}

void launch_carry(const ScanArgs& a, const ScanPlan& p, bool bwd, cudaStream_t st) {
  const int64_t batch = a.offsets != nullptr ? 1 : a.batch;
  const float* start = a.offsets != nullptr ? nullptr : (bwd ? a.dlast : a.h0);
  int shares = 4;
  while (shares < kShares && shares * 4 < p.seg.n) shares *= 2;
  count_launch();
  scan_carry_kernel<<<dim3(static_cast<unsigned>(batch), (a.width + kShareCols - 1) / kShareCols),
                      dim3(kShareCols, shares), 0, st>>>(p.maps, start, p.seg.n, batch, a.width, bwd, p.carry);
}

// Rows k, k + m, k + 2m, ... of partial [n, H] added up in order into row k of out [m, H]:
// 32 channels x 32 shares per block. `last`: out is ddecay, c sigmoid(decay) times the
// sum (of -dz sigmoid(r)).
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
      param_store(out, decay_bf16, c, rate * sigmoid_f(param_at(decay, decay_bf16, c)) * t);
    else
      static_cast<float*>(out)[static_cast<int64_t>(blockIdx.y) * H + c] = t;
  }
}

// One new token per row: a thread per V channels, states read and written in place. 600 rows of
// 100 channels: 2.2 us, the launch itself; 70,915 rows of 260 bf16: 61 us, 4.8 TB/s over rows of
// the table in any order.
template <class T, int V>
__global__ void __launch_bounds__(256) scan_step_kernel(const ScanStepArgs A) {
  const int lanes = A.width / V;
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (e >= A.rows * lanes) return;
  const int64_t row = e / lanes;
  const int c = static_cast<int>(e - row * lanes) * V;
  const T* p = static_cast<const T*>(A.p) + row * A.p_sb + c;
  Pack<T, V> in[3], out;
#pragma unroll
  for (int w = 0; w < 3; ++w) in[w].load(p + w * static_cast<int64_t>(A.width));
  Vf<V> x, r, i, k, h;
  in[0].get(x.v);
  in[1].get(r.v);
  in[2].get(i.v);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    k[v] = decay_factor(param_at(A.decay, A.decay_bf16, c + v), A.rate);
    h[v] = 0.f;
  }
  const int64_t at = A.index != nullptr ? A.index[row] : row;
  if (at < 0 || at >= A.table_rows) {
    record_status(A.status, kBadIndex);  // the row is left out
  } else {
    auto* to = reinterpret_cast<typename Pack<float, V>::Raw*>(A.state + at * A.state_sb + c);
    Pack<float, V> s;
    s.raw = *to;
    s.get(h.v);
    const Step<V> g = step_of(x, r, i, k);
    h = fma(g.a, h, g.add);
    s.set(h.v);
    *to = s.raw;
  }
  out.set(h.v);
  out.store(static_cast<T*>(A.h) + row * A.width + c);
}

constexpr int64_t kSumRows = 64;  // above 8 times it the partial sums are added up in two launches

}  // namespace

// Segments: as many as fill the SMs once with the forward kernels' threads (1024 an SM with the
// slots of fp32 channels by four, else 768; a partly filled second round costs as much as a whole
// one: the four passes over 2 x 65,537 x 256 bf16 293 us with 768, 303 with 1024), none shorter than
// 2 kStateEvery; at most 4096, whose states the carry kernel walks in under 20 us (8192 for packed
// 1,000,000 x 100 fp32: the passes 15 us less in all, the two carries 11 us more). Sequences that fill half
// of that by themselves are left whole: the second read would cost more than the idle threads.
ScanPlan scan_plan(const ScanArgs& a, int sms, void* workspace) {
  const int64_t batch = a.offsets != nullptr ? 1 : a.batch;
  const int64_t lanes = batch * ((a.width + a.vec - 1) / a.vec);
  const int64_t want = static_cast<int64_t>(sms) * (a.vec == 4 && !a.bf16 ? 1024 : 768);
  ScanPlan p;
  p.seg = {1, (a.steps + kStateEvery - 1) / kStateEvery * kStateEvery};
  if (lanes * 2 < want && a.steps > 4 * kStateEvery) {
    int64_t n = want / lanes;
    n = n < 4096 ? n : 4096;
    int64_t len = (a.steps + n - 1) / n;
    len = len > 2 * kStateEvery ? len : 2 * kStateEvery;
    len = (len + kStateEvery - 1) / kStateEvery * kStateEvery;
    p.seg = {(a.steps + len - 1) / len, len};
  }
  p.maps = static_cast<float2*>(workspace);
  p.carry = reinterpret_cast<float*>(p.maps + p.seg.n * batch * a.width);
  p.reach = reinterpret_cast<int*>(p.carry + p.seg.n * batch * a.width);
  return p;
}

size_t scan_workspace(const ScanArgs& a, int sms) {
  const ScanPlan p = scan_plan(a, sms, nullptr);
  const int64_t batch = a.offsets != nullptr ? 1 : a.batch;
  if (p.seg.n == 1) return 0;
  return static_cast<size_t>(p.seg.n * batch * a.width) * (sizeof(float2) + sizeof(float)) +
         (a.offsets != nullptr ? static_cast<size_t>(p.seg.n) * sizeof(int) : 0);
}

int64_t scan_partials(const ScanArgs& a, int sms) {
  const int64_t n = scan_bwd_blocks(a, scan_plan(a, sms, nullptr), sms);
  return n > 8 * kSumRows ? n + kSumRows : n;
}

void launch_scan_fwd(const ScanArgs& a, int sms, void* workspace, cudaStream_t st) {
  const ScanPlan p = scan_plan(a, sms, workspace);
  if (a.offsets != nullptr) launch_sequences(a, p, false, st);
  if (a.steps == 0 && a.offsets != nullptr) return;
  if (p.seg.n > 1) {
    scan_fwd_maps(a, p, sms, st);
    launch_carry(a, p, false, st);
  }
  scan_fwd_rows(a, p, sms, st);
}

void launch_scan_bwd(const ScanArgs& a, int sms, void* workspace, void* ddecay, cudaStream_t st) {
  const ScanPlan p = scan_plan(a, sms, workspace);
  if (a.offsets != nullptr) launch_sequences(a, p, true, st);
  if (p.seg.n > 1) {
    scan_bwd_maps(a, p, sms, st);
    launch_carry(a, p, true, st);
  }
  scan_bwd_rows(a, p, sms, st);
  int64_t n = scan_bwd_blocks(a, p, sms);
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

template <class T, int V>
static void run_step(const ScanStepArgs& a, cudaStream_t st) {
  const int64_t n = a.rows * (a.width / V);
  scan_step_kernel<T, V><<<static_cast<unsigned>((n + 255) / 256), 256, 0, st>>>(a);
}

void launch_scan_step(const ScanStepArgs& a, cudaStream_t st) {
  count_launch();
  if (a.bf16)
    a.vec == 4 ? run_step<__nv_bfloat16, 4>(a, st) : run_step<__nv_bfloat16, 1>(a, st);
  else
    a.vec == 4 ? run_step<float, 4>(a, st) : run_step<float, 1>(a, st);
}

}  // namespace su
