// Activations in 8 bits: per group of 32 values of a row, scale = amax / 127 and
// code = rint(v * (127 / amax)). Bound by bytes: each value is read once, and one byte
// is written for it and four for the group's scale. 1,600,000 x 64 fp32: 101 us to codes
// (5.2 TB/s; three exchanges a group, a division on each of its eight lanes and the rounding cost
// issue), 84 us back (6.3 TB/s).
#include "scan_shape.cuh"

namespace su {
namespace {

constexpr int kUnroll = 4;  // rows whose loads are under way together

// A group of 32 values per 32 / V lanes; every group of a row has lanes of its own.
template <class T, int V, bool NARROW>
__global__ void __launch_bounds__(256) quantize8_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int H,
                                                        int8_t* __restrict__ codes, float* __restrict__ scales,
                                                        const Lanes L) {
  const int G = groups_in(H);
  const int group = group_lanes(H, V);
  const int64_t step = static_cast<int64_t>(gridDim.x) * L.rows;
  for (int cb = blockIdx.y; cb < L.blocks; cb += gridDim.y)  // very long rows
    for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * L.rows + threadIdx.x / L.count; r0 < rows;
       r0 += kUnroll * step) {
    const int c = (cb * L.count + threadIdx.x % L.count) * V;
    const bool live = c < H;
    Pack<T, V> a[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      a[j].zero();
      if (live && r0 + j * step < rows) a[j].load(x + (r0 + j * step) * ld + c);
    }
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int64_t row = r0 + j * step;
      if (row >= rows) break;
      float f[V];
      a[j].get(f);
      Codes<V> q;
      const float s = encode8<NARROW>(f, q, group);
      if (live) {
        q.store(codes + row * H + c);
        if (c % kGroup8 == 0) scales[row * G + c / kGroup8] = s;
      }
    }
  }
}

template <class T, int V>
__global__ void __launch_bounds__(256) dequantize8_kernel(const int8_t* __restrict__ codes,
                                                          const float* __restrict__ scales, int64_t rows, int H,
                                                          T* __restrict__ x, const Lanes L) {
  const int G = groups_in(H);
  const int64_t step = static_cast<int64_t>(gridDim.x) * L.rows;
  for (int cb = blockIdx.y; cb < L.blocks; cb += gridDim.y)  // very long rows
    for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * L.rows + threadIdx.x / L.count; r0 < rows;
       r0 += kUnroll * step) {
    const int c = (cb * L.count + threadIdx.x % L.count) * V;
    if (c >= H) break;
    Codes<V> q[kUnroll];
    float s[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      if (r0 + j * step < rows) {
        q[j].load(codes + (r0 + j * step) * H + c);
        s[j] = scales[(r0 + j * step) * G + c / kGroup8];
      }
    }
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int64_t row = r0 + j * step;
      if (row >= rows) break;
      float f[V];
      q[j].get(s[j], f);
      Pack<T, V> o;
      o.set(f);
      o.store(x + row * H + c);
    }
  }
}

// A row block takes kUnroll of its rows at once; up to 32 blocks of rows per SM.
dim3 grid_of(int64_t rows, const Lanes& l, int sms) {
  const int64_t want = (rows + l.rows * kUnroll - 1) / (l.rows * kUnroll);
  const int64_t most = (static_cast<int64_t>(sms) * 32 + l.blocks - 1) / l.blocks;
  return dim3(static_cast<unsigned>(want < most ? want : most), l.blocks < 65535 ? l.blocks : 65535);
}

template <class T, int V>
void run_quantize(const void* x, int64_t ld, int64_t rows, int width, int8_t* codes, float* scales, int sms,
                  cudaStream_t st) {
  const Lanes l = lanes_of(width, V, true, 256);
  auto kernel = width < kGroup8 ? quantize8_kernel<T, V, true> : quantize8_kernel<T, V, false>;
  kernel<<<grid_of(rows, l, sms), l.count * l.rows, 0, st>>>(static_cast<const T*>(x), ld, rows, width, codes, scales, l);
}
template <class T, int V>
void run_dequantize(const int8_t* codes, const float* scales, int64_t rows, int width, void* x, int sms,
                    cudaStream_t st) {
  const Lanes l = lanes_of(width, V, false, 256);
  dequantize8_kernel<T, V><<<grid_of(rows, l, sms), l.count * l.rows, 0, st>>>(codes, scales, rows, width,
                                                                               static_cast<T*>(x), l);
}

}  // namespace

void launch_quantize8(const void* x, int bf16, int64_t ld, int64_t rows, int width, int8_t* codes, float* scales,
                      int vec, int sms, cudaStream_t st) {
  count_launch();
  if (bf16)
    vec ? run_quantize<__nv_bfloat16, 4>(x, ld, rows, width, codes, scales, sms, st)
        : run_quantize<__nv_bfloat16, 1>(x, ld, rows, width, codes, scales, sms, st);
  else
    vec ? run_quantize<float, 4>(x, ld, rows, width, codes, scales, sms, st)
        : run_quantize<float, 1>(x, ld, rows, width, codes, scales, sms, st);
}

void launch_dequantize8(const int8_t* codes, const float* scales, int64_t rows, int width, void* x, int bf16, int vec,
                        int sms, cudaStream_t st) {
  count_launch();
  if (bf16)
    vec ? run_dequantize<__nv_bfloat16, 4>(codes, scales, rows, width, x, sms, st)
        : run_dequantize<__nv_bfloat16, 1>(codes, scales, rows, width, x, sms, st);
  else
    vec ? run_dequantize<float, 4>(codes, scales, rows, width, x, sms, st)
        : run_dequantize<float, 1>(codes, scales, rows, width, x, sms, st);
}

}  // namespace su
