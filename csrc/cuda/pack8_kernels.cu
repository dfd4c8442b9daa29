// Activations in 8 bits: per group of 32 values of a row, scale = amax / 127 and
// code = rint(v * (127 / amax)). Bound by bytes: each value is read once, and one byte
// plus an eighth of the scale's four bytes is written.
#include "kernels.h"
#include "recurrence.h"
#include "vec_io.cuh"

namespace su {
namespace {

// A group of 32 values per 32 / V lanes, groups of all rows side by side over the threads.
template <class T, int V>
__global__ void __launch_bounds__(256) quantize8_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int H,
                                                        int8_t* __restrict__ codes, float* __restrict__ scales) {
  constexpr int kLanes = kGroup8 / V;
  const int G = (H + kGroup8 - 1) / kGroup8;
  const int64_t groups = rows * G;
  const int lane = threadIdx.x % kLanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (256 / kLanes);
  for (int64_t g = static_cast<int64_t>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes; g < groups; g += step) {
    const int64_t row = g / G;
    const int c = static_cast<int>(g - row * G) * kGroup8 + lane * V;
    const bool live = c < H;
    Pack<T, V> a;
    a.zero();
    if (live) a.load(x + row * ld + c);
    float f[V];
    a.get(f);
    Codes<V> q;
    const float s = encode8(f, q);
    if (live) q.store(codes + row * H + c);
    if (lane == 0) scales[g] = s;
  }
}

template <class T, int V>
__global__ void __launch_bounds__(256) dequantize8_kernel(const int8_t* __restrict__ codes,
                                                          const float* __restrict__ scales, int64_t rows, int H,
                                                          T* __restrict__ x) {
  const int lanes = (H + V - 1) / V;
  const int G = (H + kGroup8 - 1) / kGroup8;
  const int64_t n = rows * lanes;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < n;
       e += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = e / lanes;
    const int c = static_cast<int>(e - row * lanes) * V;
    float f[V];
    Codes<V> q;
    q.load(codes + row * H + c);
    q.get(scales[row * G + c / kGroup8], f);
    Pack<T, V> o;
    o.set(f);
    o.store(x + row * H + c);
  }
}

unsigned grid_for(int64_t threads) {
  const int64_t blocks = (threads + 255) / 256;
  return static_cast<unsigned>(blocks < (1 << 20) ? blocks : (1 << 20));
}

}  // namespace

void launch_quantize8(const void* x, int bf16, int64_t ld, int64_t rows, int width, int8_t* codes, float* scales,
                      int vec, cudaStream_t st) {
  count_launch();
  const int64_t groups = rows * ((width + kGroup8 - 1) / kGroup8);
  const unsigned grid = grid_for(groups * (kGroup8 / (vec ? 4 : 1)));
  if (bf16) {
    const auto* p = static_cast<const __nv_bfloat16*>(x);
    vec ? quantize8_kernel<__nv_bfloat16, 4><<<grid, 256, 0, st>>>(p, ld, rows, width, codes, scales)
        : quantize8_kernel<__nv_bfloat16, 1><<<grid, 256, 0, st>>>(p, ld, rows, width, codes, scales);
  } else {
    const auto* p = static_cast<const float*>(x);
    vec ? quantize8_kernel<float, 4><<<grid, 256, 0, st>>>(p, ld, rows, width, codes, scales)
        : quantize8_kernel<float, 1><<<grid, 256, 0, st>>>(p, ld, rows, width, codes, scales);
  }
}

void launch_dequantize8(const int8_t* codes, const float* scales, int64_t rows, int width, void* x, int bf16, int vec,
                        cudaStream_t st) {
  count_launch();
  const unsigned grid = grid_for(rows * ((width + (vec ? 3 : 0)) / (vec ? 4 : 1)));
  if (bf16) {
    auto* p = static_cast<__nv_bfloat16*>(x);
    vec ? dequantize8_kernel<__nv_bfloat16, 4><<<grid, 256, 0, st>>>(codes, scales, rows, width, p)
        : dequantize8_kernel<__nv_bfloat16, 1><<<grid, 256, 0, st>>>(codes, scales, rows, width, p);
  } else {
    auto* p = static_cast<float*>(x);
    vec ? dequantize8_kernel<float, 4><<<grid, 256, 0, st>>>(codes, scales, rows, width, p)
        : dequantize8_kernel<float, 1><<<grid, 256, 0, st>>>(codes, scales, rows, width, p);
  }
}

}  // namespace su
