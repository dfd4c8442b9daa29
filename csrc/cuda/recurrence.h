// Launchers of the gated recurrent block: gated linear recurrence, norms around
// a block, 8-bit activations. Nothing here depends on torch headers.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace su {

// Steps between the fp32 states that the recurrence's forward pass keeps for its backward
// pass, which recomputes the steps in between: 16 with 8-bit inputs (the gradients'
// definition has them), else 8, whose factors of two channels fit a thread's registers.
constexpr int kStateEvery = 16;
constexpr int kStateShort = 8;

// Shared memory above the default limit, allowed once per kernel and device (`done` is the
// launcher's own, a bit per device): the call costs as much as a small launch.
template <class K>
inline void allow_smem(K kernel, size_t bytes, uint64_t& done) {
  if (bytes <= 40 * 1024) return;
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (done & bit) return;
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
  done |= bit;
}

constexpr int kGroup8 = 32;  // values of a row that share one scale in the 8-bit format
// groups of a row of 1 to 2^31 - 1 values
#ifdef __CUDACC__
__host__ __device__
#endif
inline int groups_in(int width) { return (width - 1) / kGroup8 + 1; }

// One call of the gated linear recurrence. Sequences lie in a [batch, steps] grid
// (offsets == nullptr) or one after another on one axis of `steps` rows (packed).
// Row (b, t) of the dense outputs is b * row_sb + t * row_st.
struct ScanArgs {
  int bf16 = 0;                // p, h, dh and dp are bf16 (else fp32)
  int64_t batch = 0;           // sequences
  int64_t steps = 0;           // steps of every sequence; packed: rows of all sequences
  int width = 0;               // H
  float rate = 0.f;
  const void* p = nullptr;     // [.., 3H]: x | r | i; element strides of batch and step
  int64_t p_sb = 0, p_st = 0;
  const uint8_t* mask = nullptr;  // 0: the step carries the state
  int64_t m_sb = 0, m_st = 0;
  const void* decay = nullptr;  // [H]
  int decay_bf16 = 0;
  const float* h0 = nullptr;    // [batch, H] or nullptr (zeros)
  const int64_t* offsets = nullptr;  // [batch + 1]
  int* marks = nullptr;         // packed: [steps], first and last rows of the sequences (the forward pass writes it)
  int64_t row_sb = 0, row_st = 0;
  void* h = nullptr;            // dense rows of H
  float* last = nullptr;        // [batch, H]
  int state_every = kStateShort;
  float* states = nullptr;      // state before step k * state_every, k >= 1: [batch, n_states, H] (packed: [n_states, H])
  int64_t n_states = 0;
  int8_t* codes = nullptr;      // dense rows of 3H: the inputs in 8 bits (nullptr: not kept)
  float* scales = nullptr;      // dense rows of 3 * ceil(H / 32)
  int* status = nullptr;
  // backward
  const void* dh = nullptr;     // [.., H] or nullptr
  int64_t dh_sb = 0, dh_st = 0;
  const float* dlast = nullptr;  // [batch, H] or nullptr
  void* dp = nullptr;           // dense rows of 3H
  float* dh0 = nullptr;         // [batch, H] or nullptr
  float* partial = nullptr;     // [n_partial, H] per-block sums of -dz sigmoid(r)
  int vec = 1;                  // 4 or 2: every row of p, dh, h, dp starts on a multiple of so many values; else 1
};

// Bytes of workspace that a call needs (16-byte aligned, no initial value).
size_t scan_workspace(const ScanArgs& a, int sms);
// Rows of `partial` that the backward pass writes, the ones it adds them up in included.
int64_t scan_partials(const ScanArgs& a, int sms);
void launch_scan_fwd(const ScanArgs& a, int sms, void* workspace, cudaStream_t st);
// also adds `partial` up into ddecay [H] (in the type of decay)
void launch_scan_bwd(const ScanArgs& a, int sms, void* workspace, void* ddecay, cudaStream_t st);

// One step of `rows` sequences whose fp32 states live in a table of table_rows rows;
// index[i] (nullptr: i) is row i's place in the table.
struct ScanStepArgs {
  int bf16 = 0;
  int vec = 1;  // 4: width, rows of p and of the table are multiples of four values
  int64_t rows = 0, table_rows = 0;
  int width = 0;
  float rate = 0.f;
  const void* p = nullptr;
  int64_t p_sb = 0;
  const void* decay = nullptr;
  int decay_bf16 = 0;
  const int64_t* index = nullptr;
  float* state = nullptr;
  int64_t state_sb = 0;
  void* h = nullptr;
  int* status = nullptr;
};
void launch_scan_step(const ScanStepArgs& a, cudaStream_t st);

// Norms before and after a block with its gate and residual scale. Null pointers
// leave their part out.
struct NormArgs {
  int bf16 = 0;
  int64_t rows = 0;
  int width = 0;
  float eps = 0.f;
  const void* x = nullptr;
  const void* u = nullptr;
  const void* gate = nullptr;
  int64_t x_ld = 0, u_ld = 0, gate_ld = 0;
  const void* w_post = nullptr;
  const void* w_pre = nullptr;
  const void* scale = nullptr;
  int post_bf16 = 0, pre_bf16 = 0, scale_bf16 = 0;
  void* y = nullptr;            // dense rows
  void* n = nullptr;
  int8_t* codes = nullptr;      // [parts, rows, H]: x, then u and gate where given
  float* scales = nullptr;      // [parts, rows, ceil(H / 32)]
  // backward
  const void* dy = nullptr;
  const void* dn = nullptr;
  int64_t dy_ld = 0, dn_ld = 0;
  void* dx = nullptr;           // dense rows
  void* du = nullptr;
  void* dgate = nullptr;
  float* partial = nullptr;     // [n_partial, 3, H]
  int n_partial = 0;
  void* dw_post = nullptr;
  void* dw_pre = nullptr;
  void* dscale = nullptr;
  int vec = 1;                  // every row starts on a multiple of 4 values, H % 4 == 0
  int vec8 = 0;                 // the same of 8
};
constexpr int kNormMaxWidth = 16384;
int norm_partials(const NormArgs& a, int sms);
void launch_norm_fwd(const NormArgs& a, int sms, cudaStream_t st);
void launch_norm_bwd(const NormArgs& a, int sms, cudaStream_t st);

// 8-bit codes of dense rows
void launch_quantize8(const void* x, int bf16, int64_t ld, int64_t rows, int width, int8_t* codes, float* scales,
                      int vec, int sms, cudaStream_t st);
void launch_dequantize8(const int8_t* codes, const float* scales, int64_t rows, int width, void* x, int bf16, int vec,
                        int sms, cudaStream_t st);

}  // namespace su
