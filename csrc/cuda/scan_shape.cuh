// Shared by the forward and backward kernels of the gated recurrence: how channels,
// sequences and segments of steps map to threads, and what marks the packed sequences.
#pragma once

#include "kernels.h"
#include "scan_math.cuh"

namespace su {

// A thread's V channels: lanes of a row side by side, rows over threadIdx / lanes.
struct Lanes {
  int count;   // lanes that one row takes in a block
  int rows;    // rows side by side in a block
  int blocks;  // blocks over the channels
};

// Lanes of H channels at V per lane in blocks of up to `threads` threads; with 8-bit codes
// every group of 32 channels gets its own aligned lanes, the last one's beyond H included.
inline Lanes lanes_of(int width, int V, bool codes, int threads) {
  const int unit = codes ? group_lanes(width, V) : 1;
  // (64 bits: the lanes of 2^31 - 1 columns in whole groups are 2^31)
  const int64_t all = codes ? static_cast<int64_t>(groups_in(width)) * unit : (width - 1) / V + 1;
  Lanes l;
  l.blocks = static_cast<int>((all + threads - 1) / threads);
  l.count = static_cast<int>((all + l.blocks - 1) / l.blocks);
  l.count = (l.count + unit - 1) / unit * unit;
  l.rows = threads / l.count;
  return l;
}

// Steps [k * len, (k + 1) * len) of every sequence are segment k, walked by threads of
// their own. len is a multiple of kStateEvery; n == 1: the whole sequence.
struct Segments {
  int64_t n, len;
};

// Rows of threads over batch x segments: sequences side by side, whose rows are neighbours
// in memory where snapshots are stacked. `turn`: from the last segment to the first.
struct SegRow {
  int64_t q, b;
};
__device__ __forceinline__ SegRow seg_row(int64_t r, int64_t batch, const Segments& S, bool turn) {
  SegRow s;
  s.q = S.n == 1 ? 0 : r / batch;
  s.b = S.n == 1 ? r : r - s.q * batch;
  if (turn) s.q = S.n - 1 - s.q;
  return s;
}

// Packed sequences: marks[row] is -1 inside a sequence; at its first row 4 s + 1, at its last
// 4 s + 2, at an only row 4 s + 3 (a row belongs to one sequence).
constexpr int kMarkFirst = 1, kMarkLast = 2;

enum ScanKind { kPlain = 0, kMasked = 1, kPacked = 2 };  // kPacked checks for a mask itself

inline ScanKind kind_of(const ScanArgs& a) {
  return a.offsets != nullptr ? kPacked : (a.mask != nullptr ? kMasked : kPlain);
}

// blocks over `rows` rows of threads: every SM filled a few times, so that per-block sums stay few
inline int row_blocks(int64_t rows, const Lanes& l, int sms) {
  const int64_t want = (rows + l.rows - 1) / l.rows;
  const int64_t most = (static_cast<int64_t>(sms) * 16 + l.blocks - 1) / l.blocks;
  return static_cast<int>(want < most ? want : most);
}

// What a launch works with beside the arguments: segments, and where there are several, per
// segment, sequence and channel the map (A, B) of the state before it to the state after it
// (backwards: of the gradient after it to the one before it) and the state before it.
struct ScanPlan {
  Segments seg;
  float2* maps;
  float* carry;
  // Packed sequences: a segment's map needs the steps from its last first row on only (backwards:
  // up to its first last row), since a state starts anew there. Per segment the step that
  // the map begins with, or -1 (backwards: the steps of a segment behind the map's). Where there
  // is one, the map's A is kAnew.
  int* reach;
};

// A of a map that forgets the state before it. Not 0, which products of many factors reach: 0 times
// a NaN or an infinity is NaN, right inside a sequence, but nothing of one sequence enters another.
constexpr float kAnew = -1.f;
__device__ __forceinline__ float through(const float2& map, float h) {
  return map.x == kAnew ? map.y : fmaf(map.x, h, map.y);
}
// the map of `first`, then `second`
__device__ __forceinline__ float2 compose(const float2& first, const float2& second) {
  const float a = first.x == kAnew || second.x == kAnew ? kAnew : first.x * second.x;
  return make_float2(a, through(second, first.y));
}

ScanPlan scan_plan(const ScanArgs& a, int sms, void* workspace);
int scan_bwd_blocks(const ScanArgs& a, const ScanPlan& p, int sms);
void scan_fwd_maps(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st);
void scan_fwd_rows(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st);
void scan_bwd_maps(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st);
void scan_bwd_rows(const ScanArgs& a, const ScanPlan& p, int sms, cudaStream_t st);

}  // namespace su
