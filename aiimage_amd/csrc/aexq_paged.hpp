// A paged key/value cache as the kernels see it, and what they share: the
// pieces of attention with scores kept in log2 units.
#pragma once

#include "aexq_dma.hpp"
#include "aexq_serving.hpp"

namespace aexq {

typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Positions sequence s keeps: its device-side length, within what its row of
// the table can hold (the host refuses tables of more than 2^31 - 1 positions).
__device__ __forceinline__ int paged_length(const PagedView& kv, int s) {
  return min(max(kv.lengths[s], 0), kv.width << kv.shift);
}
// The page of sequence s at table column b, moved into the pool as token ids
// are moved into the vocabulary: no entry reads outside it.
__device__ __forceinline__ int paged_page(const PagedView& kv, int s, int b) {
  return min(max(kv.table[(long long)s * kv.width + b], 0), kv.pages - 1);
}

constexpr int kCoherent = 16;  // buffer cache policy sc1: through to what all XCDs share

// Softmax weights are kept as 2^(score - m + kLift), m a running maximum that
// is moved only where a score passes it by more than kLag: weights stay below
// 2^(kLift + kLag) = 2^15 in fp16, and those down to 2^-21 of the largest keep
// all their fp16 bits.  The factor 2^kLift falls out in the division.
constexpr float kLift = 7.0f, kLag = 8.0f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// An output in fp16.  An average of finite fp16 values is within them; the weights'
// rounding may take it up to 2^-11 further, past 65520, where fp16 rounds to infinity.
__device__ __forceinline__ f16 average_f16(float y) {
  return (f16)(fabsf(y) < INFINITY ? fminf(fmaxf(y, -65504.0f), 65504.0f) : y);
}

// Maximum (sum) of v over the four 16-lane rows of the wave, in every lane.
__device__ __forceinline__ float rows_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float rows_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// The sequence whose packed rows hold row t (the one after those that end at or
// before t; offsets[1..n] do not decrease), where its rows end, and its length.
// By a whole wave; the answer is uniform, and one load deep for n <= 64.
struct PackedRow {
  bool found;
  int seq, end, length;
};
__device__ __forceinline__ PackedRow packed_row(const int32_t* offsets, const int32_t* lengths,
                                                int n, int t) {
  const int lane = threadIdx.x & 63;
  for (int b = 0; b < n; b += 64) {
    const int i = min(b + lane, n - 1);
    const int first = offsets[i], end = offsets[i + 1], length = lengths[i];
    const uint64_t after = __ballot(end > t);
    if (!after) continue;
    const int at = __ffsll((unsigned long long)after) - 1;
    return PackedRow{__builtin_amdgcn_readlane(first, at) <= t, b + at,
                     __builtin_amdgcn_readlane(end, at), __builtin_amdgcn_readlane(length, at)};
  }
  return PackedRow{false, 0, 0, 0};
}

}  // namespace aexq
