// The rows and the state of a sequence of packed tokens, as the kernels of the
// recurrent layers see them.
#pragma once

#include "aexq_device.hpp"
#include "aexq_recurrent.hpp"

namespace aexq {

typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));

// Rows first .. first + rows - 1 of the packed tokens, whatever the offsets hold kept
// within them; the first `kept` are taken.  slot < 0: the state begins at zero and is
// not stored.  fresh: it begins at zero.
struct Span {
  int first, rows, kept, slot;
  bool fresh;
};
__device__ __forceinline__ Span span_of(const SlotsView& v, const int32_t* offsets, int tokens,
                                        int s) {
  Span r;
  if (offsets) {
    r.first = min(max(offsets[s], 0), tokens);
    r.rows = min(max(offsets[s + 1], r.first), tokens) - r.first;
  } else {
    r.first = s;
    r.rows = 1;
  }
  r.kept = v.counts ? min(max(v.counts[s], 0), r.rows) : r.rows;
  r.slot = v.slot ? v.slot[s] : s;
  if (r.slot >= v.count) r.slot = -1;
  r.fresh = r.slot < 0 || (v.lengths && v.lengths[s] <= r.rows);
  return r;
}

// Packed rows in blocks of B that start anew with each sequence: block b of sequence s
// is number offsets[s] / B + s + b, so that no sums over sequences are needed; numbers
// that no block has lie between.  The blocks of all sequences are numbers below
// tokens / B + sequences.
__host__ __device__ constexpr long long row_blocks(int tokens, int sequences, int b) {
  return (long long)tokens / b + sequences;
}
struct RowBlock {
  int seq, block;
};
// The sequence and block of number `id` (a block past every sequence's last one where
// there is none).  By a whole wave; 64 sequences a load, the answer is uniform.
template <int B>
__device__ __forceinline__ RowBlock row_block(const int32_t* offsets, int tokens, int n, int id) {
  const int lane = threadIdx.x & 63;
  auto base = [&](int s) { return min(max(offsets[s], 0), tokens) / B + s; };
  int lo = 0, step = 1;
  while (step * 64 < n) step *= 64;
  // the last sequence whose first number is at most id, 64 candidates at a time
  for (;; step /= 64) {
    const int s = lo + lane * step;
    const uint64_t at = __ballot(s < n && base(min(s, n - 1)) <= id);
    lo += max((int)__popcll(at) - 1, 0) * step;
    if (step == 1) break;
  }
  lo = sreg(lo);
  const int block = id - sreg(base(lo));
  return RowBlock{lo, block < 0 ? 1 << 24 : block};
}

// A DPP move of a double; 0 where a lane has no source.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0u, (uint32_t)b, CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0u, (uint32_t)(b >> 32), CTRL, ROWS, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double last_lane(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)b, 63);
  const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(b >> 32), 63);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sums up to and with each lane's, without a trip through LDS: inside rows of 16 lanes
// (row_shr), then the last lane's of a row to the next, of two rows to the next two.
__device__ __forceinline__ double wave_scan(double v) {
  v += dpp64<0x111, 0xF>(v);
  v += dpp64<0x112, 0xF>(v);
  v += dpp64<0x114, 0xF>(v);
  v += dpp64<0x118, 0xF>(v);
  v += dpp64<0x142, 0xA>(v);
  v += dpp64<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ double wave_sum(double v) { return last_lane(wave_scan(v)); }
}  // namespace aexq
