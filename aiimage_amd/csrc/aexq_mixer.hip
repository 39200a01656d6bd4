// What stands around the gated delta rule in a recurrent layer (gfx950): the short
// causal convolution before it and the gated norm behind it.
#include <math.h>

#include "aexq_rows.hpp"

namespace aexq {

// x sigmoid(x); the reciprocal is v_rcp's, 1 ulp off at most.
__device__ __forceinline__ float silu_of(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + __expf(-x));
}
__device__ __forceinline__ f16x8 load8(const f16* p) { return *(const f16x8*)p; }

// ---------------------------------------------------------------------------
// Short causal convolution, channel by channel along a sequence,
//   y[t][c] = act(bias[c] + sum_j w[c][j] x[t - (W - 1) + j][c])
// in fp32, rounded once; the inputs before the first are the sequence's state, the
// last W - 1 ones before.  A thread takes 4 channels over a block of B rows, the next four
// on their way while four are computed: each input is read once, but for the W - 1 rows
// before a block, and what bounds it is memory.  (8 channels a thread left two waves a
// SIMD of long prompts: 57 us where 4 take 54, and 2 as well.)  The block that starts a sequence reads
// the state and stores the new one, so no other workgroup meets it.
// ---------------------------------------------------------------------------
constexpr int kConvChannels = 4;
__host__ __device__ constexpr int channel_groups(int channels) {
  return (channels / kConvChannels + kThreads - 1) / kThreads;
}

template <int W, int B>
__global__ __launch_bounds__(kThreads) void short_conv_kernel(const ShortConvParams p) {
  constexpr int kBatch = 4, C = kConvChannels;
  typedef f16 Row __attribute__((ext_vector_type(C)));
  auto load = [](const f16* p) { return *(const Row*)p; };
  const int groups = channel_groups(p.channels);
  const int id = blockIdx.x / groups, group = blockIdx.x % groups;
  const RowBlock at = row_block<B>(p.offsets, p.tokens, p.slots.n, id);
  const Span span = span_of(p.slots, p.offsets, p.tokens, at.seq);
  const int c = C * (group * kThreads + threadIdx.x);
  const int t0 = at.block * B, t1 = min(t0 + B, span.kept);
  if (t0 >= span.kept || c >= p.channels) return;

  // input of place t among the sequence's rows, the state's below 0
  f16* state = p.state + (long long)max(span.slot, 0) * (W - 1) * p.channels + c;
  const f16* x = p.x + span.first * p.x_stride + c;
  auto input = [&](int t) {
    if (t >= 0) return load(x + t * p.x_stride);
    return span.fresh ? Row{} : load(state + (long long)(t + W - 1) * p.channels);
  };
  if (p.out) {
    Row row[W - 1 + kBatch], next[kBatch];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) row[j] = input(t0 + j - (W - 1));
    // (rows behind the last one: the last one, again)
    auto fetch = [&](int t) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) next[b] = load(x + min(t + b, t1 - 1) * p.x_stride);
    };
    fetch(t0);
    float w[C][W], bias[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
#pragma unroll
      for (int j = 0; j < W; ++j) w[i][j] = p.weight[(long long)(c + i) * W + j];
      bias[i] = p.bias ? p.bias[c + i] : 0.0f;
    }
    f16* out = p.out + span.first * p.out_stride + c;
    for (int t = t0; t < t1; t += kBatch) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) row[W - 1 + b] = next[b];
      fetch(t + kBatch);
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        Row y;
#pragma unroll
        for (int i = 0; i < C; ++i) {
          float v = bias[i];
#pragma unroll
          for (int j = 0; j < W; ++j) v = fmaf(w[i][j], (float)row[b + j][i], v);
          y[i] = (f16)(p.silu ? silu_of(v) : v);
        }
        if (t + b < t1) *(Row*)(out + (t + b) * p.out_stride) = y;
      }
#pragma unroll
      for (int j = 0; j < W - 1; ++j) row[j] = row[kBatch + j];
    }
  }
  if (at.block || !p.slots.store || span.slot < 0) return;
  // the last W - 1 inputs; the state's rows that stay move up
  Row last[W];
#pragma unroll
  for (int j = 1; j < W; ++j) last[j] = input(span.kept + j - W);
#pragma unroll
  for (int j = 1; j < W; ++j) *(Row*)(state + (long long)(j - 1) * p.channels) = last[j];
}

template <int B>
static hipError_t short_conv_rows(const ShortConvParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)(row_blocks(p.tokens, p.slots.n, B) * channel_groups(p.channels)));
  switch (p.width) {
    case 2: hipLaunchKernelGGL((short_conv_kernel<2, B>), grid, dim3(kThreads), 0, stream, p); break;
    case 3: hipLaunchKernelGGL((short_conv_kernel<3, B>), grid, dim3(kThreads), 0, stream, p); break;
    case 4: hipLaunchKernelGGL((short_conv_kernel<4, B>), grid, dim3(kThreads), 0, stream, p); break;
    default: hipLaunchKernelGGL((short_conv_kernel<5, B>), grid, dim3(kThreads), 0, stream, p); break;
  }
  return hipGetLastError();
}

long long conv_groups(int tokens, int sequences, int channels) {
  return row_blocks(tokens, sequences, 16) * channel_groups(channels);
}

// Blocks of 64 rows where they make two workgroups per CU (256 of them), which read their
// weights and the rows before the block once for 64 rows: 9627 rows of 6144 channels take
// 54 us so and 65 with blocks of 16.  Fewer rows are spread over more workgroups.
hipError_t short_conv_launch(const ShortConvParams& p, hipStream_t stream) {
  return (long long)p.tokens / 64 * channel_groups(p.channels) >= 512 ? short_conv_rows<64>(p, stream)
                                                                   : short_conv_rows<16>(p, stream);
}

// ---------------------------------------------------------------------------
// Root-mean-square norm of each head, gated by silu:
//   y = x rsqrt(max(mean(x^2) + eps, 1e-20)) gamma silu(z)
// in fp32, rounded once.  LPR lanes take a row, 8 values each, and R rows at once, so that
// long calls have eight loads a lane on their way: 159568 rows of 128 take 25.7 us with
// R = 4 (122 MB, 4.8 TB/s; a copy of that size runs at 5.3), 27.9 with 2, 42.9 with 1 and
// 32.1 with 8.  Calls too small to fill the card (below 2^22 values) keep R = 1.
// ---------------------------------------------------------------------------
template <int LPR>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (LPR == 8) {
    v += dpp<0xB1>(v);   // quad_perm [1,0,3,2]
    v += dpp<0x4E>(v);   // quad_perm [2,3,0,1]
    v += dpp<0x141>(v);  // row_half_mirror
    return v;
  } else {
    return group_sum<LPR>(v);
  }
}

template <int LPR, int R>
__global__ __launch_bounds__(kThreads) void gated_norm_kernel(const GatedNormParams p) {
  constexpr int kRows = kThreads / LPR;
  const int i = threadIdx.x % LPR * 8, at = min(i, p.dim - 8);
  const long long row0 = (long long)blockIdx.x * (R * kRows) + threadIdx.x / LPR;
  f16x8 x[R], z[R];
  f16* out[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const unsigned row = (unsigned)min(row0 + r * kRows, p.rows - 1);
    const long long token = row / (unsigned)p.heads;
    const int place = (int)(row % (unsigned)p.heads) * p.dim + at;
    x[r] = load8(p.x + token * p.x_stride + place);
    z[r] = load8(p.z + token * p.z_stride + place);
    out[r] = p.out + token * p.out_stride + place;
  }
  float gamma[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) gamma[e] = p.gamma ? p.gamma[at + e] : 1.0f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf((float)x[r][e], (float)x[r][e], sum);
    sum = lanes_sum<LPR>(i < p.dim ? sum : 0.0f);
    // (a maximum that keeps a NaN: the row's mean is one then, and so are its values)
    const float k = 1.0f / sqrtf(__builtin_elementwise_maximum(sum / p.dim + p.eps, 1e-20f));
    f16x8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (f16)((float)x[r][e] * k * gamma[e] * silu_of((float)z[r][e]));
    if (row0 + r * kRows < p.rows && i < p.dim) *(f16x8*)out[r] = y;
  }
}

static int norm_lanes(int dim) {
  int lanes = 8;
  while (8 * lanes < dim) lanes *= 2;
  return lanes;
}
static int norm_rows_of(long long rows, int dim) { return rows * dim >= 1 << 22 ? 4 : 1; }
long long gated_norm_groups(long long rows, int dim) {
  const long long per = kThreads / norm_lanes(dim) * norm_rows_of(rows, dim);
  return (rows + per - 1) / per;
}

template <int R>
static void gated_norm_rows(const GatedNormParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)gated_norm_groups(p.rows, p.dim));
  switch (norm_lanes(p.dim)) {
    case 8: hipLaunchKernelGGL((gated_norm_kernel<8, R>), grid, dim3(kThreads), 0, stream, p); break;
    case 16: hipLaunchKernelGGL((gated_norm_kernel<16, R>), grid, dim3(kThreads), 0, stream, p); break;
    case 32: hipLaunchKernelGGL((gated_norm_kernel<32, R>), grid, dim3(kThreads), 0, stream, p); break;
    default: hipLaunchKernelGGL((gated_norm_kernel<64, R>), grid, dim3(kThreads), 0, stream, p); break;
  }
}

hipError_t gated_norm_launch(const GatedNormParams& p, hipStream_t stream) {
  if (norm_rows_of(p.rows, p.dim) == 4)
    gated_norm_rows<4>(p, stream);
  else
    gated_norm_rows<1>(p, stream);
  return hipGetLastError();
}

}  // namespace aexq
