// What stands around the gated delta rule in a recurrent layer (gfx950): the short
// causal convolution before it and the gated norm behind it.
#include <math.h>

#include "aexq_rows.hpp"

namespace aexq {

// ---------------------------------------------------------------------------
// Short causal convolution, channel by channel along a sequence,
//   y[t][c] = act(bias[c] + sum_j w[c][j] x[t - (W - 1) + j][c])
// in fp32, rounded once; the inputs before the first are the sequence's state, the
// last W - 1 ones before.  A thread takes 8 channels over a block of kConvRows rows,
// its last W - 1 inputs in registers.  The block that starts a sequence reads the
// state and stores the new one, so no other workgroup meets it.
// ---------------------------------------------------------------------------
constexpr int kConvRows = 16;

__device__ __forceinline__ f16x8 load8(const f16* p) { return *(const f16x8*)p; }

template <int W>
__global__ __launch_bounds__(kThreads) void short_conv_kernel(const ShortConvParams p) {
  const int groups = (p.channels / 8 + kThreads - 1) / kThreads;
  const int id = blockIdx.x / groups, group = blockIdx.x % groups;
  const RowBlock at = row_block<kConvRows>(p.offsets, p.tokens, p.slots.n, id);
  const Span span = span_of(p.slots, p.offsets, p.tokens, at.seq);
  const int c = 8 * (group * kThreads + threadIdx.x);
  const int t0 = at.block * kConvRows, t1 = min(t0 + kConvRows, span.kept);
  if (t0 >= span.kept || c >= p.channels) return;

  // input of place t among the sequence's rows, the state's below 0
  f16* state = p.state + (long long)max(span.slot, 0) * (W - 1) * p.channels + c;
  auto input = [&](int t) {
    if (t >= 0) return load8(p.x + (span.first + t) * p.x_stride + c);
    return span.fresh ? f16x8{} : load8(state + (long long)(t + W - 1) * p.channels);
  };
  f16x8 last[W];  // inputs t - W .. t - 1 (the first unused)
#pragma unroll
  for (int j = 1; j < W; ++j) last[j] = input(t0 + j - W);
  if (p.out) {
    float w[8][W], bias[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int j = 0; j < W; ++j) w[i][j] = p.weight[(long long)(c + i) * W + j];
      bias[i] = p.bias ? p.bias[c + i] : 0.0f;
    }
    f16x8 row[W];
#pragma unroll
    for (int j = 1; j < W; ++j) row[j] = last[j];
    for (int t = t0; t < t1; ++t) {
#pragma unroll
      for (int j = 0; j + 1 < W; ++j) row[j] = row[j + 1];
      row[W - 1] = input(t);
      f16x8 y;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float v = bias[i];
#pragma unroll
        for (int j = 0; j < W; ++j) v = fmaf(w[i][j], (float)row[j][i], v);
        y[i] = (f16)(p.silu ? v / (1.0f + __expf(-v)) : v);
      }
      *(f16x8*)(p.out + (span.first + t) * p.out_stride + c) = y;
    }
  }
  if (at.block || !p.slots.store || span.slot < 0) return;
  // the last W - 1 inputs; the state's rows that stay move up
  f16x8 next[W];
#pragma unroll
  for (int j = 1; j < W; ++j) next[j] = input(span.kept + j - W);
#pragma unroll
  for (int j = 1; j < W; ++j) *(f16x8*)(state + (long long)(j - 1) * p.channels) = next[j];
}

hipError_t short_conv_launch(const ShortConvParams& p, hipStream_t stream) {
  const long long groups = (p.channels / 8 + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)(row_blocks(p.tokens, p.slots.n, kConvRows) * groups));
  switch (p.width) {
    case 2: hipLaunchKernelGGL(short_conv_kernel<2>, grid, dim3(kThreads), 0, stream, p); break;
    case 3: hipLaunchKernelGGL(short_conv_kernel<3>, grid, dim3(kThreads), 0, stream, p); break;
    case 4: hipLaunchKernelGGL(short_conv_kernel<4>, grid, dim3(kThreads), 0, stream, p); break;
    default: hipLaunchKernelGGL(short_conv_kernel<5>, grid, dim3(kThreads), 0, stream, p); break;
  }
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Root-mean-square norm of each head, gated by silu:
//   y = x rsqrt(max(mean(x^2) + eps, 1e-20)) gamma silu(z)
// in fp32, rounded once.  LPR lanes take a row, 8 values each.
// ---------------------------------------------------------------------------
template <int LPR>
__global__ __launch_bounds__(kThreads) void gated_norm_kernel(const GatedNormParams p) {
  const long long row = (long long)blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  const int i = threadIdx.x % LPR * 8;
  const bool on = row < p.rows && i < p.dim;
  const long long token = min(row, p.rows - 1) / p.heads;
  const int head = (int)(min(row, p.rows - 1) % p.heads);
  f16x8 x = f16x8{}, z = f16x8{};
  if (on) {
    x = load8(p.x + token * p.x_stride + (long long)head * p.dim + i);
    z = load8(p.z + token * p.z_stride + (long long)head * p.dim + i);
  }
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum = fmaf((float)x[e], (float)x[e], sum);
#pragma unroll
  for (int off = LPR / 2; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if (!on) return;
  const float r = 1.0f / sqrtf(fmaxf(sum / p.dim + p.eps, 1e-20f));
  f16x8 y;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float gate = (float)z[e];
    const float v = (float)x[e] * r * (p.gamma ? p.gamma[i + e] : 1.0f);
    y[e] = (f16)(v * (gate / (1.0f + __expf(-gate))));
  }
  *(f16x8*)(p.out + token * p.out_stride + (long long)head * p.dim + i) = y;
}

hipError_t gated_norm_launch(const GatedNormParams& p, hipStream_t stream) {
  int lpr = 8;
  while (8 * lpr < p.dim) lpr *= 2;
  const long long per = kThreads / lpr;
  const dim3 grid((unsigned)((p.rows + per - 1) / per));
  switch (lpr) {
    case 8: hipLaunchKernelGGL(gated_norm_kernel<8>, grid, dim3(kThreads), 0, stream, p); break;
    case 16: hipLaunchKernelGGL(gated_norm_kernel<16>, grid, dim3(kThreads), 0, stream, p); break;
    case 32: hipLaunchKernelGGL(gated_norm_kernel<32>, grid, dim3(kThreads), 0, stream, p); break;
    default: hipLaunchKernelGGL(gated_norm_kernel<64>, grid, dim3(kThreads), 0, stream, p); break;
  }
  return hipGetLastError();
}

}  // namespace aexq
