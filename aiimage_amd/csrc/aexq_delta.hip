// The gated delta rule (gfx950), a recurrence along each sequence over a state S
// [dim_k][dim_v] per value head:
//   S <- e^g S,  u = beta (v - S^T k^),  S <- S + k^ u^T,  o = scale S^T q^
// with g = -e^a_log softplus(a + dt_bias), beta = sigmoid(b), q^ and k^ of unit length.
// States and all sums are fp32.
#include <math.h>

#include "aexq_rows.hpp"

namespace aexq {

// Log decay and strength of a row; a decay past fp32's range is 0 all the same.
struct Gate {
  float g, beta;
};
__device__ __forceinline__ Gate gate_of(const DeltaParams& p, long long row, int head) {
  const float t = (float)p.a[row * p.a_stride + head] + p.dt_bias[head];
  const float b = (float)p.b[row * p.b_stride + head];
  const float soft = fmaxf(t, 0.0f) + log1pf(expf(-fabsf(t)));
  const float g = -expf(p.a_log[head]) * soft;
  return Gate{g < -1e5f ? -1e5f : g, 1.0f / (1.0f + expf(-b))};
}

// Sum of v over the four 16-lane rows of the wave, in every lane.
__device__ __forceinline__ float rows_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// ---------------------------------------------------------------------------
// Packed prompts.  A workgroup takes NC blocks of 16 columns of S (columns are
// independent of one another) of one value head of one sequence; its wave w holds
// rows w DK / 4 .. of them in the layout of a matrix product's result: lane (c = l %
// 16, g = l / 16) has rows 16 t + 4 g + r, column c of block n.
// ---------------------------------------------------------------------------
template <int DK, int NC>
struct DeltaLds {
  float sums[2][kWaves][2][NC][16];
};

template <int DK, int NC>
struct DeltaState {
  static constexpr int NT = DK / 64;  // 16-row tiles of a wave
  f32x4 s[NT][NC];
};

// Row after row of [t0, t1).
template <int DK, int NC>
__device__ __forceinline__ void delta_rows(const DeltaParams& p, const Span& span, int head,
                                           int col, int t0, int t1, DeltaState<DK, NC>& S,
                                           DeltaLds<DK, NC>& lds) {
  constexpr int NT = DK / 64;
  const int lane = threadIdx.x & 63, wave = sreg((int)threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  for (int t = t0; t < t1; ++t) {
    const long long row = span.first + t;
    const f16* kr = p.k + row * p.k_stride + head / p.group * DK;
    const f16* qr = p.q + row * p.q_stride + head / p.group * DK;
    float kk = 0.0f, qq = 0.0f, kq = 0.0f;
#pragma unroll
    for (int i = 0; i < DK / 64; ++i) {
      const float k = (float)kr[lane + 64 * i], q = (float)qr[lane + 64 * i];
      kk = fmaf(k, k, kk);
      qq = fmaf(q, q, qq);
      kq = fmaf(k, q, kq);
    }
    const float rk = 1.0f / sqrtf(wave_sum(kk) + p.eps), rq = 1.0f / sqrtf(wave_sum(qq) + p.eps);
    kq = wave_sum(kq) * rk;
    const Gate gate = gate_of(p, row, head);
    const float decay = expf(gate.g);
    f16x4 k[NT], q[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      k[i] = *(const f16x4*)(kr + wave * (DK / 4) + 16 * i + 4 * g);
      q[i] = *(const f16x4*)(qr + wave * (DK / 4) + 16 * i + 4 * g);
    }
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      float sk = 0.0f, sq = 0.0f;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          S.s[i][n][r] *= decay;
          sk = fmaf(S.s[i][n][r], (float)k[i][r], sk);
          sq = fmaf(S.s[i][n][r], (float)q[i][r], sq);
        }
      sk = rows_sum(sk);
      sq = rows_sum(sq);
      if (g == 0) {
        lds.sums[t & 1][wave][0][n][c] = sk;
        lds.sums[t & 1][wave][1][n][c] = sq;
      }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      float sk = 0.0f, sq = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        sk += lds.sums[t & 1][w][0][n][c];
        sq += lds.sums[t & 1][w][1][n][c];
      }
      const int at = col + 16 * n + c;
      const float v = (float)p.v[row * p.v_stride + head * p.dv + at];
      const float u = gate.beta * (v - rk * sk);
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          S.s[i][n][r] = fmaf((float)k[i][r] * rk, u, S.s[i][n][r]);
      if (p.out && wave == 0 && g == 0)
        p.out[row * p.out_stride + head * p.dv + at] = (f16)(p.scale * rq * fmaf(u, kq, sq));
    }
  }
}

template <int DK, int NC>
__global__ __launch_bounds__(kThreads) void delta_prompt_kernel(const DeltaParams p) {
  constexpr int NT = DK / 64;
  __shared__ DeltaLds<DK, NC> lds;
  const int parts = p.dv / (16 * NC);
  const int part = blockIdx.x % parts, head = blockIdx.x / parts % p.hv;
  const int s = blockIdx.x / parts / p.hv;
  const int lane = threadIdx.x & 63, wave = sreg((int)threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4, col = part * 16 * NC;
  const Span span = span_of(p.slots, p.offsets, p.tokens, s);
  if (!span.kept) return;
  DeltaState<DK, NC> S;
  float* state = p.state + ((long long)max(span.slot, 0) * p.hv + head) * DK * p.dv +
                 (wave * (DK / 4) + 4 * g) * p.dv + col + c;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        S.s[i][n][r] = span.fresh ? 0.0f : state[(16 * i + r) * p.dv + 16 * n];
  delta_rows<DK, NC>(p, span, head, col, 0, span.kept, S, lds);
  if (!p.slots.store || span.slot < 0) return;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) state[(16 * i + r) * p.dv + 16 * n] = S.s[i][n][r];
}

hipError_t delta_prompt_launch(const DeltaParams& p, int cus, hipStream_t stream) {
  const dim3 grid((unsigned)((long long)p.slots.n * p.hv * (p.dv / 32)));
  if (p.dk == 64)
    hipLaunchKernelGGL((delta_prompt_kernel<64, 2>), grid, dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((delta_prompt_kernel<128, 2>), grid, dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// One row per sequence.  A workgroup takes 4 QW columns of S of one value head;
// thread (y = t % QW, r = t / QW) has columns 4 y .. of the DK QW / 256 rows from r's
// on, so loads and stores are 16 bytes wide.  S^T k^ and S^T q^ are summed together
// before the update, o = scale (e^g S^T q^ + (k^ . q^) u).
// ---------------------------------------------------------------------------
template <int DK, int QW>
__global__ __launch_bounds__(kThreads) void delta_decode_kernel(const DeltaParams p) {
  constexpr int RPT = DK * QW / kThreads;  // rows of a thread
  __shared__ float kn[DK], qn[DK];
  __shared__ f32x4 sums[kWaves][2][QW];
  const int parts = p.dv / (4 * QW), tid = threadIdx.x, lane = tid & 63;
  const int part = blockIdx.x % parts, head = blockIdx.x / parts % p.hv;
  const int s = blockIdx.x / parts / p.hv;
  const Span span = span_of(p.slots, nullptr, p.slots.n, s);
  if (!span.kept) return;
  const int wave = sreg(tid >> 6), y = tid % QW, r = tid / QW, col = part * 4 * QW + 4 * y;
  float* state = p.state + ((long long)max(span.slot, 0) * p.hv + head) * DK * p.dv +
                 (long long)r * RPT * p.dv + col;
  f32x4 S[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) S[i] = span.fresh ? f32x4{} : *(const f32x4*)(state + i * p.dv);

  const f16* kr = p.k + s * p.k_stride + head / p.group * DK;
  const f16* qr = p.q + s * p.q_stride + head / p.group * DK;
  const f16x4 v = *(const f16x4*)(p.v + s * p.v_stride + head * p.dv + col);
  float kk = 0.0f, qq = 0.0f, kq = 0.0f, ke[DK / 64], qe[DK / 64];
#pragma unroll
  for (int i = 0; i < DK / 64; ++i) {
    ke[i] = (float)kr[lane + 64 * i];
    qe[i] = (float)qr[lane + 64 * i];
    kk = fmaf(ke[i], ke[i], kk);
    qq = fmaf(qe[i], qe[i], qq);
    kq = fmaf(ke[i], qe[i], kq);
  }
  const float rk = 1.0f / sqrtf(wave_sum(kk) + p.eps), rq = 1.0f / sqrtf(wave_sum(qq) + p.eps);
  kq = wave_sum(kq) * rk * rq;
  if (wave == 0)
#pragma unroll
    for (int i = 0; i < DK / 64; ++i) {
      kn[lane + 64 * i] = ke[i] * rk;
      qn[lane + 64 * i] = qe[i] * rq;
    }
  const Gate gate = gate_of(p, s, head);
  const float decay = expf(gate.g);
  __syncthreads();
  f32x4 sk = f32x4{}, sq = f32x4{};
  float k[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    k[i] = kn[r * RPT + i];
    const float q = qn[r * RPT + i];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      S[i][e] *= decay;
      sk[e] = fmaf(S[i][e], k[i], sk[e]);
      sq[e] = fmaf(S[i][e], q, sq[e]);
    }
  }
#pragma unroll
  for (int off = 32; off >= QW; off >>= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sk[e] += __shfl_xor(sk[e], off, 64);
      sq[e] += __shfl_xor(sq[e], off, 64);
    }
  if (lane < QW) {
    sums[wave][0][y] = sk;
    sums[wave][1][y] = sq;
  }
  __syncthreads();
  sk = sq = f32x4{};
#pragma unroll
  for (int w = 0; w < kWaves; ++w)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sk[e] += sums[w][0][y][e];
      sq[e] += sums[w][1][y][e];
    }
  f32x4 u;
#pragma unroll
  for (int e = 0; e < 4; ++e) u[e] = gate.beta * ((float)v[e] - sk[e]);
  if (p.out && tid < QW) {
    f16x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (f16)(p.scale * fmaf(u[e], kq, sq[e]));
    *(f16x4*)(p.out + s * p.out_stride + head * p.dv + col) = o;
  }
  if (!p.slots.store || span.slot < 0) return;
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) S[i][e] = fmaf(k[i], u[e], S[i][e]);
    *(f32x4*)(state + i * p.dv) = S[i];
  }
}

template <int DK>
static void decode_launch(const DeltaParams& p, int qw, hipStream_t stream) {
  const dim3 grid((unsigned)((long long)p.slots.n * p.hv * (p.dv / (4 * qw))));
  if (qw == 8)
    hipLaunchKernelGGL((delta_decode_kernel<DK, 8>), grid, dim3(kThreads), 0, stream, p);
  else if (qw == 16)
    hipLaunchKernelGGL((delta_decode_kernel<DK, 16>), grid, dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((delta_decode_kernel<DK, 32>), grid, dim3(kThreads), 0, stream, p);
}

hipError_t delta_decode_launch(const DeltaParams& p, int cus, hipStream_t stream) {
  // columns of a workgroup: few while there are fewer workgroups than places
  const long long heads = (long long)p.slots.n * p.hv;
  int qw = p.dv == 64 ? 16 : 32;
  while (qw > 8 && heads * (p.dv / (4 * qw)) < 2LL * cus) qw /= 2;
  if (p.dk == 64)
    decode_launch<64>(p, qw, stream);
  else
    decode_launch<128>(p, qw, stream);
  return hipGetLastError();
}

}  // namespace aexq
