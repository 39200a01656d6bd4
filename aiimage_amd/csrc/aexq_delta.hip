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
  f16x8 s[2][DK / 32][NC][64];  // parts of S, R, U and U with the rows' factors
  f16x8 r[2][2][NC][64];
  f16x8 u[4][2][NC][64];
  // the waves' largest magnitudes by column
  alignas(16) float first[NC][16][kWaves], top_s[NC][16][kWaves], top_v[NC][16][kWaves];
  alignas(16) float top_r[NC][16][kWaves], top_u[NC][16][kWaves];
  int odd[kWaves];
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

// ---------------------------------------------------------------------------
// Blocks of 64 rows.  With G the sums of g inside a block, K and Q its rows of k^ and q^,
// S the state before it, and
//   A_ij = beta_i e^(G_i - G_j) k^_i . k^_j  (j < i),   T = (1 + A)^-1,
//   P_ij = e^(G_i - G_j) q^_i . k^_j  (j <= i),
// the rows' u are U = T R, R_i = beta_i (v_i - e^G_i S^T k^_i), and
//   out_i = scale (e^G_i S^T q^_i + sum_j P_ij u_j),
//   S <- e^G_63 S + sum_j e^(G_63 - G_j) k^_j u_j^T.
// T, P and the factors do not depend on S: delta_block_kernel makes them for all blocks
// at once, the blocks of a sequence then follow one another in delta_prompt_kernel.
// No exponent above is positive, and |T_ij| <= 1: T_ij is k^_i^T times products of
// decays and of 1 - beta k^ k^T, which lengthen nothing, times k^_j.
//
// fp32 results from fp16 matrix products: k and q are fp16 already and taken as they
// are, their lengths put into the rows' factors; S, T, R and U are split into two fp16
// numbers, x = x0 + x1 up to 2^-22 of x, scaled by powers of two so that neither part
// leaves fp16's range.  P is rounded to fp16 once, by 2^-11, as it only enters outputs.
//
// Pieces of T and P lie in scratch in the order in which a lane of a matrix product
// takes them: 16 rows by 32 columns, lane (m = l % 16, g = l / 16) row m, columns 4 g ..
// 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3.  In that order a result's column blocks are, as
// they stand, the right operand of the next product: lane (c, g) of a result holds rows
// 4 g + r of column c.
// ---------------------------------------------------------------------------
// Piece (row tile w, columns 32 b ..) of a lower triangle of 64 x 64, b <= w / 2.
__device__ __forceinline__ int piece_of(int w, int b) { return w < 2 ? w : 2 * w - 2 + b; }
constexpr float kPieceScale = 2048.0f;  // of T and P: small entries keep their bits

// Row factors of a block and head: beta, beta e^G / |k|, scale e^G / |q|, and e^(G_63 - G)
// over |k| as the transposed keys have it; then e^G_63.
enum : int { kBeta = 0, kSeen = 1, kAsk = 2, kLeft = 3, kDecay = 4 };
__device__ __forceinline__ float* factors_of(char* head, int which) {
  return (float*)(head + 18 * 1024) + which * kDeltaRows;
}

// e^x of a difference in 64 bits, to fp32's precision.
__device__ __forceinline__ float exp_of(double x) {
  const float hi = (float)x, e = expf(hi);
  return fmaf(e, (float)(x - (double)hi), e);
}

template <int DK>
struct BlockLds {
  alignas(16) f16 k[kDeltaRows][DK + 8];
  alignas(16) float a[kDeltaRows][kDeltaRows + 4], t[kDeltaRows][kDeltaRows + 4];
  alignas(16) f16 p[kDeltaRows][kDeltaRows + 8];
  double sums[kDeltaRows];
  float beta[kDeltaRows], rk[kDeltaRows], rq[kDeltaRows];
};

// One block and key head; the value heads of its group in turn.
template <int DK>
__global__ __launch_bounds__(kThreads) void delta_block_kernel(const DeltaParams p) {
  constexpr int KB = DK / 32;
  __shared__ BlockLds<DK> lds;
  const int hk = blockIdx.x % p.hk, id = blockIdx.x / p.hk;
  const int tid = threadIdx.x, lane = tid & 63, wave = sreg(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const RowBlock at = row_block<kDeltaRows>(p.offsets, p.tokens, p.slots.n, id);
  const Span span = span_of(p.slots, p.offsets, p.tokens, at.seq);
  const int t0 = at.block * kDeltaRows, live = min(kDeltaRows, span.kept - t0);
  if (live <= 0) return;
  // rows past the last one repeat it; their factors are 0
  const long long row = span.first + t0 + min(16 * wave + c, live - 1);
  f16x8 k[KB], q[KB];
#pragma unroll
  for (int i = 0; i < KB; ++i) {
    k[i] = *(const f16x8*)(p.k + row * p.k_stride + hk * DK + 32 * i + 8 * g);
    q[i] = *(const f16x8*)(p.q + row * p.q_stride + hk * DK + 32 * i + 8 * g);
  }
  float kk = 0.0f, qq = 0.0f;
#pragma unroll
  for (int i = 0; i < KB; ++i) {
    *(f16x8*)&lds.k[16 * wave + c][32 * i + 8 * g] = k[i];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      kk = fmaf((float)k[i][e], (float)k[i][e], kk);
      qq = fmaf((float)q[i][e], (float)q[i][e], qq);
    }
  }
  kk = rows_sum(kk);
  qq = rows_sum(qq);
  if (g == 0) {
    lds.rk[16 * wave + c] = 1.0f / sqrtf(kk + p.eps);
    lds.rq[16 * wave + c] = 1.0f / sqrtf(qq + p.eps);
  }
  __syncthreads();
  // products of the wave's 16 rows with the rows up to their last one
  f32x4 ak[4], aq[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    ak[j] = aq[j] = f32x4{};
    if (j > wave) continue;
#pragma unroll
    for (int i = 0; i < KB; ++i) {
      const f16x8 b = *(const f16x8*)&lds.k[16 * j + c][32 * i + 8 * g];
      ak[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[i], b, ak[j], 0, 0, 0);
      aq[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(q[i], b, aq[j], 0, 0, 0);
    }
  }
  // the keys transposed, in the products' order, times a power of two that leaves rows a
  // length of 1/2 to 1 (exact but for values below 2^-14, by 2^-25)
  auto power = [&](float rk) { return as_f32(f32_bits(rk) & 0x7f800000u); };
  {
    f16* to = (f16*)(p.keys + ((long long)id * p.hk + hk) * (DK * kDeltaRows * 2));
#pragma unroll
    for (int i = 0; i < DK / 32; ++i) {  // pieces (tile, block): two a tile
      const int n = wave * (DK / 32) + i, tile = n >> 1, b = n & 1;
      f16x8 y;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int t = 32 * b + (e < 4 ? 0 : 16) + 4 * g + e % 4;
        y[e] = (f16)((float)lds.k[t][16 * tile + c] * power(lds.rk[t]));
      }
      *(f16x8*)(to + (n * 64 + lane) * 8) = y;
    }
  }
  for (int h = 0; h < p.group; ++h) {
    const int head = hk * p.group + h;
    char* to = p.heads + ((long long)id * p.hv + head) * kDeltaHead;
    if (wave == 0) {
      // a row a lane: sums of g in 64 bits, as differences of large ones are taken
      Gate gate = {0.0f, 0.0f};
      if (lane < live) gate = gate_of(p, span.first + t0 + lane, head);
      double G = gate.g;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const double up = __shfl_up(G, off, 64);
        if (lane >= off) G += up;
      }
      const double last = __shfl(G, 63, 64);
      const float rk = lds.rk[lane], e = exp_of(G);
      lds.sums[lane] = G;
      lds.beta[lane] = gate.beta;
      const bool in = lane < live;
      factors_of(to, kBeta)[lane] = gate.beta;
      factors_of(to, kSeen)[lane] = in ? gate.beta * e * rk : 0.0f;
      factors_of(to, kAsk)[lane] = in ? p.scale * e * lds.rq[lane] : 0.0f;
      factors_of(to, kLeft)[lane] = in ? exp_of(last - G) * (rk / power(rk)) : 0.0f;
      if (lane == 63) factors_of(to, kDecay)[0] = e;
    }
    __syncthreads();
    f32x4 rowk, rowq, beta;
    double G[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * wave + 4 * g + r;
      rowk[r] = lds.rk[i];
      rowq[r] = lds.rq[i];
      beta[r] = lds.beta[i];
      G[r] = lds.sums[i];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = 16 * j + c;
      const float rk = lds.rk[col];
      const double Gj = lds.sums[col];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * wave + 4 * g + r;
        float a = 0.0f, w = 0.0f;
        if (col <= i && i < live) {
          const float e = exp_of(G[r] - Gj) * rk;
          a = col < i ? ak[j][r] * rowk[r] * e * beta[r] : 0.0f;
          w = aq[j][r] * rowq[r] * e;
        }
        lds.a[i][col] = a;
        lds.p[i][col] = (f16)(w * kPieceScale);
      }
    }
    __syncthreads();
    // T's diagonal tiles, a column a lane (the four rows of lanes do the same)
    {
      float t[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float v = i == c ? 1.0f : 0.0f;
#pragma unroll
        for (int j = 0; j < i; ++j) v = fmaf(-lds.a[16 * wave + i][16 * wave + j], t[j], v);
        t[i] = v;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i % 4 == g) lds.t[16 * wave + i][16 * wave + c] = t[i];
    }
    __syncthreads();
    // the tiles below them: T_wj = -T_ww sum_l A_wl T_lj, step k of a product taking row
    // 4 g + k of its right operand
    for (int d = 1; d < 4; ++d) {
      const int j = wave - d;
      if (j >= 0) {
        f32x4 x = f32x4{}, y = f32x4{};
        for (int l = j; l < wave; ++l) {
          const f32x4 a = *(const f32x4*)&lds.a[16 * wave + c][16 * l + 4 * g];
#pragma unroll
          for (int s = 0; s < 4; ++s)
            x = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], lds.t[16 * l + 4 * g + s][16 * j + c], x,
                                                     0, 0, 0);
        }
        const f32x4 t = *(const f32x4*)&lds.t[16 * wave + c][16 * wave + 4 * g];
#pragma unroll
        for (int s = 0; s < 4; ++s)
          y = __builtin_amdgcn_mfma_f32_16x16x4f32(t[s], x[s], y, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) lds.t[16 * wave + 4 * g + r][16 * j + c] = -y[r];
      }
      __syncthreads();
    }
    // the wave's rows of T and P as the products take them
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (b > wave / 2) continue;
      const int piece = piece_of(wave, b);
      f16x8 t0, t1, w;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int col = 32 * b + (e < 4 ? 0 : 16) + 4 * g + e % 4;
        const float v = col < 16 * (wave + 1) ? lds.t[16 * wave + c][col] * kPieceScale : 0.0f;
        t0[e] = (f16)v;
        t1[e] = (f16)(v - (float)t0[e]);
        w[e] = lds.p[16 * wave + c][col];
      }
      *(f16x8*)(to + ((piece * 2) * 64 + lane) * 16) = t0;
      *(f16x8*)(to + ((piece * 2 + 1) * 64 + lane) * 16) = t1;
      *(f16x8*)(to + ((12 + piece) * 64 + lane) * 16) = w;
    }
    __syncthreads();
  }
}

// A power of two that takes values of up to `bound` to at most 2^14, and its inverse.
struct Lift {
  float by, back;
};
__device__ __forceinline__ Lift lift_of(float bound) {
  const int e = min(max((int)(f32_bits(bound) >> 23 & 255), 14), 254);
  return Lift{as_f32((uint32_t)(267 - e) << 23), as_f32((uint32_t)(e - 13) << 23)};
}

// A wave's part of the blocks' operands; each is loaded for the next block as soon as
// the present one has used it.
template <int DK, int NC>
struct DeltaBlock {
  f16x8 k[DK / 32], q[DK / 32];     // 16 rows
  f16x8 t[2][2], w[2];              // of T and P, by 32 columns
  f16x8 kt[DK / 64][2];             // keys transposed: DK / 4 rows, by 32 of the block's
  f32x4 beta, seen, ask, left;      // of rows 4 g + r
  f16 v[NC][4];
  float decay;
};

template <int DK, int NC>
__global__ __launch_bounds__(kThreads) void delta_prompt_kernel(const DeltaParams p) {
  constexpr int NT = DK / 64, KB = DK / 32;
  __shared__ DeltaLds<DK, NC> lds;
  // the parts of one head lie on one XCD (workgroup b runs on XCD b % 8): they read the
  // same rows and pieces
  const int parts = p.dv / (16 * NC), units = p.slots.n * p.hv;
  const int unit = blockIdx.x / (8 * parts) * 8 + blockIdx.x % 8;
  const int part = blockIdx.x / 8 % parts;
  if (unit >= units) return;
  const int head = unit % p.hv, s = unit / p.hv, hk = head / p.group;
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

  const int blocks = (span.kept + kDeltaRows - 1) / kDeltaRows;
  const int id0 = span.first / kDeltaRows + s;
  DeltaBlock<DK, NC> B;
  auto head_at = [&](int b) { return p.heads + ((long long)(id0 + b) * p.hv + head) * kDeltaHead; };
  auto load_rows = [&](int b) {  // k, q and v
    const int last = min(kDeltaRows, span.kept - b * kDeltaRows) - 1;
    const long long first = span.first + b * kDeltaRows, row = first + min(16 * wave + c, last);
    const f16* k = p.k + row * p.k_stride + hk * DK + 4 * g;
    const f16* q = p.q + row * p.q_stride + hk * DK + 4 * g;
#pragma unroll
    for (int i = 0; i < KB; ++i) {
      const f16x4 k0 = *(const f16x4*)(k + 32 * i), k1 = *(const f16x4*)(k + 32 * i + 16);
      const f16x4 q0 = *(const f16x4*)(q + 32 * i), q1 = *(const f16x4*)(q + 32 * i + 16);
      B.k[i] = __builtin_shufflevector(k0, k1, 0, 1, 2, 3, 4, 5, 6, 7);
      B.q[i] = __builtin_shufflevector(q0, q1, 0, 1, 2, 3, 4, 5, 6, 7);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 16 * wave + 4 * g + r;
      const f16* v = p.v + (first + min(t, last)) * p.v_stride + head * p.dv + col + c;
#pragma unroll
      for (int n = 0; n < NC; ++n) B.v[n][r] = t <= last ? v[16 * n] : (f16)0.0f;
    }
  };
  auto load_factors = [&](int b) {
    char* at = head_at(b);
    const int i = 16 * wave + 4 * g;
    B.beta = *(const f32x4*)(factors_of(at, kBeta) + i);
    B.seen = *(const f32x4*)(factors_of(at, kSeen) + i);
    B.ask = *(const f32x4*)(factors_of(at, kAsk) + i);
    B.left = *(const f32x4*)(factors_of(at, kLeft) + i);
    B.decay = factors_of(at, kDecay)[0];
  };
  auto load_t = [&](int b) {
    const char* at = head_at(b) + lane * 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int piece = piece_of(wave, min(i, wave / 2));
      B.t[i][0] = *(const f16x8*)(at + piece * 2048);
      B.t[i][1] = *(const f16x8*)(at + piece * 2048 + 1024);
    }
  };
  auto load_out = [&](int b) {  // P and the transposed keys
    const char* at = head_at(b) + 12 * 1024 + lane * 16;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      B.w[i] = *(const f16x8*)(at + piece_of(wave, min(i, wave / 2)) * 1024);
    const char* keys = p.keys + ((long long)(id0 + b) * p.hk + hk) * (DK * kDeltaRows * 2);
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        B.kt[i][j] = *(const f16x8*)(keys + (((wave * NT + i) * 2 + j) * 64 + lane) * 16);
  };

  // largest |S| of a column, as bits: a NaN is above every number
  auto state_max = [&](int n) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) m = max(m, f32_bits(S.s[i][n][r]) & 0x7fffffffu);
    m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
    return max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
  };
  auto top4 = [&](const f32x4& v) { return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])); };
  auto bits4 = [&](const f32x4& v) {
    return as_f32(max(max(f32_bits(v[0]), f32_bits(v[1])), max(f32_bits(v[2]), f32_bits(v[3]))));
  };
  float bound[NC];  // of |S|, by column
  auto meet = [&]() {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const uint32_t m = state_max(n);
      if (g == 0) lds.first[n][c][wave] = as_f32(m);
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NC; ++n) bound[n] = bits4(*(const f32x4*)lds.first[n][c]);
    __syncthreads();
  };
  load_rows(0);
  load_factors(0);
  load_t(0);
  load_out(0);
  meet();

  for (int b = 0; b < blocks; ++b) {
    const int next = min(b + 1, blocks - 1);
    // S in two parts, where all waves read them
    Lift ls[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      ls[n] = lift_of(bound[n]);
      f16 x0[4 * NT], x1[4 * NT];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = S.s[i][n][r] * ls[n].by;
          x0[4 * i + r] = (f16)x;
          x1[4 * i + r] = (f16)(x - (float)x0[4 * i + r]);
        }
      if constexpr (NT == 2) {
        __builtin_memcpy(&lds.s[0][wave][n][lane], x0, 16);
        __builtin_memcpy(&lds.s[1][wave][n][lane], x1, 16);
      } else {
        __builtin_memcpy((char*)&lds.s[0][wave / 2][n][lane] + 8 * (wave & 1), x0, 8);
        __builtin_memcpy((char*)&lds.s[1][wave / 2][n][lane] + 8 * (wave & 1), x1, 8);
      }
      const uint32_t m = state_max(n);
      float mv = 0.0f;
#pragma unroll
      for (int r = 0; r < 4; ++r) mv = fmaxf(mv, fabsf((float)B.v[n][r]));
      mv = fmaxf(mv, __shfl_xor(mv, 16, 64));
      mv = fmaxf(mv, __shfl_xor(mv, 32, 64));
      if (g == 0) {
        lds.top_s[n][c][wave] = as_f32(m);
        lds.top_v[n][c][wave] = mv;
      }
    }
    __syncthreads();
    // S^T k and S^T q of the wave's 16 rows
    f32x4 seen[NC], asked[NC];
    float top_s[NC], top_v[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      seen[n] = asked[n] = f32x4{};
      top_s[n] = bits4(*(const f32x4*)lds.top_s[n][c]);
      top_v[n] = top4(*(const f32x4*)lds.top_v[n][c]);
    }
#pragma unroll
    for (int i = 0; i < KB; ++i)
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const f16x8 y = lds.s[x][i][n][lane];
          seen[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(B.k[i], y, seen[n], 0, 0, 0);
          asked[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(B.q[i], y, asked[n], 0, 0, 0);
        }
    // R in two parts; |R| is within |v| and the column's length
    Lift lr[NC];
    bool odd = false;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      lr[n] = lift_of(fmaf(top_s[n], 12.0f, top_v[n]));
      f16 x0[4], x1[4];
      float m = 0.0f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x =
            B.beta[r] * (float)B.v[n][r] - B.seen[r] * (seen[n][r] * ls[n].back);
        // (what is not finite in a column that was)
        odd |= !(fabsf(x) < INFINITY) && top_s[n] < INFINITY;
        m = fmaxf(m, fabsf(x));
        const float y = x * lr[n].by;
        x0[r] = (f16)y;
        x1[r] = (f16)(y - (float)x0[r]);
      }
      __builtin_memcpy((char*)&lds.r[0][wave / 2][n][lane] + 8 * (wave & 1), x0, 8);
      __builtin_memcpy((char*)&lds.r[1][wave / 2][n][lane] + 8 * (wave & 1), x1, 8);
      m = fmaxf(m, __shfl_xor(m, 16, 64));
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      if (g == 0) lds.top_r[n][c][wave] = m;
    }
    odd = __any(odd);
    if (lane == 0) lds.odd[wave] = odd;
    __syncthreads();
    if (lds.odd[0] | lds.odd[1] | lds.odd[2] | lds.odd[3]) {
      // a product with zeros would take what is not finite to the rows before it
      __syncthreads();
      delta_rows<DK, NC>(p, span, head, col, b * kDeltaRows,
                         min(span.kept, (b + 1) * kDeltaRows), S, lds);
      load_rows(next);
      load_factors(next);
      load_t(next);
      load_out(next);
      meet();
      continue;
    }
    // U = T R of the wave's rows
    f32x4 u[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) u[n] = f32x4{};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i > wave / 2) continue;
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const f16x8 r0 = lds.r[0][i][n][lane], r1 = lds.r[1][i][n][lane];
        u[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(B.t[i][0], r0, u[n], 0, 0, 0);
        u[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(B.t[i][0], r1, u[n], 0, 0, 0);
        u[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(B.t[i][1], r0, u[n], 0, 0, 0);
      }
    }
    // U as it is for the outputs, times the rows' factors for the state; |U| is within
    // 64 |R|
    Lift lu[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      lu[n] = lift_of(64.0f * top4(*(const f32x4*)lds.top_r[n][c]));
      f16 x0[4], x1[4], y0[4], y1[4];
      float m = 0.0f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = u[n][r] * (lr[n].back * (1.0f / kPieceScale));
        const float y = x * B.left[r];
        m = fmaxf(m, fabsf(y));
        const float xs = x * lu[n].by, ys = y * lu[n].by;
        x0[r] = (f16)xs;
        x1[r] = (f16)(xs - (float)x0[r]);
        y0[r] = (f16)ys;
        y1[r] = (f16)(ys - (float)y0[r]);
      }
      __builtin_memcpy((char*)&lds.u[0][wave / 2][n][lane] + 8 * (wave & 1), x0, 8);
      __builtin_memcpy((char*)&lds.u[1][wave / 2][n][lane] + 8 * (wave & 1), x1, 8);
      __builtin_memcpy((char*)&lds.u[2][wave / 2][n][lane] + 8 * (wave & 1), y0, 8);
      __builtin_memcpy((char*)&lds.u[3][wave / 2][n][lane] + 8 * (wave & 1), y1, 8);
      m = fmaxf(m, __shfl_xor(m, 16, 64));
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      if (g == 0) lds.top_u[n][c][wave] = m;
    }
    __syncthreads();
    // the state behind the block
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      f32x4 add[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) add[i] = f32x4{};
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const f16x8 y = lds.u[2 + x][j][n][lane];
#pragma unroll
          for (int i = 0; i < NT; ++i)
            add[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(B.kt[i][j], y, add[i], 0, 0, 0);
        }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          S.s[i][n][r] = fmaf(S.s[i][n][r], B.decay, add[i][r] * lu[n].back);
      bound[n] = fmaf(128.0f, top4(*(const f32x4*)lds.top_u[n][c]), top_s[n] * B.decay);
    }
    if (p.out) {
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        f32x4 o = f32x4{};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i > wave / 2) continue;
          o = __builtin_amdgcn_mfma_f32_16x16x32_f16(B.w[i], lds.u[0][i][n][lane], o, 0, 0, 0);
          o = __builtin_amdgcn_mfma_f32_16x16x32_f16(B.w[i], lds.u[1][i][n][lane], o, 0, 0, 0);
        }
        const float back = p.scale * lu[n].back * (1.0f / kPieceScale);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int t = b * kDeltaRows + 16 * wave + 4 * g + r;
          const float y = fmaf(o[r], back, B.ask[r] * (asked[n][r] * ls[n].back));
          if (t < span.kept)
            p.out[(span.first + t) * p.out_stride + head * p.dv + col + 16 * n + c] = (f16)y;
        }
      }
    }
    load_rows(next);
    load_factors(next);
    load_t(next);
    load_out(next);
  }
  if (!p.slots.store || span.slot < 0) return;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) state[(16 * i + r) * p.dv + 16 * n] = S.s[i][n][r];
}

template <int DK, int NC>
static hipError_t prompt_launch(const DeltaParams& p, hipStream_t stream) {
  const long long blocks = row_blocks(p.tokens, p.slots.n, kDeltaRows);
  hipLaunchKernelGGL(delta_block_kernel<DK>, dim3((unsigned)(blocks * p.hk)), dim3(kThreads), 0,
                     stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const long long units = ((long long)p.slots.n * p.hv + 7) / 8 * 8;
  hipLaunchKernelGGL((delta_prompt_kernel<DK, NC>), dim3((unsigned)(units * (p.dv / (16 * NC)))),
                     dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

hipError_t delta_prompt_launch(const DeltaParams& p, int cus, hipStream_t stream) {
  const bool few = (long long)p.slots.n * p.hv * (p.dv / 32) < cus;
  if (p.dk == 64) return few ? prompt_launch<64, 1>(p, stream) : prompt_launch<64, 2>(p, stream);
  return few ? prompt_launch<128, 1>(p, stream) : prompt_launch<128, 2>(p, stream);
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
