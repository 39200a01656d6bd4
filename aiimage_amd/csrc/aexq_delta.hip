// The gated delta rule (gfx950), a recurrence along each sequence over a state S
// [dim_k][dim_v] per value head:
//   S <- e^g S,  u = beta (v - S^T k^),  S <- S + k^ u^T,  o = scale S^T q^
// with g = -e^a_log softplus(a + dt_bias), beta = sigmoid(b), q^ and k^ of unit length.
// States and all sums are fp32.
#include <math.h>

#include <type_traits>

#include "aexq_dma.hpp"
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

// Sum and maximum of v over the four 16-lane rows of the wave, in every lane: rows swapped
// between two copies of it (v_permlane), no trip through LDS.
template <typename F>
__device__ __forceinline__ float rows_join(float v, F join) {
  const auto a = __builtin_amdgcn_permlane16_swap(f32_bits(v), f32_bits(v), false, false);
  v = join(as_f32(a[0]), as_f32(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
  return join(as_f32(b[0]), as_f32(b[1]));
}
__device__ __forceinline__ float rows_sum(float v) {
  return rows_join(v, [](float x, float y) { return x + y; });
}
__device__ __forceinline__ float rows_max(float v) {
  return rows_join(v, [](float x, float y) { return fmaxf(x, y); });
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
  float back_s[NC][16];  // what the parts of S are to be multiplied by
  int odd[kWaves];
  float sums[2][kWaves][2][NC][16];
};

template <int DK, int NC>
struct DeltaState {
  static constexpr int NT = DK / 64;  // 16-row tiles of a wave
  f32x4 s[NT][NC];
};

// Row after row of [t0, t1), by four waves; a barrier a row.
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

// 2^x of a difference in 64 bits, x <= 0: v_exp_f32 is within 2^-23 of it, the rounding
// of x takes 2^-24 |x| ln 2 (and the weight is 2^x).
__device__ __forceinline__ float exp2_of(double x) { return __builtin_amdgcn_exp2f((float)x); }

// Row factors of a block and head: beta, beta e^G / |k|, scale e^G / |q|, and e^(G_63 - G)
// over |k| as the transposed keys have it; then e^G_63.
enum : int { kBeta = 0, kSeen = 1, kAsk = 2, kLeft = 3, kDecay = 4 };

// The power of two that takes a key of length 1 / rk to a length of 1/2 to 1.
__device__ __forceinline__ float near_one(float rk) {
  return as_f32(f32_bits(rk) & 0x7f800000u);
}

// v of lane I of each row of 16 lanes.
template <int I>
__device__ __forceinline__ float row_value(float v) {
  return as_f32(__builtin_amdgcn_update_dpp(0u, f32_bits(v), 0x150 + I, 0xF, 0xF, true));
}
// f(0), f(1), .. f(N - 1), each number a constant.
template <int N, int I = 0, typename F>
__device__ __forceinline__ void unrolled(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    unrolled<N, I + 1>(f);
  }
}

constexpr int kGateHeads = kWaves;  // heads whose gates are made together, a wave each
template <int DK>
struct BlockLds {
  alignas(16) f16 k[kDeltaRows][DK + 8];
  alignas(16) float t[kDeltaRows][kDeltaRows + 4];
  double sums[kGateHeads][kDeltaRows];  // of log2 of the decays, up to each row
  float beta[kGateHeads][kDeltaRows], rk[kDeltaRows], rq[kDeltaRows];
};

// One block and key head; the value heads of its group in turn.  Products of keys are
// formed with the earlier rows on the left: lane (c, g) then has row 16 w + c and columns
// 16 j + 4 g + r, which is how A and P enter the products behind.
template <int DK>
__global__ __launch_bounds__(kThreads, 4) void delta_block_kernel(const DeltaParams p) {
  constexpr int KB = DK / 32;
  __shared__ BlockLds<DK> lds;
  const int hk = blockIdx.x % p.hk, id = blockIdx.x / p.hk;
  const int tid = threadIdx.x, lane = tid & 63, wave = sreg(tid >> 6);
  const int c = lane & 15, g = lane >> 4, own = 16 * wave + c;
  const RowBlock at = row_block<kDeltaRows>(p.offsets, p.tokens, p.slots.n, id);
  const Span span = span_of(p.slots, p.offsets, p.tokens, at.seq);
  const int t0 = at.block * kDeltaRows, live = min(kDeltaRows, span.kept - t0);
  if (live <= 0) return;
  // rows past the last one repeat it; their factors are 0
  const long long row = span.first + t0 + min(own, live - 1);
  f16x8 k[KB], q[KB];
#pragma unroll
  for (int i = 0; i < KB; ++i) {
    k[i] = *(const f16x8*)(p.k + row * p.k_stride + hk * DK + 32 * i + 8 * g);
    q[i] = *(const f16x8*)(p.q + row * p.q_stride + hk * DK + 32 * i + 8 * g);
  }
  // rows for the next kernel, whose workgroups read them often: heads of one row spread
  // over memory's channels, rows of one head, a power of two apart, would share one
  char* keys = p.keys + ((long long)id * p.hk + hk) * delta_key_bytes(DK);
  float kk = 0.0f, qq = 0.0f;
#pragma unroll
  for (int i = 0; i < KB; ++i) {
    *(f16x8*)&lds.k[own][32 * i + 8 * g] = k[i];
    *(f16x8*)(keys + ((wave * KB + i) * 64 + lane) * 16) = k[i];
    *(f16x8*)(keys + ((4 * KB + wave * KB + i) * 64 + lane) * 16) = q[i];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      kk = fmaf((float)k[i][e], (float)k[i][e], kk);
      qq = fmaf((float)q[i][e], (float)q[i][e], qq);
    }
  }
  const float rk = 1.0f / sqrtf(rows_sum(kk) + p.eps), rq = 1.0f / sqrtf(rows_sum(qq) + p.eps);
  if (g == 0) {
    lds.rk[own] = rk;
    lds.rq[own] = rq;
  }
  __syncthreads();
  f32x4 ak[4], aq[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    ak[j] = aq[j] = f32x4{};
    if (j > wave) continue;
#pragma unroll
    for (int i = 0; i < KB; ++i) {
      const f16x8 x = *(const f16x8*)&lds.k[16 * j + c][32 * i + 8 * g];
      ak[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, k[i], ak[j], 0, 0, 0);
      aq[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q[i], aq[j], 0, 0, 0);
    }
    const f32x4 rj = *(const f32x4*)&lds.rk[16 * j + 4 * g];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      ak[j][r] *= rk * rj[r];
      aq[j][r] *= rq * rj[r];
    }
  }
  // the keys transposed, times a power of two (exact but for values below 2^-14, by 2^-25)
#pragma unroll
  for (int i = 0; i < DK / 32; ++i) {  // pieces (16 of DK, 32 rows): two a tile
    const int n = wave * (DK / 32) + i, tile = n >> 1, b = n & 1;
    f16x8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int t = 32 * b + (e < 4 ? 0 : 16) + 4 * g + e % 4;
      y[e] = (f16)((float)lds.k[t][16 * tile + c] * near_one(lds.rk[t]));
    }
    *(f16x8*)(keys + ((8 * KB + n) * 64 + lane) * 16) = y;
  }
  for (int h = 0; h < p.group; ++h) {
    const int head = hk * p.group + h, slot = h % kGateHeads;
    char* to = p.heads + ((long long)id * p.hv + head) * kDeltaHead;
    if (slot == 0) {
      __syncthreads();
      if (h + wave < p.group) {
        // a row a lane: sums in 64 bits, as differences of large ones are taken
        const int mine = head + wave;
        Gate gate = {0.0f, 0.0f};
        if (lane < live) gate = gate_of(p, span.first + t0 + lane, mine);
        double G = (double)gate.g * 1.4426950408889634;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          const double up = __shfl_up(G, off, 64);
          if (lane >= off) G += up;
        }
        lds.sums[wave][lane] = G;
        lds.beta[wave][lane] = gate.beta;
        float* f = (float*)(to + wave * (long long)kDeltaHead + kDeltaFactors) + lane;
        const bool in = lane < live;
        const float rk = lds.rk[lane], e = exp2_of(G), last = exp2_of(__shfl(G, 63, 64) - G);
        f[kBeta * kDeltaRows] = gate.beta;
        f[kSeen * kDeltaRows] = in ? gate.beta * e * rk : 0.0f;
        f[kAsk * kDeltaRows] = in ? p.scale * e * lds.rq[lane] : 0.0f;
        f[kLeft * kDeltaRows] = in ? last * (rk / near_one(rk)) : 0.0f;
        if (lane == 63) f[kDecay * kDeltaRows - 63] = e;
      }
      __syncthreads();
    }
    // (so that comparisons with the lane's row are made here, not kept over the loop)
    int here = c;
    asm volatile("" : "+v"(here));
    // A and P of the wave's rows
    const double G = lds.sums[slot][own];
    const float beta = lds.beta[slot][own];
    f32x4 a[4], own_tile = f32x4{};
    f16x4 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = f32x4{};
      w[j] = f16x4{};
      if (j > wave) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int ahead = 4 * g + r - here;  // of the wave's own tile: the column less the row
        const bool seen = own < live && (j < wave || ahead <= 0);
        const float e = exp2_of(G - lds.sums[slot][16 * j + 4 * g + r]);
        a[j][r] = seen && (j < wave || ahead < 0) ? ak[j][r] * (e * beta) : 0.0f;
        w[j][r] = (f16)(seen ? aq[j][r] * e * kPieceScale : 0.0f);
      }
      if (j == wave) own_tile = a[j];
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
      if (b <= wave / 2)
        *(f16x8*)(to + ((12 + piece_of(wave, b)) * 64 + lane) * 16) =
            __builtin_shufflevector(w[2 * b], w[2 * b + 1], 0, 1, 2, 3, 4, 5, 6, 7);
    // T's diagonal tiles by substitution, column c in lane c (the four rows of lanes do the
    // same): row i of A comes from lane i of each row of lanes
    *(f32x4*)&lds.t[own][16 * wave + 4 * g] = own_tile;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    {
      float x[16], t[16];
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 y = *(const f32x4*)&lds.t[own][16 * wave + i];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[i + r] = y[r];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      unrolled<16>([&](auto step) {
        constexpr int i = decltype(step)::value;
        float v = i == here ? 1.0f : 0.0f, u = 0.0f;
#pragma unroll
        for (int j = 0; j < i; ++j) {
          const float a = row_value<i>(x[j]);
          if (j % 2)
            u = fmaf(-a, t[j], u);
          else
            v = fmaf(-a, t[j], v);
        }
        t[i] = v + u;
        asm volatile("" : "+v"(t[i]));  // (computed here, not where it is stored)
      });
#pragma unroll
      for (int i = 0; i < 16; i += 4) {  // every row of lanes stores every fourth one
        const float y = g & 2 ? (g & 1 ? t[i + 3] : t[i + 2]) : (g & 1 ? t[i + 1] : t[i]);
        lds.t[16 * wave + i + g][16 * wave + c] = y;
      }
    }
    __syncthreads();
    // the tiles below them: T_wj = -T_ww sum_l A_wl T_lj, step k of a product taking row
    // 4 g + k of its right operand
    const f32x4 diagonal = *(const f32x4*)&lds.t[own][16 * wave + 4 * g];
#pragma unroll
    for (int d = 1; d < 4; ++d) {
      const int j = wave - d;
      if (j >= 0) {
        f32x4 x = f32x4{}, y = f32x4{};
#pragma unroll
        for (int l = 0; l < 3; ++l) {
          if (l < j || l >= wave) continue;
#pragma unroll
          for (int s = 0; s < 4; ++s)
            x = __builtin_amdgcn_mfma_f32_16x16x4f32(
                a[l][s], lds.t[16 * l + 4 * g + s][16 * j + c], x, 0, 0, 0);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s)
          y = __builtin_amdgcn_mfma_f32_16x16x4f32(diagonal[s], x[s], y, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) lds.t[16 * wave + 4 * g + r][16 * j + c] = -y[r];
      }
      __syncthreads();
    }
    // the wave's rows of T as the products take them
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (b > wave / 2) continue;
      const int piece = piece_of(wave, b);
      f16x8 t0, t1;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int tile = 2 * b + half;
        f32x4 v = f32x4{};
        if (tile <= wave) v = *(const f32x4*)&lds.t[own][16 * tile + 4 * g];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float y = v[r] * kPieceScale;
          t0[4 * half + r] = (f16)y;
          t1[4 * half + r] = (f16)(y - (float)t0[4 * half + r]);
        }
      }
      *(f16x8*)(to + ((piece * 2) * 64 + lane) * 16) = t0;
      *(f16x8*)(to + ((piece * 2 + 1) * 64 + lane) * 16) = t1;
    }
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

// Two fp16 numbers x0 + x1 for four values.
__device__ __forceinline__ void split4(const f32x4& x, f16x4& x0, f16x4& x1) {
  x0 = __builtin_convertvector(x, f16x4);
#pragma unroll
  for (int r = 0; r < 4; ++r) x1[r] = (f16)(x[r] - (float)x0[r]);
}
__device__ __forceinline__ float top4(const f32x4& v) {
  return fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
}

// Where a wave's values 4 g + r of a column go in a right operand of 32 rows, two fp16
// numbers to a value (`half`: which 16 rows).
__device__ __forceinline__ void put_split(f16x8* part0, f16x8* part1, int to, int half,
                                          const f32x4& x) {
  f16x4 x0, x1;
  split4(x, x0, x1);
  __builtin_memcpy((char*)(part0 + to) + 8 * half, &x0, 8);
  __builtin_memcpy((char*)(part1 + to) + 8 * half, &x1, 8);
}

// What the two halves of a workgroup have in common.
struct DeltaPlace {
  Span span;
  int part, head, hk, col, blocks, id0;
};
__device__ __forceinline__ __amdgpu_buffer_rsrc_t head_of(const DeltaParams& p,
                                                          const DeltaPlace& at, int b) {
  return __builtin_amdgcn_make_buffer_rsrc(
      p.heads + ((long long)(at.id0 + b) * p.hv + at.head) * kDeltaHead, 0, kDeltaHead,
      kBufferRsrcWord3);
}
template <int DK>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t keys_of(const DeltaParams& p,
                                                          const DeltaPlace& at, int b) {
  return __builtin_amdgcn_make_buffer_rsrc(
      p.keys + ((long long)(at.id0 + b) * p.hk + at.hk) * delta_key_bytes(DK), 0,
      delta_key_bytes(DK), kBufferRsrcWord3);
}
// Rows of v and out (x: the sequence's first) are addressed by resources that end with the
// block's last row: rows behind it read as zeros and are not stored, and a lane's offsets
// are the same in every block.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const DeltaPlace& at, const f16* x,
                                                          uint32_t step, int width, int b) {
  const int live = min(kDeltaRows, at.span.kept - b * kDeltaRows);
  return __builtin_amdgcn_make_buffer_rsrc((void*)(x + (long long)b * kDeltaRows * (step / 2)), 0,
                                           (uint32_t)(live - 1) * step + 2 * width,
                                           kBufferRsrcWord3);
}
__device__ __forceinline__ f32x4 factor_of(__amdgpu_buffer_rsrc_t head, int which, int row) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                       head, row * 4, kDeltaFactors + which * kDeltaRows * 4, 0));
}
__device__ __forceinline__ f16x8 piece_at(__amdgpu_buffer_rsrc_t at, int number) {
  const int lane = threadIdx.x & 63;
  return __builtin_bit_cast(
      f16x8, __builtin_amdgcn_raw_buffer_load_b128(at, lane * 16, number * 1024, 0));
}
// (a piece past the resource's end, where the wave's rows have no column in it)
__device__ __forceinline__ int needed(int wave, int b, int number) {
  return b <= wave / 2 ? number : 64;
}

// The first four waves: the state from block to block.  Wave w has 16 rows of each block
// and DK / 4 of the state.
template <int DK, int NC>
__device__ __forceinline__ void delta_chain(const DeltaParams& p, const DeltaPlace& at,
                                            DeltaLds<DK, NC>& lds) {
  constexpr int NT = DK / 64, KB = DK / 32;
  const int lane = threadIdx.x & 63, wave = sreg((int)threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4, rows4 = 16 * wave + 4 * g;
  const Span& span = at.span;
  DeltaState<DK, NC> S;
  float* state = p.state + ((long long)max(span.slot, 0) * p.hv + at.head) * DK * p.dv +
                 (wave * (DK / 4) + 4 * g) * p.dv + at.col + c;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        S.s[i][n][r] = span.fresh ? 0.0f : state[(16 * i + r) * p.dv + 16 * n];

  // Each operand of the next block is on its way as soon as the present one is used, and
  // not before (it takes the same registers), a few at a time.
  f16x8 k[KB], t[2][2], kt[NT][2];
  f32x4 beta, seen_by, left;
  f16 v[NC][4];
  float decay;
  const uint32_t step = 2 * (uint32_t)p.v_stride, at_v = (uint32_t)rows4 * step + 2 * c;
  const f16* v0 = sreg(p.v + span.first * p.v_stride + at.head * p.dv + at.col);
  auto load_k = [&](int b) {
    const auto keys = keys_of<DK>(p, at, b);
#pragma unroll
    for (int i = 0; i < KB; ++i) k[i] = piece_at(keys, wave * KB + i);
  };
  auto load_v = [&](int b) {
    const auto rows = rows_of(at, v0, step, 16 * NC, b), head = head_of(p, at, b);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int n = 0; n < NC; ++n)
        v[n][r] = __builtin_bit_cast(
            f16, __builtin_amdgcn_raw_buffer_load_b16(rows, at_v + r * step + 32 * n, 0, 0));
    beta = factor_of(head, kBeta, rows4);
    seen_by = factor_of(head, kSeen, rows4);
  };
  auto load_t = [&](int b) {
    const auto head = head_of(p, at, b);
    left = factor_of(head, kLeft, rows4);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int number = needed(wave, i, 2 * piece_of(wave, i));
      t[i][0] = piece_at(head, number);
      t[i][1] = piece_at(head, number + 1);
    }
  };
  auto load_kt = [&](int b) {
    const auto keys = keys_of<DK>(p, at, b);
    decay = as_f32(__builtin_amdgcn_raw_buffer_load_b32(
        head_of(p, at, b), 0, kDeltaFactors + kDecay * kDeltaRows * 4, 0));
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) kt[i][j] = piece_at(keys, 8 * KB + (wave * NT + i) * 2 + j);
  };
  auto state_top = [&](int n) {
    float m = top4(S.s[0][n]);
#pragma unroll
    for (int i = 1; i < NT; ++i) m = fmaxf(m, top4(S.s[i][n]));
    return rows_max(m);
  };
  load_k(0);
  __builtin_amdgcn_sched_barrier(0);  // (in the order in which they are waited for)
  load_v(0);
  __builtin_amdgcn_sched_barrier(0);
  load_t(0);
  __builtin_amdgcn_sched_barrier(0);
  load_kt(0);
  __builtin_amdgcn_sched_barrier(0);
  float bound[NC], top[NC];  // of |S| by column: at most, and in the wave's rows
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    top[n] = state_top(n);
    lds.first[n][c][wave] = top[n];  // (the four lanes of a column write the same)
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NC; ++n) bound[n] = top4(*(const f32x4*)lds.first[n][c]);

  // The first block in which something is not finite, and the state before it: a product
  // with zeros takes it to rows before it, so that from there on the blocks are passed a
  // second time, row after row.  (No way out of the loop: the waits of one that has another
  // end are those of its worst path.)
  int odd_block = at.blocks;
  DeltaState<DK, NC> before = S;
  for (int b = 0; b < at.blocks; ++b) {
    const int next = min(b + 1, at.blocks - 1);
    // S in two parts, where all waves read them
    Lift ls[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      ls[n] = lift_of(bound[n]);
      // rows 16 i + 4 g .. of the wave's are an even or odd half of a lane's eight
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int row = wave * (DK / 4) + 16 * i + 4 * g;
        put_split(lds.s[0][row / 32][n], lds.s[1][row / 32][n], c + row % 32 / 8 * 16, row / 4 % 2,
                  S.s[i][n] * ls[n].by);
      }
      lds.back_s[n][c] = ls[n].back;
      lds.top_s[n][c][wave] = top[n];
      f32x4 x;
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = (float)v[n][r];
      lds.top_v[n][c][wave] = rows_max(top4(x));
    }
    __syncthreads();
    // S^T k of the wave's 16 rows
    f32x4 seen[NC];
    float top_s[NC], top_v[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      f32x4 seen1 = f32x4{};
      seen[n] = f32x4{};
#pragma unroll
      for (int i = 0; i < KB; ++i) {
        seen[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[i], lds.s[0][i][n][lane], seen[n], 0, 0, 0);
        seen1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[i], lds.s[1][i][n][lane], seen1, 0, 0, 0);
      }
      top_s[n] = top4(*(const f32x4*)lds.top_s[n][c]);
      top_v[n] = top4(*(const f32x4*)lds.top_v[n][c]);
      seen[n] = (seen[n] + seen1) * ls[n].back;
    }
    __builtin_amdgcn_sched_barrier(0);
    load_k(next);
    __builtin_amdgcn_sched_barrier(0);
    // R in two parts; |R| is within |v| and the column's length
    Lift lr[NC];
    bool odd = false;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      lr[n] = lift_of(fmaf(top_s[n], 12.0f, top_v[n]));
      f32x4 x;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = beta[r] * (float)v[n][r] - seen_by[r] * seen[n][r];
        odd |= !(fabsf(x[r]) < INFINITY);
      }
      put_split(lds.r[0][wave / 2][n], lds.r[1][wave / 2][n], lane, wave & 1, x * lr[n].by);
      lds.top_r[n][c][wave] = rows_max(top4(x));
    }
    const bool any = __any(odd);
    if (lane == 0) lds.odd[wave] = any;
    __syncthreads();
    if (odd_block == at.blocks && sreg(lds.odd[0] | lds.odd[1] | lds.odd[2] | lds.odd[3])) {
      odd_block = b;
      before = S;
    }
    __builtin_amdgcn_sched_barrier(0);
    load_v(next);
    __builtin_amdgcn_sched_barrier(0);
    // U = T R of the wave's rows
    f32x4 u[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      f32x4 u1 = f32x4{}, u2 = f32x4{};
      u[n] = f32x4{};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i > wave / 2) continue;
        const f16x8 r0 = lds.r[0][i][n][lane], r1 = lds.r[1][i][n][lane];
        u[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(t[i][0], r0, u[n], 0, 0, 0);
        u1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(t[i][0], r1, u1, 0, 0, 0);
        u2 = __builtin_amdgcn_mfma_f32_16x16x32_f16(t[i][1], r0, u2, 0, 0, 0);
      }
      u[n] = (u[n] + (u1 + u2)) * (lr[n].back * (1.0f / kPieceScale));
    }
    // U times the rows' factors for the state, as it is for the outputs; |U| is within
    // 64 |R|
    Lift lu[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      lu[n] = lift_of(64.0f * top4(*(const f32x4*)lds.top_r[n][c]));
      const f32x4 y = u[n] * left;
      put_split(lds.u[2][wave / 2][n], lds.u[3][wave / 2][n], lane, wave & 1, y * lu[n].by);
      put_split(lds.u[0][wave / 2][n], lds.u[1][wave / 2][n], lane, wave & 1, u[n] * lu[n].by);
      lds.top_u[n][c][wave] = rows_max(top4(y));
    }
    __builtin_amdgcn_sched_barrier(0);
    load_t(next);
    __syncthreads();
    // the state behind the block
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      f32x4 add[NT][2];
#pragma unroll
      for (int i = 0; i < NT; ++i) add[i][0] = add[i][1] = f32x4{};
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const f16x8 z = lds.u[2 + x][j][n][lane];
#pragma unroll
          for (int i = 0; i < NT; ++i)
            add[i][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kt[i][j], z, add[i][x], 0, 0, 0);
        }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          S.s[i][n][r] = fmaf(S.s[i][n][r], decay, (add[i][0][r] + add[i][1][r]) * lu[n].back);
      bound[n] = fmaf(128.0f, top4(*(const f32x4*)lds.top_u[n][c]), top_s[n] * decay);
      top[n] = state_top(n);
    }
    // (what the old operands are for is done before the new ones take their registers)
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      asm volatile("" : "+v"(bound[n]));
#pragma unroll
      for (int i = 0; i < NT; ++i) asm volatile("" : "+v"(S.s[i][n]));
    }
    __builtin_amdgcn_sched_barrier(0);
    load_kt(next);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (odd_block < at.blocks) {
    S = before;
    __syncthreads();  // the rows' first outputs are in place before the second ones
    delta_rows<DK, NC>(p, span, at.head, at.col, odd_block * kDeltaRows, span.kept, S, lds);
  }
  if (!p.slots.store || span.slot < 0) return;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) state[(16 * i + r) * p.dv + 16 * n] = S.s[i][n][r];
}

// The other four: the outputs, from the parts of S and U that the first four leave in LDS.
template <int DK, int NC>
__device__ __forceinline__ void delta_outputs(const DeltaParams& p, const DeltaPlace& at,
                                              DeltaLds<DK, NC>& lds) {
  constexpr int KB = DK / 32;
  const int lane = threadIdx.x & 63, wave = sreg((int)threadIdx.x >> 6) - kWaves;
  const int c = lane & 15, g = lane >> 4, rows4 = 16 * wave + 4 * g;
  const Span& span = at.span;
  f16x8 q[KB], w[2];
  f32x4 ask;
  const uint32_t step = 2 * (uint32_t)p.out_stride, at_out = (uint32_t)rows4 * step + 2 * c;
  const f16* out0 = sreg(p.out + span.first * p.out_stride + at.head * p.dv + at.col);
  auto load_q = [&](int b) {
    const auto keys = keys_of<DK>(p, at, b);
#pragma unroll
    for (int i = 0; i < KB; ++i) q[i] = piece_at(keys, 4 * KB + wave * KB + i);
  };
  auto load_w = [&](int b) {
    const auto head = head_of(p, at, b);
    ask = factor_of(head, kAsk, rows4);
#pragma unroll
    for (int i = 0; i < 2; ++i) w[i] = piece_at(head, needed(wave, i, 12 + piece_of(wave, i)));
  };
  // What a block takes comes from memory, later than a block takes to pass: a byte of each
  // of its 128-byte lines is read two blocks ahead, a line a lane over the head's
  // workgroups, so that the loads find them in the L2 that these share.
  constexpr int kAhead = 2, key_lines = delta_key_bytes(DK) / 128;
  constexpr int head_lines = (kDeltaHead + 127) / 128;
  const int row_lines = p.dv / 64;  // of v
  const int line = (at.part * kWaves + wave) * 64 + lane, v_line = line - key_lines - head_lines;
  const char* warm = p.heads + ((long long)at.id0 * p.hv + at.head) * kDeltaHead;
  long long warm_step = (long long)p.hv * kDeltaHead;
  if (line < key_lines) {
    warm = p.keys + ((long long)at.id0 * p.hk + at.hk) * delta_key_bytes(DK) + line * 128;
    warm_step = (long long)p.hk * delta_key_bytes(DK);
  } else if (v_line < 0) {
    warm += (line - key_lines) * 128;
  } else if (v_line < min(kDeltaRows, span.kept) * row_lines) {
    warm = (const char*)(p.v + (span.first + v_line / row_lines) * p.v_stride + at.head * p.dv) +
           v_line % row_lines * 128;
    warm_step = kDeltaRows * p.v_stride * 2;
  }
  uint32_t warmed = 0;
  auto warm_up = [&](int b) {  // (but the last block, which may have fewer rows)
    asm volatile("" ::"v"(warmed));
    warmed = *(const __attribute__((address_space(1))) uint8_t*)(
        warm + max(min(b, at.blocks - 2), 0) * warm_step);
  };
  warm_up(1);
  load_q(0);
  __builtin_amdgcn_sched_barrier(0);
  load_w(0);
  __builtin_amdgcn_sched_barrier(0);
  __syncthreads();
  int odd_block = at.blocks;
  for (int b = 0; b < at.blocks; ++b) {
    const int next = min(b + 1, at.blocks - 1);
    warm_up(b + kAhead);
    __syncthreads();
    f32x4 asked[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      f32x4 asked1 = f32x4{};
      asked[n] = f32x4{};
#pragma unroll
      for (int i = 0; i < KB; ++i) {
        asked[n] =
            __builtin_amdgcn_mfma_f32_16x16x32_f16(q[i], lds.s[0][i][n][lane], asked[n], 0, 0, 0);
        asked1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(q[i], lds.s[1][i][n][lane], asked1, 0, 0, 0);
      }
      const float back = lds.back_s[n][c];
#pragma unroll
      for (int r = 0; r < 4; ++r) asked[n][r] = ask[r] * ((asked[n][r] + asked1[r]) * back);
      asm volatile("" : "+v"(asked[n]));
    }
    __builtin_amdgcn_sched_barrier(0);
    load_q(next);
    __builtin_amdgcn_sched_barrier(0);
    __syncthreads();
    if (odd_block == at.blocks && sreg(lds.odd[0] | lds.odd[1] | lds.odd[2] | lds.odd[3]))
      odd_block = b;
    float back[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n)
      back[n] = p.scale * (1.0f / kPieceScale) *
                lift_of(64.0f * top4(*(const f32x4*)lds.top_r[n][c])).back;
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      f32x4 o[2];
      o[0] = o[1] = f32x4{};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (j > wave / 2) continue;
#pragma unroll
        for (int x = 0; x < 2; ++x)
          o[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[j], lds.u[x][j][n][lane], o[x], 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) asked[n][r] = fmaf(o[0][r] + o[1][r], back[n], asked[n][r]);
      asm volatile("" : "+v"(asked[n]));
    }
    __builtin_amdgcn_sched_barrier(0);
    load_w(next);
    __builtin_amdgcn_sched_barrier(0);
    if (p.out) {
      const auto to = rows_of(at, out0, step, 16 * NC, b);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int n = 0; n < NC; ++n)
          __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, (f16)asked[n][r]), to,
                                                at_out + r * step + 32 * n, 0, 0);
    }
  }
  if (odd_block == at.blocks) return;
  // (the others' second pass, a barrier a row)
  wait_vm<0>();
  __syncthreads();
  for (int t = odd_block * kDeltaRows; t < span.kept; ++t) __syncthreads();
}

template <int DK, int NC>
__global__ __launch_bounds__(2 * kThreads, 2) void delta_prompt_kernel(const DeltaParams p) {
  __shared__ DeltaLds<DK, NC> lds;
  // the parts of one head lie on one XCD (workgroup b runs on XCD b % 8): they read the
  // same rows and pieces
  const int parts = p.dv / (16 * NC), unit = blockIdx.x / (8 * parts) * 8 + blockIdx.x % 8;
  if (unit >= p.slots.n * p.hv) return;
  DeltaPlace at;
  at.part = blockIdx.x / 8 % parts;
  at.head = unit % p.hv;
  at.hk = at.head / p.group;
  at.col = at.part * 16 * NC;
  const int s = unit / p.hv;
  at.span = span_of(p.slots, p.offsets, p.tokens, s);
  if (!at.span.kept) return;
  at.blocks = sreg((at.span.kept + kDeltaRows - 1) / kDeltaRows);
  at.id0 = at.span.first / kDeltaRows + s;
  if (sreg((int)threadIdx.x >> 6) < kWaves)
    delta_chain<DK, NC>(p, at, lds);
  else
    delta_outputs<DK, NC>(p, at, lds);
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
                     dim3(2 * kThreads), 0, stream, p);
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
