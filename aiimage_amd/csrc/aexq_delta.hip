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
struct GateInputs {
  f16 a, b;
  float dt_bias, a_log;
  __device__ __forceinline__ Gate gate() const {
    const float t = (float)a + dt_bias;
    // below -30 the softplus is e^t up to 2^-44 of it and goes into the rate's exponent:
    // e^a_log may be past fp32 where their product is not (above, both are past 1e5)
    const bool far = t < -30.0f;
    const float soft = far ? 1.0f : fmaxf(t, 0.0f) + log1pf(expf(-fabsf(t)));
    const float g = -expf(far ? a_log + t : a_log) * soft;
    return Gate{g < -1e5f ? -1e5f : g, 1.0f / (1.0f + expf(-(float)b))};
  }
};
__device__ __forceinline__ GateInputs gate_inputs(const DeltaParams& p, long long row, int head) {
  return GateInputs{p.a[row * p.a_stride + head], p.b[row * p.b_stride + head], p.dt_bias[head],
                    p.a_log[head]};
}
__device__ __forceinline__ Gate gate_of(const DeltaParams& p, long long row, int head) {
  return gate_inputs(p, row, head).gate();
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
// (maxima here are NaN where a value is)
__device__ __forceinline__ float rows_max(float v) {
  return rows_join(v, [](float x, float y) { return __builtin_elementwise_maximum(x, y); });
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
// are, their lengths put into the rows' factors; S, T, P, R and U are split into two fp16
// numbers, x = x0 + x1, scaled by powers of two so that neither part leaves fp16's range:
// up to 2^-22 of x, and where x1 is too small for that (x below 2^-16 of the largest of its
// column in the block) up to 2^-38 of that one; of T and P, which are at most 1, 2^-36.  (P in one part, 2^-11 of it, takes outputs half as far again from
// the exact ones as their own rounding does.)
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

// Row of S that row m of tile i of a state in registers is: a lane's rows of a pair of
// tiles are eight in a row, as the products take them of k and q.
__device__ __forceinline__ int state_row(int tile, int m) {
  return tile / 2 * 32 + m / 4 * 8 + tile % 2 * 4 + m % 4;
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

// Eight values as two fp16 numbers x0 + x1 each.
struct Split {
  f16x8 x0, x1;
};
__device__ __forceinline__ Split split8(const f32x4& a, const f32x4& b) {
  const f16x4 a0 = __builtin_convertvector(a, f16x4), b0 = __builtin_convertvector(b, f16x4);
  f16x4 a1, b1;
  float one = 1.0f;  // (a product that is seen as one: v_fma_mix takes x0 as it is, and rounds)
  asm("" : "+s"(one));
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    a1[r] = (f16)fmaf(a[r], one, -(float)a0[r]);
    b1[r] = (f16)fmaf(b[r], one, -(float)b0[r]);
  }
  return Split{__builtin_shufflevector(a0, b0, 0, 1, 2, 3, 4, 5, 6, 7),
               __builtin_shufflevector(a1, b1, 0, 1, 2, 3, 4, 5, 6, 7)};
}

constexpr int kGateHeads = kWaves;  // heads whose gates are made together, a wave each
template <int DK>
struct BlockLds {
  alignas(16) f16 k[kDeltaRows][DK + 8];
  alignas(16) float t[kDeltaRows][kDeltaRows + 4];
  alignas(32) double sums[kGateHeads][kDeltaRows];  // of log2 of the decays, up to each row
  float beta[kGateHeads][kDeltaRows], rk[kDeltaRows], rq[kDeltaRows];
};

// One block and key head; the value heads of its group in turn.  Products of keys are
// formed with the earlier rows on the left: lane (c, g) then has row 16 w + c and columns
// 16 j + 4 g + r, which is how A and P enter the products behind.
//
// Bound by memory: a block reads 32 KB of k and q (heads of 128) and writes 48 KB of them
// in the products' order and 25 KB of T, P and factors for each value head.  16384 rows of
// 16 key and 32 value heads: 97 us for 560 MB (a copy of that size runs at 5.3 TB/s).
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
  // a block of up to 16 rows has one row tile, its first wave's; the others only share in
  // the transposed keys
  const bool small = live <= kDeltaEnd;
  // gates of the first heads, a wave each, a row a lane
  auto gates_from = [&](int h) {
    return gate_inputs(p, span.first + t0 + min(lane, live - 1),
                       hk * p.group + min(h + wave, p.group - 1));
  };
  GateInputs gates = gates_from(0);
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
    if (!small || wave == 0) {
      *(f16x8*)(keys + ((wave * KB + i) * 64 + lane) * 16) = k[i];
      *(f16x8*)(keys + ((4 * KB + wave * KB + i) * 64 + lane) * 16) = q[i];
    }
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
  // Sums of the decays and the rows' factors of heads h .., a wave each, a row a lane: sums
  // in 64 bits, as differences of large ones are taken
  auto pass_gates = [&](int h) {
    if (h + wave >= p.group) return;
    Gate gate = gates.gate();
    const bool in = lane < live;
    if (!in) gate = Gate{0.0f, 0.0f};
    const double G = wave_scan((double)gate.g * 1.4426950408889634);
    lds.sums[wave][lane] = G;
    lds.beta[wave][lane] = gate.beta;
    const long long head = (long long)id * p.hv + hk * p.group + h + wave;
    float* f = (float*)(p.heads + head * kDeltaHead + kDeltaFactors) + lane;
    const float rk = lds.rk[lane], e = exp2_of(G), last = exp2_of(last_lane(G) - G);
    f[kBeta * kDeltaRows] = gate.beta;
    f[kSeen * kDeltaRows] = in ? gate.beta * e * rk : 0.0f;
    f[kAsk * kDeltaRows] = in ? p.scale * e * lds.rq[lane] : 0.0f;
    f[kLeft * kDeltaRows] = in ? last * (rk / near_one(rk)) : 0.0f;
    if (lane == 63) f[kDecay * kDeltaRows - 63] = e;
  };
  pass_gates(0);  // (the first waves, which have the fewest tiles below)
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
      // (one length at a time: of two rows of zeros their product, 1 / eps, may be past fp32)
      ak[j][r] = own < live ? ak[j][r] * rk * rj[r] : 0.0f;
      aq[j][r] = own < live ? aq[j][r] * rq * rj[r] : 0.0f;
    }
  }
  // the keys transposed, times a power of two (exact but for values below 2^-14, by 2^-25)
#pragma unroll
  for (int i = 0; i < DK / 32; ++i) {  // pieces (16 of DK, 32 rows): two a tile
    const int n = wave * (DK / 32) + i, tile = n >> 1, b = n & 1;
    if (small && b) continue;
    f16x8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int t = 32 * b + (e < 4 ? 0 : 16) + 4 * g + e % 4;
      y[e] = (f16)((float)lds.k[t][state_row(tile, c)] * near_one(lds.rk[t]));
    }
    *(f16x8*)(keys + ((8 * KB + n) * 64 + lane) * 16) = y;
  }
  for (int h = 0; h < p.group; ++h) {
    const int head = hk * p.group + h, slot = h % kGateHeads;
    char* to = p.heads + ((long long)id * p.hv + head) * kDeltaHead;
    if (slot == 0) {
      __syncthreads();
      if (h) {
        gates = gates_from(h);
        pass_gates(h);
        __syncthreads();
      }
    }
    if (small && wave) continue;
    // (so that comparisons with the lane's row are made here, not kept over the loop)
    int here = c;
    asm volatile("" : "+v"(here));
    // A and P of the wave's rows
    const double G = lds.sums[slot][own];
    const float beta = lds.beta[slot][own];
    f32x4 a[4], w[4], own_tile = f32x4{};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = f32x4{};
      w[j] = f32x4{};
      if (j > wave) continue;
      // columns up to the lane's row; of the tiles before the wave's own, all
      const int upto = j < wave ? 16 : here - 4 * g;
      typedef double f64x4 __attribute__((ext_vector_type(4)));
      const f64x4 Gj = *(const f64x4*)&lds.sums[slot][16 * j + 4 * g];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = exp2_of(G - Gj[r]);
        const float x = ak[j][r] * (e * beta), y = aq[j][r] * (e * kPieceScale);
        a[j][r] = r < upto ? x : 0.0f;
        w[j][r] = r <= upto ? y : 0.0f;
      }
      if (j == wave) own_tile = a[j];
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
      if (b <= wave / 2) {
        const Split x = split8(w[2 * b], w[2 * b + 1]);
        *(f16x8*)(to + ((12 + piece_of(wave, b) * 2) * 64 + lane) * 16) = x.x0;
        *(f16x8*)(to + ((13 + piece_of(wave, b) * 2) * 64 + lane) * 16) = x.x1;
      }
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
    if (!small) __syncthreads();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
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
      if (!small) __syncthreads();
    }
    // the wave's rows of T as the products take them
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (b > wave / 2) continue;
      const int piece = piece_of(wave, b);
      f32x4 v[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int tile = 2 * b + half;
        v[half] = f32x4{};
        if (tile <= wave) v[half] = *(const f32x4*)&lds.t[own][16 * tile + 4 * g] * kPieceScale;
      }
      const Split x = split8(v[0], v[1]);
      *(f16x8*)(to + ((piece * 2) * 64 + lane) * 16) = x.x0;
      *(f16x8*)(to + ((piece * 2 + 1) * 64 + lane) * 16) = x.x1;
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
// The larger of m and the magnitudes of v.
__device__ __forceinline__ float top4(float m, const f32x4& v) {
#pragma unroll
  for (int r = 0; r < 4; r += 2)
    m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(m, fabsf(v[r])), fabsf(v[r + 1]));
  return m;
}
__device__ __forceinline__ f32x4 mfma(const f16x8& a, const f16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// The blocks of a sequence in turn.  A wave takes 16 columns of S of one value head, and
// nothing passes between waves: columns are independent of one another.  It holds them as
// a product's result (state_row), which is a product's right operand as it stands, and so
// are R and U; K, Q, T, P and the transposed keys come from scratch as left operands, each
// piece for the next block as soon as the present one is done with it.
//
// S is kept times a power of two, by column, that takes it to fp16's range; the parts of R
// and U have theirs, from their largest values.
// ---------------------------------------------------------------------------
template <int DK>
struct DeltaWave {
  static constexpr int KB = DK / 32;
  const DeltaParams& p;
  Span span;
  int head, hk, col, id0, lane, c, g;
  f32x4 S[2 * KB];  // times scale.by
  Lift scale;

  __device__ __forceinline__ DeltaWave(const DeltaParams& p) : p(p) {}

  __device__ __forceinline__ float* state_at(int tile) const {
    return p.state + ((long long)max(span.slot, 0) * p.hv + head) * DK * p.dv +
           (long long)state_row(tile, 4 * g) * p.dv + col + c;
  }
  __device__ __forceinline__ void rescale(float by) {
#pragma unroll
    for (int i = 0; i < 2 * KB; ++i) S[i] *= by;
  }
  __device__ __forceinline__ float top() const {
    float m = 0.0f, n = 0.0f;
#pragma unroll
    for (int i = 0; i < KB; ++i) {
      m = top4(m, S[2 * i]);
      n = top4(n, S[2 * i + 1]);
    }
    return rows_max(__builtin_elementwise_maximum(m, n));
  }
  __device__ __forceinline__ void read(f32x4 (&S)[2 * KB]) const {
#pragma unroll
    for (int i = 0; i < 2 * KB; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[i][r] = span.fresh ? 0.0f : state_at(i)[r * p.dv];
  }
  __device__ __forceinline__ void lift(float top) {
    scale = lift_of(top);
    rescale(scale.by);
  }
  __device__ __forceinline__ void write() {
    if (!p.slots.store || span.slot < 0) return;
    rescale(scale.back);
#pragma unroll
    for (int i = 0; i < 2 * KB; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) state_at(i)[r * p.dv] = S[i][r];
  }

  // Outputs of rows [t0, t1) row after row from the state `S` before them, of the lanes'
  // columns that are to be `taken`.
  __device__ __forceinline__ void rows(f32x4 (&S)[2 * KB], int t0, int t1, bool taken) const {
    if (!p.out) return;
    taken &= g == 0;
    for (int t = t0; t < t1; ++t) {
      const long long row = span.first + t;
      const f16* kr = p.k + row * p.k_stride + hk * DK + 8 * g;
      const f16* qr = p.q + row * p.q_stride + hk * DK + 8 * g;
      const Gate gate = gate_of(p, row, head);
      const float decay = expf(gate.g);
      float k[2 * KB][4], kk = 0.0f, qq = 0.0f, kq = 0.0f, sk = 0.0f, sq = 0.0f;
#pragma unroll
      for (int i = 0; i < KB; ++i) {
        const f16x8 ki = *(const f16x8*)(kr + 32 * i), qi = *(const f16x8*)(qr + 32 * i);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = (float)ki[e], y = (float)qi[e];
          const float s = S[2 * i + e / 4][e % 4] * decay;
          S[2 * i + e / 4][e % 4] = s;
          k[2 * i + e / 4][e % 4] = x;
          kk = fmaf(x, x, kk);
          qq = fmaf(y, y, qq);
          kq = fmaf(x, y, kq);
          sk = fmaf(s, x, sk);
          sq = fmaf(s, y, sq);
        }
      }
      const float rk = 1.0f / sqrtf(rows_sum(kk) + p.eps), rq = 1.0f / sqrtf(rows_sum(qq) + p.eps);
      const float v = (float)p.v[row * p.v_stride + head * p.dv + col + c];
      const float u = gate.beta * (v - rk * rows_sum(sk));
      const float o = p.scale * rq * fmaf(u, rk * rows_sum(kq), rows_sum(sq));
#pragma unroll
      for (int i = 0; i < 2 * KB; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[i][r] = fmaf(k[i][r] * rk, u, S[i][r]);
      if (taken) p.out[row * p.out_stride + head * p.dv + col + c] = (f16)o;
    }
  }

  // ---- what a block takes
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t head_of(int b) const {
    return __builtin_amdgcn_make_buffer_rsrc(
        p.heads + ((long long)(id0 + b) * p.hv + head) * kDeltaHead, 0, kDeltaHead,
        kBufferRsrcWord3);
  }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t keys_of(int b) const {
    return __builtin_amdgcn_make_buffer_rsrc(
        p.keys + ((long long)(id0 + b) * p.hk + hk) * delta_key_bytes(DK), 0, delta_key_bytes(DK),
        kBufferRsrcWord3);
  }
  // Rows of v and out are addressed by resources that end with the block's last row: rows
  // behind it read as zeros and are not stored, nor is any where there is no out, and a
  // lane's offsets are the same in every block.
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const f16* x, long long stride,
                                                            int b) const {
    const int live = min(kDeltaRows, span.kept - b * kDeltaRows);
    return __builtin_amdgcn_make_buffer_rsrc(
        (void*)(x + (span.first + (long long)b * kDeltaRows) * stride + head * p.dv + col), 0,
        x ? 2 * ((uint32_t)(live - 1) * (uint32_t)stride + 16) : 0, kBufferRsrcWord3);
  }
  __device__ __forceinline__ f16x8 piece(__amdgpu_buffer_rsrc_t at, int number) const {
    return __builtin_bit_cast(
        f16x8, __builtin_amdgcn_raw_buffer_load_b128(at, lane * 16, number * 1024, 0));
  }
  __device__ __forceinline__ f32x4 factor(__amdgpu_buffer_rsrc_t at, int which, int tile) const {
    return __builtin_bit_cast(
        f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                   at, 16 * g, kDeltaFactors + (which * kDeltaRows + 16 * tile) * 4, 0));
  }
  __device__ __forceinline__ float decay_of(__amdgpu_buffer_rsrc_t at) const {
    return as_f32(
        __builtin_amdgcn_raw_buffer_load_b32(at, 0, kDeltaFactors + kDecay * kDeltaRows * 4, 0));
  }
};

// The last block of a sequence, of up to 16 rows: the outputs, and the state behind it.
// True in the lanes of a column that stops being finite in this block: a product with zeros
// takes that to the rows before it.  `first`: the state is as it was read.
template <int DK>
__device__ __forceinline__ bool delta_end(DeltaWave<DK>& x, int b, bool first) {
  constexpr int KB = DK / 32;
  const DeltaParams& p = x.p;
  const auto keys = x.keys_of(b), head = x.head_of(b);
  f16x8 k[KB], q[KB], kt[2 * KB];
  f16 v[4];
#pragma unroll
  for (int i = 0; i < KB; ++i) k[i] = x.piece(keys, i);
  {
    const auto from = x.rows_of(p.v, p.v_stride, b);
    const uint32_t step = 2 * (uint32_t)p.v_stride, at = 4 * x.g * step + 2 * x.c;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[e] = __builtin_bit_cast(
          f16, __builtin_amdgcn_raw_buffer_load_b16(from, at + e * step, 0, 0));
  }
  const f32x4 beta = x.factor(head, kBeta, 0), seen_by = x.factor(head, kSeen, 0);
#pragma unroll
  for (int i = 0; i < KB; ++i) q[i] = x.piece(keys, 4 * KB + i);
  const f16x8 t0 = x.piece(head, 0), t1 = x.piece(head, 1);
  const f16x8 w0 = x.piece(head, 12), w1 = x.piece(head, 13);
  const f32x4 left = x.factor(head, kLeft, 0), ask = x.factor(head, kAsk, 0);
#pragma unroll
  for (int i = 0; i < 2 * KB; ++i) kt[i] = x.piece(keys, 8 * KB + 2 * i);
  const float decay = x.decay_of(head);
  __builtin_amdgcn_sched_barrier(0);  // (all of it on its way together, behind the state)
  if (first) x.lift(x.top());
  f32x4 seen = f32x4{}, asked = f32x4{};
#pragma unroll
  for (int i = 0; i < KB; ++i) {
    const Split s = split8(x.S[2 * i], x.S[2 * i + 1]);
    seen = mfma(k[i], s.x0, seen);
    asked = mfma(q[i], s.x0, asked);
    seen = mfma(k[i], s.x1, seen);
    asked = mfma(q[i], s.x1, asked);
  }
  f32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    r[e] = fmaf(-seen_by[e], seen[e] * x.scale.back, beta[e] * (float)v[e]);
  const float m = rows_max(top4(0.0f, r));
  const Lift lr = lift_of(m);
  const Split rs = split8(r * lr.by, f32x4{});
  f32x4 u = mfma(t0, rs.x0, f32x4{});
  u = mfma(t0, rs.x1, u);
  u = mfma(t1, rs.x0, u);
  u *= lr.back * (1.0f / kPieceScale);
  // S is within its decayed columns and 16 of U's, the new scale within that of 64
  const f32x4 y = u * left;
  const float top = x.top();
  const bool bad = !(m < INFINITY) && top < INFINITY;
  const Lift lu = lift_of(rows_max(top4(0.0f, u)));
  const Lift ls = lift_of(fmaf(64.0f, rows_max(top4(0.0f, y)), top * (x.scale.back * decay)));
  const Split us = split8(u * lu.by, f32x4{}), ys = split8(y * ls.by, f32x4{});
  const float back_s = x.scale.back;
  x.rescale(decay * back_s * ls.by);
  x.scale = ls;
#pragma unroll
  for (int i = 0; i < 2 * KB; ++i) {
    x.S[i] = mfma(kt[i], ys.x0, x.S[i]);
    x.S[i] = mfma(kt[i], ys.x1, x.S[i]);
  }
  f32x4 a = mfma(w0, us.x0, f32x4{});
  a = mfma(w0, us.x1, a);
  a = mfma(w1, us.x0, a);
  const float back = p.scale * lu.back * (1.0f / kPieceScale);
  if (p.out) {
    const auto to = x.rows_of(p.out, p.out_stride, b);
    const uint32_t step = 2 * (uint32_t)p.out_stride, at = 4 * x.g * step + 2 * x.c;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      __builtin_amdgcn_raw_buffer_store_b16(
          __builtin_bit_cast(short, (f16)fmaf(a[e], back, ask[e] * (asked[e] * back_s))), to,
          at + e * step, 0, 0);
  }
  return bad;
}

// ---------------------------------------------------------------------------
// Blocks of more than 16 rows go through two waves: one passes the state from block to
// block, the other forms the outputs a block behind, from the parts of S and from U that
// the first one leaves in LDS, and the first one's beta v a block ahead.  One barrier a
// block.
//
// A block takes the first wave 1.8 us: 82 matrix products (1300 cycles), 300 vector
// operations, which hide behind them in part, and 45 loads, each of which holds it up for
// 20 to 30 cycles, all in one chain from state to state.  16384 rows of 32 value heads of
// 128 x 128, one sequence: 462 us, 256 blocks in turn; 6657 rows of 12 sequences and 16
// heads: 83 us.  Steps on the way, in that order: one wave for all of it 777 and 112 us;
// eight waves that each hold 16 rows of S of 16 columns and add their products through
// LDS: 450 and 103 (but 77 for blocks of 16 rows, where the last ones now go through one
// wave in 35); two waves, each waiting for its own loads: 510 and 97; waits of the second
// one that leave later loads on their way, keys a block ahead, LDS reads ahead of their
// use: 478 and 85; parts of S and loads between the products of a step: 462 and 83.
// ---------------------------------------------------------------------------
template <int DK>
struct DeltaLds {
  static constexpr int kPitch = 24;  // of 16 columns: no two rows of a read share banks
  f16x8 s[2][DK / 32][2][64];        // by the block's parity: parts of S
  f32x4 u[2][4][64], v[2][4][64];
  f32x4 factors[2][kDecay * kDeltaRows / 4];
  float back_s[2][64], back_u[2][64];  // what S and U are to be multiplied by
  alignas(16) f16 rows[kDeltaRows][kPitch];  // of v, then of the outputs: the second wave's
  int stop;  // block behind which the first wave stops (delta_solve)
  // Factors of rows 16 tile + 4 g ..
  __device__ __forceinline__ f32x4 factor(int at, int which, int tile, int g) const {
    return factors[at][(which * kDeltaRows + 16 * tile) / 4 + g];
  }
};

// Kinds of instructions that places in a schedule are kept for.
enum : int { kSchedValu = 0x2, kSchedMfma = 0x8, kSchedLoad = 0x20, kSchedLds = 0x300 };

// The state from block b0 on.  Stops behind a block in which a column stops being finite:
// its lanes are in `bad`, those of all that are not in `dead`.  Returns the block to go on
// with.
template <int DK>
__device__ __forceinline__ int delta_solve(DeltaWave<DK>& x, DeltaLds<DK>& lds, int b0, int blocks,
                                           uint64_t& dead, uint64_t& bad) {
  constexpr int KB = DK / 32;
  const int lane = x.lane;
  // Each operand is on its way as soon as the one before it in its registers is used, and
  // not earlier; the keys and the transposed keys take turns in `a`, but for the first
  // kEarly keys, which a block begins with and which would come too late so.
  constexpr int kEarly = 8;
  f16x8 a[4 * KB], begin[kEarly], t[4][2][2];
  f32x4 seen_by[4], left[4];
  float decay;
  auto load_k = [&](__amdgpu_buffer_rsrc_t at, int n) {
    (n < kEarly ? begin[n] : a[n]) = x.piece(at, n % 4 * KB + n / 4);
  };
  auto load_kt = [&](__amdgpu_buffer_rsrc_t at, int n) {
    a[n] = x.piece(at, 8 * KB + 2 * (n % (2 * KB)) + n / (2 * KB));
  };
  auto load_t = [&](__amdgpu_buffer_rsrc_t h) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int w = 2 * j; w < 4; ++w)
#pragma unroll
        for (int i = 0; i < 2; ++i) t[w][j][i] = x.piece(h, piece_of(w, j) * 2 + i);
  };
  {
    const auto keys = x.keys_of(b0), head = x.head_of(b0);
#pragma unroll
    for (int n = 0; n < kEarly; ++n) load_k(keys, n);
    __builtin_amdgcn_sched_barrier(0);  // (in the loop's order)
    load_t(head);
    __builtin_amdgcn_sched_barrier(0);
    decay = x.decay_of(head);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = kEarly; n < 4 * KB; ++n) load_k(keys, n);
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();  // the first block's v and factors
  for (int b = b0; b < blocks; ++b) {
    const int next = min(b + 1, blocks - 1), at = b & 1;
    const auto keys = x.keys_of(b), after = x.keys_of(next);
    f32x4 seen[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      seen[w] = f32x4{};
      seen_by[w] = lds.factor(at, kSeen, w, x.g);
    }
    f32x4 v[4];
    // (between a step's products: the parts of S for the next one, and loads into the
    // registers that it is done with)
    Split s = split8(x.S[0], x.S[1]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < KB; ++i) {
      Split then = s;
      if (i + 1 < KB) then = split8(x.S[2 * i + 2], x.S[2 * i + 3]);
      if (i == KB - 1)
#pragma unroll
        for (int w = 0; w < 4; ++w) v[w] = lds.v[at][w][lane];
      lds.s[at][i][0][lane] = s.x0;
      lds.s[at][i][1][lane] = s.x1;
      const f16x8* const k = 4 * i < kEarly ? begin : a;
#pragma unroll
      for (int w = 0; w < 4; ++w) seen[w] = mfma(k[4 * i + w], s.x0, seen[w]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        seen[w] = mfma(k[4 * i + w], s.x1, seen[w]);
        load_kt(keys, 4 * i + w);
        if (4 * i < kEarly) load_k(after, 4 * i + w);
      }
      s = then;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedValu | kSchedLds, 3, 0);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedLoad, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedValu | kSchedLds, 1, 0);
        if (4 * i < kEarly) __builtin_amdgcn_sched_group_barrier(kSchedLoad, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // R, times what takes its largest value to fp16's range
    f32x4 r[4];
    float m = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        r[w][e] = fmaf(-seen_by[w][e], seen[w][e] * x.scale.back, v[w][e]);
      m = top4(m, r[w]);
    }
    m = rows_max(m);
    const uint64_t odd = __ballot(!(m < INFINITY));
    bad = odd & ~dead;
    dead = odd;
    lds.stop = bad ? b : -1;
    const float top_s = x.top() * x.scale.back;
    lds.back_s[at][lane] = x.scale.back;
    const Lift lr = lift_of(m);
    Split rs[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) rs[j] = split8(r[2 * j] * lr.by, r[2 * j + 1] * lr.by);
    const auto head = x.head_of(next);
#pragma unroll
    for (int w = 0; w < 4; ++w) left[w] = lds.factor(at, kLeft, w, x.g);
    __builtin_amdgcn_sched_barrier(0);
    // U = T R
    f32x4 u[4], y[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) u[w] = f32x4{};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int w = 2 * j; w < 4; ++w) u[w] = mfma(t[w][j][0], rs[j].x0, u[w]);
#pragma unroll
      for (int w = 2 * j; w < 4; ++w) u[w] = mfma(t[w][j][0], rs[j].x1, u[w]);
#pragma unroll
      for (int w = 2 * j; w < 4; ++w) u[w] = mfma(t[w][j][1], rs[j].x0, u[w]);
    }
    __builtin_amdgcn_sched_barrier(0);
    load_t(head);
    __builtin_amdgcn_sched_barrier(0);
    // U for the outputs, and times the rows' factors for the state, which stays within its
    // decayed columns and 64 of these
    const float back_u = lr.back * (1.0f / kPieceScale);
    float my = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      lds.u[at][w][lane] = u[w];
      y[w] = u[w] * left[w];
      my = top4(my, y[w]);
    }
    lds.back_u[at][lane] = back_u;
    const Lift ls = lift_of(fmaf(64.0f, rows_max(my) * back_u, top_s * decay));
    const float to_y = back_u * ls.by, keep = decay * x.scale.back * ls.by;
    Split ys[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) ys[j] = split8(y[2 * j] * to_y, y[2 * j + 1] * to_y);
    x.scale = ls;
#pragma unroll
    for (int i = 0; i < 4; ++i) x.S[i] *= keep;
    __builtin_amdgcn_sched_barrier(0);
    decay = x.decay_of(head);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 4 * KB; n += 4) {
      const int j = n / (2 * KB);
      if (n + 4 < 2 * KB)
#pragma unroll
        for (int i = n + 4; i < n + 8; ++i) x.S[i] *= keep;
#pragma unroll
      for (int i = n; i < n + 4; ++i) x.S[i % (2 * KB)] = mfma(a[i], ys[j].x0, x.S[i % (2 * KB)]);
#pragma unroll
      for (int i = n; i < n + 4; ++i) {
        x.S[i % (2 * KB)] = mfma(a[i], ys[j].x1, x.S[i % (2 * KB)]);
        if (n >= kEarly) load_k(after, i);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedValu, 3, 0);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
        if (n >= kEarly) __builtin_amdgcn_sched_group_barrier(kSchedLoad, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedValu, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    if (bad) return b + 1;
  }
  return blocks;
}

// Outputs from block b0 on, as far as the other wave goes; its return value.
template <int DK>
__device__ __forceinline__ int delta_outputs(DeltaWave<DK>& x, DeltaLds<DK>& lds, int b0, int blocks,
                                             bool& stop) {
  constexpr int KB = DK / 32;
  const DeltaParams& p = x.p;
  const int lane = x.lane;
  f16x8 q[4][KB], w[4][2][2];
  // v and the outputs move 16 bytes a lane, eight columns of row lane / 2 (and 32 more),
  // and change places in LDS: 16 loads or stores of two bytes a lane take a CU's address
  // unit as long as the operands' 16 of 16
  struct Rows {
    f16x8 v[2];
    f32x4 factors;
  } first, rows;
  const int row = lane / 2, part = lane % 2 * 8;
  const uint32_t step_v = 2 * (uint32_t)p.v_stride, step_out = 2 * (uint32_t)p.out_stride;
  auto load_v = [&](Rows& to, int b) {
    const auto from = x.rows_of(p.v, p.v_stride, b), head = x.head_of(b);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      to.v[i] = __builtin_bit_cast(f16x8, __builtin_amdgcn_raw_buffer_load_b128(
                                              from, row * step_v + 2 * part, 32 * i * step_v, 0));
    to.factors = __builtin_bit_cast(
        f32x4, __builtin_amdgcn_raw_buffer_load_b128(head, 16 * lane, kDeltaFactors, 0));
  };
  auto meet = [] {  // LDS written by one lane and read by another
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  auto put_v = [&](const Rows& from, int b) {
    lds.factors[b & 1][lane] = from.factors;
#pragma unroll
    for (int i = 0; i < 2; ++i) *(f16x8*)&lds.rows[32 * i + row][part] = from.v[i];
    meet();
    f16x4 y[4];
    f32x4 beta[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      beta[i] = lds.factor(b & 1, kBeta, i, x.g);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[i][e] = lds.rows[16 * i + 4 * x.g + e][x.c];
    }
    __builtin_amdgcn_sched_barrier(0);  // (all of it read before any of it is used)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      lds.v[b & 1][i][lane] = beta[i] * __builtin_convertvector(y[i], f32x4);
    meet();
  };
  auto load_q = [&](__amdgpu_buffer_rsrc_t keys, int i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j][i] = x.piece(keys, (4 + j) * KB + i);
  };
  auto load_w = [&](__amdgpu_buffer_rsrc_t head) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int j = 0; j <= i / 2; ++j)
#pragma unroll
        for (int part = 0; part < 2; ++part)
          w[i][j][part] = x.piece(head, 12 + piece_of(i, j) * 2 + part);
    }
  };
  // (in the loop's order: a wait for the rows at its top leaves what was asked for after
  // them on its way, which it does only if that holds on both ways there)
  load_v(first, b0);
  __builtin_amdgcn_sched_barrier(0);
  load_v(rows, min(b0 + 1, blocks - 1));
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < KB; ++i) load_q(x.keys_of(b0), i);
  __builtin_amdgcn_sched_barrier(0);
  load_w(x.head_of(b0));
  __builtin_amdgcn_sched_barrier(0);
  put_v(first, b0);
  __builtin_amdgcn_sched_barrier(0);
  __syncthreads();
  for (int b = b0; b < blocks; ++b) {
    const int next = min(b + 1, blocks - 1), at = b & 1;
    put_v(rows, b + 1);  // (behind the last block: of that one again, where nothing reads it)
    __builtin_amdgcn_sched_barrier(0);
    load_v(rows, min(b + 2, blocks - 1));
    __builtin_amdgcn_sched_barrier(0);
    __syncthreads();  // S and U of this block, v of the next
    const auto keys = x.keys_of(next);
    const int stops = lds.stop;
    f32x4 u[4], o[4], a[4];
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = lds.u[at][i][lane];
      m = top4(m, u[i]);
      a[i] = o[i] = f32x4{};
    }
    const Lift lu = lift_of(rows_max(m));
    Split us[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) us[j] = split8(u[2 * j] * lu.by, u[2 * j + 1] * lu.by);
#pragma unroll
    for (int i = 0; i < KB; ++i) {
      const f16x8 s0 = lds.s[at][i][0][lane], s1 = lds.s[at][i][1][lane];
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = mfma(q[j][i], s0, a[j]);
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = mfma(q[j][i], s1, a[j]);
      __builtin_amdgcn_sched_barrier(0);
      load_q(keys, i);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int i = 2 * j; i < 4; ++i) o[i] = mfma(w[i][j][0], us[j].x0, o[i]);
#pragma unroll
      for (int i = 2 * j; i < 4; ++i) o[i] = mfma(w[i][j][0], us[j].x1, o[i]);
#pragma unroll
      for (int i = 2 * j; i < 4; ++i) o[i] = mfma(w[i][j][1], us[j].x0, o[i]);
    }
    f32x4 ask[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ask[i] = lds.factor(at, kAsk, i, x.g);
    const float back_s = lds.back_s[at][lane];
    const float back = p.scale * lu.back * lds.back_u[at][lane] * (1.0f / kPieceScale);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = fmaf(o[i][e], back, ask[i][e] * (a[i][e] * back_s));
      asm volatile("" : "+v"(o[i]));  // (before the operands' registers are loaded again)
    }
    __builtin_amdgcn_sched_barrier(0);
    load_w(x.head_of(next));
    __builtin_amdgcn_sched_barrier(0);
    const auto to = x.rows_of(p.out, p.out_stride, b);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) lds.rows[16 * i + 4 * x.g + e][x.c] = (f16)o[i][e];
    meet();
#pragma unroll
    for (int i = 0; i < 2; ++i)
      __builtin_amdgcn_raw_buffer_store_b128(
          __builtin_bit_cast(u32x4, *(const f16x8*)&lds.rows[32 * i + row][part]), to,
          row * step_out + 2 * part, 32 * i * step_out, 0);
    meet();
    stop = sreg(stops) == b;
    if (stop) return b + 1;
  }
  return blocks;
}

// The parts of one head lie on one XCD (workgroup b runs on XCD b % 8): they read the same
// rows and pieces.  A sequence's place and head, and the part, of workgroup `id`.
struct DeltaPlace {
  int place, head, part;
};
__device__ __forceinline__ DeltaPlace place_of(const DeltaParams& p, int id) {
  const int parts = p.dv / 16, unit = id / (8 * parts) * 8 + id % 8;
  return DeltaPlace{unit / p.hv, unit % p.hv, id / 8 % parts};
}
template <int DK>
__device__ __forceinline__ void take_place(DeltaWave<DK>& x, int s, const DeltaPlace& at) {
  x.span = span_of(x.p.slots, x.p.offsets, x.p.tokens, s);
  x.head = at.head;
  x.hk = at.head / x.p.group;
  x.col = at.part * 16;
  x.id0 = x.span.first / kDeltaRows + s;
  x.lane = threadIdx.x & 63;
  x.c = x.lane & 15;
  x.g = x.lane >> 4;
}
// Outputs of rows [t0, t1), a block, of the columns that stop being finite in it, row after
// row from the state before it, over those of the block: its products have taken what is
// not finite to the column's rows before it as well.  They take it to no other column, and
// what lies behind it is not finite either way, so that a column has one such block at most
// and goes on in blocks.  16384 rows of 32 value heads of 128 x 128 with a NaN in a row of
// v take 0.77 ms, of 0.56 without.
template <int DK>
__device__ __forceinline__ void rows_again(const DeltaWave<DK>& x, f32x4 (&S)[2 * (DK / 32)], int t0,
                                           int t1, bool bad) {
  wait_vm<0>();
  // (the arguments from memory again, the kernels' only ones: kept over the blocks, they
  // cost them registers)
  auto* from = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(from));
  DeltaWave<DK> y(*(const DeltaParams*)from);
  y.span = x.span;
  y.head = x.head;
  y.hk = x.hk;
  y.col = x.col;
  y.c = x.c;
  y.g = x.g;
  y.rows(S, t0, t1, bad);
}

template <int DK>
__global__ __launch_bounds__(128, 2) void delta_prompt_kernel(const DeltaParams p) {
  __shared__ DeltaLds<DK> lds;
  const DeltaPlace at = place_of(p, blockIdx.x);
  if (at.place >= (p.longs ? p.longs[0] : p.slots.n)) return;
  DeltaWave<DK> x(p);
  take_place(x, p.longs ? p.longs[1 + at.place] : at.place, at);
  if (!x.span.kept) return;
  const int all = (x.span.kept + kDeltaRows - 1) / kDeltaRows;
  // a last block of up to 16 rows takes a quarter of the products, and one wave
  const bool short_end = x.span.kept - (all - 1) * kDeltaRows <= kDeltaEnd;
  const int blocks = sreg(all - short_end);
  if (sreg((int)threadIdx.x >> 6)) {
    for (int b = 0; b < blocks;) {
      bool stop = false;
      b = delta_outputs<DK>(x, lds, b, blocks, stop);
      if (stop) {
        wait_vm<0>();
        __syncthreads();
      }
    }
    return;
  }
  constexpr int kTiles = 2 * DeltaWave<DK>::KB;
  x.read(x.S);
  lds.stop = -1;
  uint64_t dead = 0;
  if (blocks) {
    const float top = x.top();
    dead = __ballot(!(top < INFINITY));
    x.lift(top);
  }
  for (int b = 0; b < blocks;) {
    uint64_t bad = 0;
    b = delta_solve<DK>(x, lds, b, blocks, dead, bad);
    if (bad) {
      __syncthreads();  // the block's outputs are in place
      const int at = (b - 1) & 1;
      const float back = lds.back_s[at][x.lane];
      f32x4 S[kTiles];
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        const f16x8 s0 = lds.s[at][i / 2][0][x.lane], s1 = lds.s[at][i / 2][1][x.lane];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int e = i % 2 * 4 + r;
          S[i][r] = ((float)s0[e] + (float)s1[e]) * back;
        }
      }
      rows_again(x, S, (b - 1) * kDeltaRows, min(b * kDeltaRows, x.span.kept),
                 bad >> x.lane & 1);
    }
  }
  if (short_end) {
    // (the state before it, where the other wave's last block has nothing)
    f32x4* const before = (f32x4*)lds.s[blocks & 1] + x.lane;
    const float back = blocks ? x.scale.back : 1.0f;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) before[64 * i] = x.S[i];
    const bool bad = delta_end<DK>(x, blocks, !blocks);
    if (__any(bad)) {
      f32x4 S[kTiles];
#pragma unroll
      for (int i = 0; i < kTiles; ++i) S[i] = before[64 * i] * back;
      rows_again(x, S, blocks * kDeltaRows, x.span.kept, bad);
    }
  }
  x.write();
}

// Calls of many short sequences: those of up to 16 rows, a wave a part and no LDS, which
// keeps three times as many on a CU (48 sequences of 2 to 8 rows, 16 heads of 128 x 128:
// 23.6 us, where the kernel above takes 35; 26.6 with two waves a SIMD, 41 with four and
// spilled registers).  One workgroup more lists the longer ones for that
// kernel, their number first.
template <int DK>
__global__ __launch_bounds__(64, 3) void delta_short_kernel(const DeltaParams p) {
  if (blockIdx.x == 0) {
    const int lane = threadIdx.x;
    auto rows_of = [&](int s) {
      return s < p.slots.n ? span_of(p.slots, p.offsets, p.tokens, s).kept : 0;
    };
    int n = 0, rows = rows_of(lane);
    for (int s = lane; s - lane < p.slots.n; s += 64) {
      const int next = rows_of(s + 64);
      const uint64_t at = __ballot(rows > kDeltaEnd);
      if (rows > kDeltaEnd) p.longs[1 + n + __popcll(at & ((1ull << lane) - 1))] = s;
      n += (int)__popcll(at);
      rows = next;
    }
    if (lane == 0) p.longs[0] = n;
    return;
  }
  const DeltaPlace at = place_of(p, blockIdx.x - 1);
  if (at.place >= p.slots.n) return;
  DeltaWave<DK> x(p);
  take_place(x, at.place, at);
  if (!x.span.kept || x.span.kept > kDeltaEnd) return;
  x.read(x.S);
  const bool bad = delta_end<DK>(x, 0, true);
  if (__any(bad)) {
    f32x4 S[2 * DeltaWave<DK>::KB];
    x.read(S);  // (the state in memory is still the one before)
    rows_again(x, S, 0, x.span.kept, bad);
  }
  x.write();
}

template <int DK>
static hipError_t prompt_launch(const DeltaParams& p, hipStream_t stream) {
  const long long blocks = row_blocks(p.tokens, p.slots.n, kDeltaRows);
  hipLaunchKernelGGL(delta_block_kernel<DK>, dim3((unsigned)(blocks * p.hk)), dim3(kThreads), 0,
                     stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int parts = p.dv / 16;
  auto groups = [&](long long places) { return (unsigned)((places * p.hv + 7) / 8 * 8 * parts); };
  long long places = p.slots.n;
  if (p.longs) {
    hipLaunchKernelGGL(delta_short_kernel<DK>, dim3(1 + groups(places)), dim3(64), 0, stream, p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    const long long most = p.tokens / (kDeltaEnd + 1);  // longer ones
    if (most < places) places = most;
    if (!places) return hipSuccess;
  }
  hipLaunchKernelGGL(delta_prompt_kernel<DK>, dim3(groups(places)), dim3(128), 0, stream, p);
  return hipGetLastError();
}

// Sequences of up to 16 rows apart, where the mean is at most 32 and there are more
// workgroups than the four a CU that LDS lets the longer ones' kernel have.
bool delta_splits(const DeltaParams& p, int cus) {
  return (long long)p.slots.n * p.hv * (p.dv / 16) > 4LL * cus && p.tokens <= 32LL * p.slots.n;
}

hipError_t delta_prompt_launch(const DeltaParams& p, hipStream_t stream) {
  return p.dk == 64 ? prompt_launch<64>(p, stream) : prompt_launch<128>(p, stream);
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
