// Verification of drafted tokens against the target's probabilities (gfx950).
#include <float.h>
#include <limits.h>
#include <math.h>

#include "aexq_rows.hpp"

namespace aexq {

// ---------------------------------------------------------------------------
// Row i of a sequence holds the target's logits x behind its i-th token, p = softmax(x /
// T).  The draft d behind it stays while u_i q(d) < p(d) (q: the draft's probabilities,
// or 1 where none are given).  From the first row whose draft does not, the new token
// is drawn from max(p - q, 0), where all stay from the last row's p: the first index
// whose cumulative weight passes the sequence's number times their sum.
//
// A number may lie next to a border of the cumulative sum, whose cells are 2^-17 of it
// where a vocabulary of 151936 is flat; a sum of fp32 weights, off by 2^-24 and more of it,
// would put one token in some hundreds on the other side.  So weights and sums are 64 bits
// here, 2^y from a polynomial (v_exp has no such form).
//   1. parts of rows: largest logit m, its index, Z = sum 2^((x - m) log2 e / T);
//   2. runs of the sampled rows, which every workgroup finds for itself: their sums of
//      2^((x - m) log2 e / T) and of max(p - q, 0);
//   3. a workgroup a sequence: the run the number falls into, and the index in it.
// 64-bit arithmetic bounds the first two: 265 rows of 151936 fp32 logits take 40 us (161
// MB, 4.0 TB/s), 31 with a plain sum in the weights' place (5.1 TB/s) and 37 with each
// thread's loads from one place; 64 sampled rows with draft probabilities 23 us (78 MB).
// Logits of fp16 are half the bytes and the same arithmetic: the call takes 72 us with draft
// probabilities (70 of fp32 ones), 65 without (74).  Where all rows are greedy it takes 40.
// The third takes 6 us, and 13 where its scans go through LDS.  One sequence of five rows
// is three launches of 3 to 6 us.
// ---------------------------------------------------------------------------
constexpr double kLog2eD = 1.4426950408889634074;

// 2^y for y <= 1000, |error| < 2^-39 of it; 0 below -1023 and for a NaN.  y = n + f with
// n whole, f in [-1/2, 1/2]: 2^f is the polynomial of degree 8 that is 1 at 0 and whose
// largest relative error, 1.07e-12 = 2^-39.8, is least (the exchange method; the series
// needs degree 10 for that).  Adding 1.5 * 2^52 leaves n in the sum's low bits; n is added
// to the exponent of 2^f, which at y = -1023 is that of 1: nothing is left.
__device__ __forceinline__ double exp2_series(double y) {
  y = fmax(y, -1023.0);
  const double t = y + 0x1.8p52, f = y - (t - 0x1.8p52);
  double p = 1.3255224878668817e-6;
  p = fma(p, f, 1.5310079402249296e-5);
  p = fma(p, f, 1.5403455852453838e-4);
  p = fma(p, f, 1.3333450568000645e-3);
  p = fma(p, f, 9.618129159402558e-3);
  p = fma(p, f, 5.550410941205933e-2);
  p = fma(p, f, 2.402265069581299e-1);
  p = fma(p, f, 6.931471805459335e-1);
  p = fma(p, f, 1.0);
  typedef uint32_t Words __attribute__((ext_vector_type(2)));
  Words w = __builtin_bit_cast(Words, p);
  w.y += __builtin_bit_cast(Words, t).x << 20;
  return __builtin_bit_cast(double, w);
}

// What a row's logits are scaled by, in log2 units; 0 or below: the largest one wins.
__device__ __forceinline__ double heat_of(const VerifyParams& p, int s) {
  const float t = p.temperature ? p.temperature[s] : 1.0f;
  return t > 0.0f ? kLog2eD / (double)t : -1.0;
}
// The weight of logit x relative to that of m; nothing for -inf, above all others if m
// is -inf.
__device__ __forceinline__ double weight_of(float x, float m, double heat) {
  return exp2_series(((double)x - (double)fmaxf(m, -FLT_MAX)) * heat);
}

struct Best {
  float m;
  int at;
};
// The larger logit, then the lower index.
__device__ __forceinline__ Best better(Best a, Best b) {
  return b.m > a.m || (b.m == a.m && b.at < a.at) ? b : a;
}

// Rows of a sequence, kept within the call's.
struct Rows {
  int first, n;
};
__device__ __forceinline__ Rows rows_of(const VerifyParams& p, int s) {
  const int first = min(max(p.offsets[s], 0), p.rows);
  return Rows{first, min(max(p.offsets[s + 1], first), p.rows) - first};
}
// The sequence of row t (the last one that begins at or before it).
__device__ __forceinline__ int sequence_of(const VerifyParams& p, int t) {
  const int lane = threadIdx.x & 63, n = p.sequences;
  int lo = 0, step = 1;
  while (step * 64 < n) step *= 64;
  for (;; step /= 64) {
    const int s = lo + lane * step;
    const uint64_t at = __ballot(s < n && p.offsets[min(s, n - 1)] <= t);
    lo += max((int)__popcll(at) - 1, 0) * step;
    if (step == 1) break;
  }
  return sreg(lo);
}

// The best of a wave, in every lane.
__device__ __forceinline__ Best wave_best(Best v) {
  auto join = [&](auto move) {
    v = better(v, Best{move(v.m), __builtin_bit_cast(int, move(__builtin_bit_cast(float, v.at)))});
  };
  join([](float x) { return dpp<0x128>(x); });
  join([](float x) { return dpp<0x124>(x); });
  join([](float x) { return dpp<0x4E>(x); });
  join([](float x) { return dpp<0xB1>(x); });
  join([](float x) { return dpp_rows<0x142, 0xA>(x, x); });
  join([](float x) { return dpp_rows<0x143, 0xC>(x, x); });
  return Best{__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v.m), 63)),
              __builtin_amdgcn_readlane(v.at, 63)};
}

template <typename E>
__global__ __launch_bounds__(kThreads, 4) void verify_rows_kernel(const VerifyParams p) {
  constexpr int VE = 16 / (int)sizeof(E), U = 4;
  __shared__ Best best_of[kWaves];
  __shared__ double sum_of[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const int s = sequence_of(p, row);
  const Rows rows = rows_of(p, s);
  if (row < rows.first || row >= rows.first + rows.n) return;
  const double heat = heat_of(p, s);
  const E* x = (const E*)p.x + (long long)row * p.rstride;
  if (part == 0 && tid == 0) {
    // the draft behind the row, and what its weight over Z has to pass
    VerifyDraft d = {INFINITY, -INFINITY, -1};
    if (row + 1 < rows.first + rows.n) {
      const int token = p.drafts[row];
      if (token >= 0 && token < p.n) {
        const double q = p.probs ? p.probs[row * p.probs_stride + token] : 1.0f;
        d = VerifyDraft{(double)p.accept_u[row] * q, (float)x[token], token};
      }
    }
    p.draft[row] = d;
  }
  // chunks lie on 16-byte boundaries, chunk c at logit c VE - skew; those that are not
  // whole go a logit a thread, the first one's with the first part, the last one's with
  // the last
  const int skew = (int)((uintptr_t)x % 16 / sizeof(E));
  const int whole0 = skew ? 1 : 0, whole1 = (int)(((long long)p.n + skew) / VE);
  const int c0 = max(part * p.cols, whole0), c1 = min((part + 1) * p.cols, whole1);
  const int head = skew ? min(VE - skew, p.n) : 0, tail = max(whole1 * VE - skew, head);
  typedef E Chunk __attribute__((ext_vector_type(VE)));
  E edge[2] = {(E)-INFINITY, (E)-INFINITY};
  if (part == 0 && tid < head) edge[0] = x[tid];
  if (part == p.parts - 1 && tail + tid < p.n) edge[1] = x[tail + tid];
  // U chunks of a thread, the ones of neighbours next to each other; nothing from c1 on
  auto read = [&](int c, Chunk* v) {
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = *(const Chunk*)(x + min(c + u * kThreads, c1 - 1) * VE - skew);
#pragma unroll
    for (int u = 1; u < U; ++u)
      if (c + u * kThreads >= c1) v[u] = (Chunk)(E)-INFINITY;
  };
  Best best = {-INFINITY, p.n};
  double z = 0.0;
  float from = -FLT_MAX;  // what the weights are relative to; none is above 2^500
  if (heat < 0.0) {
    bool odd = false;  // a NaN or a +inf: the row has no largest logit
    auto take = [&](float y, int at) {
      odd |= !(y < INFINITY);
      if (y > best.m) best = Best{y, at};
    };
    take((float)edge[0], tid);
    for (int c = c0 + tid; c < c1; c += U * kThreads) {
      Chunk v[U];
      read(c, v);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < VE; ++i) take((float)v[u][i], (c + u * kThreads) * VE - skew + i);
    }
    take((float)edge[1], tail + tid);
    if (odd) z = __builtin_nan("");
  } else {
    auto relate = [&]() {
      if (((double)best.m - (double)from) * heat > 500.0) {
        z *= weight_of(from, best.m, heat);
        from = best.m;
      }
    };
    for (int c = c0 + tid; c < c1; c += U * kThreads) {
      Chunk v[U];
      read(c, v);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < VE; ++i)
          best.m = __builtin_elementwise_maximum(best.m, (float)v[u][i]);
      relate();
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < VE; ++i) z += weight_of((float)v[u][i], from, heat);
    }
    if (__any(fmaxf((float)edge[0], (float)edge[1]) > -INFINITY || edge[0] != edge[1])) {
      best.m = __builtin_elementwise_maximum(best.m, (float)edge[0]);
      best.m = __builtin_elementwise_maximum(best.m, (float)edge[1]);
      relate();
      z += weight_of((float)edge[0], from, heat) + weight_of((float)edge[1], from, heat);
    }
    if (!(best.m < INFINITY)) z = __builtin_nan("");
  }
  best = wave_best(best);
  if (lane == 0) best_of[wave] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) best = better(best, best_of[w]);
  if (best.m > -INFINITY) z *= weight_of(from, best.m, fmax(heat, 0.0));
  z = wave_sum(z);
  if (lane == 0) sum_of[wave] = z;
  __syncthreads();
  if (tid) return;
  z = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) z += sum_of[w];
  const long long to = (long long)row * p.parts + part;
  p.z[to] = z;
  p.m[to] = best.m;
  p.at[to] = best.at;
}

enum : int { kNone = 0, kGreedy = 1, kFull = 2, kRest = 3 };
// The sampled row of a sequence: how its token is found, and the rows that stay.
struct Chosen {
  int row, mode, token;
  float m;
  double z;
};
// By the whole workgroup, two rows a wave at a time; a lane joins a part.
__device__ __forceinline__ Chosen choose(const VerifyParams& p, const Rows& rows, double heat,
                                         Chosen* of, int* goes_on) {
  constexpr int K = 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Chosen r = {rows.first, kNone, -1, 0.0f, 0.0};
  for (int i0 = 0; i0 < rows.n; i0 += K * kWaves) {
    Best best[K];
    double z[K];
    VerifyDraft d[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int row = rows.first + min(i0 + K * wave + k, rows.n - 1);
      const long long at = (long long)row * p.parts + min(lane, p.parts - 1);
      best[k] = Best{p.m[at], p.at[at]};
      z[k] = p.z[at];
      d[k] = p.draft[row];
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = i0 + K * wave + k;
      if (lane >= p.parts) best[k] = Best{-INFINITY, p.n}, z[k] = 0.0;
      const float own = best[k].m;
      best[k] = wave_best(best[k]);
      if (best[k].m > -INFINITY) z[k] *= weight_of(own, best[k].m, fmax(heat, 0.0));
      z[k] = wave_sum(z[k]);
      // (z is NaN where a logit is, and no sum where every one is -inf)
      const bool none = !(best[k].m > -INFINITY) || !(z[k] < INFINITY);
      const bool last = i >= rows.n - 1;
      const bool stays = heat < 0.0 ? d[k].token == best[k].at
                                    : d[k].need < weight_of(d[k].x, best[k].m, heat) / z[k];
      if (lane == 0) {
        const int mode = none ? kNone : heat < 0.0 ? kGreedy : last ? kFull : kRest;
        of[K * wave + k] = Chosen{rows.first + i, mode, best[k].at, best[k].m, z[k]};
        goes_on[K * wave + k] = !none && !last && stays;
      }
    }
    __syncthreads();
    const uint64_t ends = __ballot(!goes_on[min(lane, K * kWaves - 1)]);
    const int n = ends ? __ffsll((unsigned long long)ends) - 1 : K * kWaves - 1;
    r = of[n];
    const bool on = goes_on[n];
    __syncthreads();
    if (!on) return r;
  }
  return r;
}

// The weights of index j of the sampled row; none from `end` on.
struct Weights {
  double full, rest;
};
template <typename E, int N>
__device__ __forceinline__ void weights_of(const VerifyParams& p, const Chosen& r, double heat,
                                           int draft, int j0, int step, int end, Weights* w) {
  const E* x = (const E*)p.x + (long long)r.row * p.rstride;
  // (where there are no probabilities to take off: some float, and none of it)
  const bool less = p.probs && r.mode == kRest;
  const float* q = less ? p.probs + r.row * p.probs_stride : p.accept_u;
  const int skip = less ? -1 : draft;
  E v[N];
  float taken[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int j = min(j0 + i * step, end - 1);
    v[i] = x[j];
    taken[i] = q[less ? j : 0];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int j = j0 + i * step;
    w[i].full = weight_of(j < end ? (float)v[i] : -INFINITY, r.m, heat);
    const double rest = fmax(w[i].full - r.z * (double)(less ? taken[i] : 0.0f), 0.0);
    w[i].rest = j == skip ? 0.0 : rest;
  }
}

// A wave sums runs of the sampled row.
template <typename E>
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(const VerifyParams p) {
  __shared__ Chosen of[2 * kWaves];
  __shared__ int goes_on[2 * kWaves];
  const int s = blockIdx.x / p.blocks, lane = threadIdx.x & 63;
  const int run0 = blockIdx.x % p.blocks * kWaves + (threadIdx.x >> 6);
  const Rows rows = rows_of(p, s);
  const double heat = heat_of(p, s);
  const Chosen r = choose(p, rows, heat, of, goes_on);
  if (run0 == 0 && lane == 0) {
    p.plan[s] = int4{r.row, r.mode, r.token, rows.n ? r.row - rows.first + 1 : 0};
    p.norm[s] = double2{(double)r.m, r.z};
  }
  if (r.mode != kFull && r.mode != kRest) return;
  const int draft = r.mode == kRest ? p.draft[r.row].token : -1;
  for (int run = run0; run < p.runs; run += p.blocks * kWaves) {
    const int end = min(p.n, (run + 1) * p.run);
    double full = 0.0, rest = 0.0;
    constexpr int N = 5;
    for (int j = run * p.run; j < end; j += 64 * N) {
      Weights w[N];
      weights_of<E, N>(p, r, heat, draft, j + lane, 64, end, w);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        full += w[i].full;
        rest += w[i].rest;
      }
    }
    full = wave_sum(full);
    rest = wave_sum(rest);
    if (lane == 0) p.sums[(long long)s * p.runs + run] = double2{full, rest};
  }
}

// Sums up to and with each thread's; `total` is the last one.
__device__ __forceinline__ double block_scan(double v, double* waves, double* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan(v);
  __syncthreads();
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) v += waves[w];
    sum += waves[w];
  }
  *total = sum;
  return v;
}

// The first thread's index for which `hit` holds, in *first, and the last one's for
// which `some` does, in *last.
__device__ __forceinline__ void block_find(bool hit, bool some, int at, int* first, int* last) {
  const uint64_t hits = __ballot(hit), somes = __ballot(some);
  const int lane = threadIdx.x & 63;
  if (hits && lane == __ffsll((unsigned long long)hits) - 1) atomicMin(first, at);
  if (somes && lane == 63 - __clzll((unsigned long long)somes)) atomicMax(last, at);
  __syncthreads();
}

template <typename E>
__global__ __launch_bounds__(kThreads) void verify_token_kernel(const VerifyParams p) {
  static_assert(kVerifyRuns <= kThreads, "a thread a run");
  __shared__ double waves[kWaves];
  __shared__ int first[2], last[2], any_rest;
  __shared__ double start_of;
  const int s = blockIdx.x, tid = threadIdx.x;
  const Rows rows = rows_of(p, s);
  const int4 plan = p.plan[s];
  Chosen r = {plan.x, plan.y, plan.z, (float)p.norm[s].x, p.norm[s].y};
  int token = r.mode == kGreedy ? r.token : -1;
  if (r.mode == kFull || r.mode == kRest) {
    const double heat = heat_of(p, s);
    const int draft = r.mode == kRest ? p.draft[r.row].token : -1;
    if (tid < 2) first[tid] = INT_MAX, last[tid] = -1;
    if (tid == 0) any_rest = 0;
    __syncthreads();
    const double2 sum = tid < p.runs ? p.sums[(long long)s * p.runs + tid] : double2{0.0, 0.0};
    if (r.mode == kRest && __any(sum.y > 0.0)) any_rest = 1;
    __syncthreads();
    const bool whole = !any_rest;
    double own = whole ? sum.x : sum.y, total;
    double upto = block_scan(own, waves, &total);
    const double goal = (double)p.sample_u[s] * total;
    // (the last one that weighs something, where rounding leaves none)
    block_find(upto > goal && own > 0.0, own > 0.0, tid, first, last);
    const int run = first[0] < INT_MAX ? first[0] : last[0];
    if (run >= 0) {
      if (tid == run) start_of = upto - own;
      __syncthreads();
      double start = start_of;
      const int j0 = run * p.run, end = min(p.n, j0 + p.run);
#pragma unroll 1
      for (int j = j0; j < end; j += kThreads) {
        Weights w;
        weights_of<E, 1>(p, r, heat, draft, j + tid, 0, end, &w);
        own = whole ? w.full : w.rest;
        upto = block_scan(own, waves, &total) + start;
        start += total;
        block_find(upto > goal && own > 0.0, own > 0.0, j + tid, first + 1, last + 1);
        if (first[1] < INT_MAX) break;
      }
      token = first[1] < INT_MAX ? first[1] : last[1];
    }
  }
  if (tid == 0) p.counts[s] = plan.w;
  for (int i = tid; i < rows.n; i += kThreads)
    p.tokens[rows.first + i] = i < plan.w - 1    ? p.drafts[rows.first + i]
                               : i == plan.w - 1 ? token
                                                 : -1;
}

// Parts of a row: enough for eight workgroups per CU, each of at least 512 chunks.
int verify_parts(long long rows, int n, int esize, int cus) {
  const long long chunks = ((long long)n * esize + 15) / 16;
  const long long parts = (8LL * cus + rows - 1) / rows, most = (chunks + 511) / 512;
  const long long r = parts < most ? parts : most;
  return (int)(r < 1 ? 1 : r > kVerifyParts ? kVerifyParts : r);
}

// Runs of a sampled row: of at least 256 values, whole workgroups of them.
int verify_runs(int n) {
  const int runs = (n + 255) / 256;
  return runs >= kVerifyRuns ? kVerifyRuns : (runs + kWaves - 1) / kWaves * kWaves;
}
// Workgroups that sum the runs of a sequence: eight per CU for all sequences.
int verify_blocks(int sequences, int runs, int cus) {
  const int most = runs / kWaves, r = (8 * cus + sequences - 1) / sequences;
  return r < most ? r : most;
}

template <typename E>
static hipError_t verify_type(const VerifyParams& p, hipStream_t stream) {
  hipLaunchKernelGGL(verify_rows_kernel<E>, dim3((unsigned)((long long)p.rows * p.parts)),
                     dim3(kThreads), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(verify_sums_kernel<E>, dim3((unsigned)(p.sequences * p.blocks)),
                     dim3(kThreads), 0, stream, p);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(verify_token_kernel<E>, dim3((unsigned)p.sequences), dim3(kThreads), 0, stream,
                     p);
  return hipGetLastError();
}

hipError_t verify_launch(const VerifyParams& p, hipStream_t stream) {
  return p.f16 ? verify_type<f16>(p, stream) : verify_type<float>(p, stream);
}

}  // namespace aexq
