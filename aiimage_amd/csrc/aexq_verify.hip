// Verification of drafted tokens against the target's probabilities (gfx950).
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
// A number may lie next to a border of the cumulative sum, whose cells are as small as
// 2^-25 of it where a vocabulary of 151936 is flat; fp32 weights would put one token in
// some hundreds on the other side.  So weights and sums are 64 bits here, 2^y from a
// polynomial (v_exp has no such form).
//   1. parts of rows: largest logit m, its index, Z = sum 2^((x - m) log2 e / T);
//   2. parts of the sampled rows, which every workgroup finds for itself: their sums of
//      2^((x - m) log2 e / T) and of max(p - q, 0);
//   3. a workgroup a sequence: the part the number falls into, and the index in it.
// ---------------------------------------------------------------------------
constexpr double kLog2eD = 1.4426950408889634074;

// 2^y for y <= 1000; 0 below -1074.  |error| < 2^-41 of it: the series of 2^f, f in
// [-1/2, 1/2], has (ln 2 / 2)^11 / 11! = 2^-42 behind its tenth power.
__device__ __forceinline__ double exp2_series(double y) {
  y = fmax(y, -1100.0);
  const double n = rint(y), f = y - n;
  double p = 7.054911620801121e-9;
  p = fma(p, f, 1.0178086009239696e-7);
  p = fma(p, f, 1.3215486790144305e-6);
  p = fma(p, f, 1.5252733804059838e-5);
  p = fma(p, f, 1.5403530393381606e-4);
  p = fma(p, f, 1.3333558146428441e-3);
  p = fma(p, f, 9.618129107628477e-3);
  p = fma(p, f, 5.550410866482157e-2);
  p = fma(p, f, 2.402265069591007e-1);
  p = fma(p, f, 6.931471805599453e-1);
  p = fma(p, f, 1.0);
  return ldexp(p, (int)n);
}

// What a row's logits are scaled by, in log2 units; 0 or below: the largest one wins.
__device__ __forceinline__ double heat_of(const VerifyParams& p, int s) {
  const float t = p.temperature ? p.temperature[s] : 1.0f;
  return t > 0.0f ? kLog2eD / (double)t : -1.0;
}
// A weight relative to the largest logit's; -inf weighs nothing at any temperature.
__device__ __forceinline__ double weight_of(float x, float m, double heat) {
  return x == -INFINITY ? 0.0 : exp2_series(((double)x - (double)m) * heat);
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
    lo += max(__popcll(at) - 1, 0) * step;
    if (step == 1) break;
  }
  return sreg(lo);
}

template <typename E>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(const VerifyParams p) {
  constexpr int VE = 16 / (int)sizeof(E);
  __shared__ Best best_of[kWaves];
  __shared__ double sum_of[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const int s = sequence_of(p, row);
  const Rows rows = rows_of(p, s);
  if (row < rows.first || row >= rows.first + rows.n) return;
  const double heat = heat_of(p, s);
  const E* x = (const E*)p.x + (long long)row * p.rstride;
  // chunks lie on 16-byte boundaries: chunk c starts at logit c VE - skew
  const int skew = (int)((uintptr_t)x % 16 / sizeof(E));
  const int chunks = (int)(((long long)p.n + skew + VE - 1) / VE);
  const int c0 = min(part * p.cols, chunks), c1 = min(c0 + p.cols, chunks);
  typedef E Chunk __attribute__((ext_vector_type(VE)));
  auto read = [&](int c) {
    const int i0 = c * VE - skew;
    Chunk v;
    if (i0 >= 0 && i0 <= p.n - VE) {
      v = *(const Chunk*)(x + i0);
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        v[i] = (E)-INFINITY;
        if (i0 + i >= 0 && i0 + i < p.n) v[i] = x[i0 + i];
      }
    }
    return v;
  };
  Best best = {-INFINITY, p.n};
  bool odd = false;  // a NaN or a +inf: the row has no probabilities
  double z = 0.0;
  for (int c = c0 + tid; c < c1; c += kThreads) {
    const Chunk v = read(c);
    const float old = best.m;
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const float y = (float)v[i];
      odd |= !(y < INFINITY);
      if (y > best.m) best = Best{y, c * VE - skew + i};
    }
    if (heat < 0.0 || best.m == -INFINITY) continue;
    if (best.m > old) z *= weight_of(old, best.m, heat);
#pragma unroll
    for (int i = 0; i < VE; ++i) z += weight_of((float)v[i], best.m, heat);
  }
  if (odd) z = __builtin_nan("");
  const float own = best.m;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1)
    best = better(best, Best{__shfl_xor(best.m, off, 64), __shfl_xor(best.at, off, 64)});
  if (lane == 0) best_of[wave] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) best = better(best, best_of[w]);
  if (best.m > -INFINITY) z *= weight_of(own, best.m, fmax(heat, 0.0));
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) z += __shfl_xor(z, off, 64);
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
// Rows in turn, by a whole wave; a lane joins a part.
__device__ __forceinline__ Chosen choose(const VerifyParams& p, int s, const Rows& rows) {
  const int lane = threadIdx.x & 63;
  const double heat = heat_of(p, s);
  Chosen r = {rows.first, kNone, -1, 0.0f, 0.0};
  for (int i = 0; i < rows.n; ++i) {
    const int row = rows.first + i;
    Best best = {-INFINITY, p.n};
    double z = 0.0;
    if (lane < p.parts) {
      const long long from = (long long)row * p.parts + lane;
      best = Best{p.m[from], p.at[from]};
      z = p.z[from];
    }
    const float own = best.m;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1)
      best = better(best, Best{__shfl_xor(best.m, off, 64), __shfl_xor(best.at, off, 64)});
    if (best.m > -INFINITY) z *= weight_of(own, best.m, fmax(heat, 0.0));
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) z += __shfl_xor(z, off, 64);
    r = Chosen{row, kNone, best.at, best.m, z};
    // (z is NaN where a logit is, and no sum where every one is -inf)
    if (!(best.m > -INFINITY) || !(z < INFINITY)) return r;
    const bool last = i == rows.n - 1;
    r.mode = heat < 0.0 ? kGreedy : last ? kFull : kRest;
    if (last) return r;
    const int draft = p.drafts[row];
    bool stays = false;
    if (draft >= 0 && draft < p.n) {
      if (heat < 0.0) {
        stays = draft == best.at;
      } else {
        const long long at = (long long)row * p.rstride + draft;
        const float x = p.f16 ? (float)((const f16*)p.x)[at] : ((const float*)p.x)[at];
        const double q = p.probs ? p.probs[row * p.probs_stride + draft] : 1.0f;
        stays = (double)p.accept_u[row] * q < weight_of(x, best.m, heat) / z;
      }
    }
    if (!stays) return r;
  }
  return r;
}

// The weights of index j of the sampled row.
struct Weights {
  double full, rest;
};
__device__ __forceinline__ Weights weights_of(const VerifyParams& p, const Chosen& r, double heat,
                                              int draft, int j) {
  const long long at = (long long)r.row * p.rstride + j;
  const float x = p.f16 ? (float)((const f16*)p.x)[at] : ((const float*)p.x)[at];
  Weights w;
  w.full = weight_of(x, r.m, heat);
  if (p.probs)
    w.rest = fmax(w.full - r.z * (double)p.probs[r.row * p.probs_stride + j], 0.0);
  else
    w.rest = j == draft ? 0.0 : w.full;
  return w;
}

// Sum over the workgroup, in every thread.
__device__ __forceinline__ double block_sum(double v, double* waves) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v += waves[w];
  return v;
}

__global__ __launch_bounds__(kThreads) void verify_sums_kernel(const VerifyParams p) {
  __shared__ double waves[2][kWaves];
  const int s = blockIdx.x / p.parts2, part = blockIdx.x % p.parts2, tid = threadIdx.x;
  const Rows rows = rows_of(p, s);
  const Chosen r = choose(p, s, rows);
  if (part == 0 && tid == 0) {
    p.plan[s] = int4{r.row, r.mode, r.token, rows.n ? r.row - rows.first + 1 : 0};
    p.norm[s] = double2{(double)r.m, r.z};
  }
  if (r.mode != kFull && r.mode != kRest) return;
  const double heat = heat_of(p, s);
  const int draft = p.drafts[r.row];
  const long long end = min((long long)p.n, (part + 1LL) * p.run);
  double full = 0.0, rest = 0.0;
  for (long long j = (long long)part * p.run + tid; j < end; j += kThreads) {
    const Weights w = weights_of(p, r, heat, draft, (int)j);
    full += w.full;
    rest += w.rest;
  }
  full = block_sum(full, waves[0]);
  rest = block_sum(rest, waves[1]);
  if (tid == 0) {
    double* to = p.sums + 2LL * blockIdx.x;
    to[0] = full;
    to[1] = rest;
  }
}

__global__ __launch_bounds__(kThreads) void verify_token_kernel(const VerifyParams p) {
  __shared__ double before[kThreads + 1];
  __shared__ int found, last_one;
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const Rows rows = rows_of(p, s);
  const int4 plan = p.plan[s];
  Chosen r = {plan.x, plan.y, plan.z, (float)p.norm[s].x, p.norm[s].y};
  int token = r.mode == kGreedy ? r.token : -1;
  if (r.mode == kFull || r.mode == kRest) {
    const double heat = heat_of(p, s);
    const int draft = p.drafts[r.row];
    // the part: every wave, a lane a part
    double full = 0.0, rest = 0.0;
    if (lane < p.parts2) {
      full = p.sums[2LL * (s * p.parts2 + lane)];
      rest = p.sums[2LL * (s * p.parts2 + lane) + 1];
    }
    bool whole = r.mode == kFull || !__any(rest > 0.0);
    double own = whole ? full : rest, upto = own;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const double v = __shfl_up(upto, off, 64);
      if (lane >= off) upto += v;
    }
    const double total = __shfl(upto, 63, 64), goal = (double)p.sample_u[s] * total;
    // (the last one that weighs something, where rounding leaves none)
    const uint64_t over = __ballot(upto > goal && own > 0.0), some = __ballot(own > 0.0);
    const int part = over ? __ffsll((unsigned long long)over) - 1
                          : 63 - __clzll((unsigned long long)some);
    const double start = __shfl(upto - own, max(part, 0), 64);
    const int j0 = max(part, 0) * p.run, j1 = (int)min((long long)p.n, (long long)j0 + p.run);
    const int each = (p.run + kThreads - 1) / kThreads;
    const int a = min(j0 + tid * each, j1), b = min(a + each, j1);
    auto weight = [&](int j) {
      const Weights w = weights_of(p, r, heat, draft, j);
      return whole ? w.full : w.rest;
    };
    double sum = 0.0;
    for (int j = a; j < b; ++j) sum += weight(j);
    before[tid + 1] = sum;
    if (tid == 0) {
      before[0] = start;
      found = p.n;
      last_one = -1;
    }
    __syncthreads();
    if (tid == 0)
      for (int i = 0; i < kThreads; ++i) before[i + 1] += before[i];
    __syncthreads();
    double at = before[tid];
    int hit = p.n, some_one = -1;
    for (int j = a; j < b; ++j) {
      const double w = weight(j);
      at += w;
      if (w > 0.0) {
        some_one = j;
        if (at > goal && hit == p.n) hit = j;
      }
    }
    if (hit < p.n) atomicMin(&found, hit);
    if (some_one >= 0) atomicMax(&last_one, some_one);
    __syncthreads();
    token = found < p.n ? found : last_one;
  }
  if (tid == 0) p.counts[s] = plan.w;
  for (int i = tid; i < rows.n; i += kThreads)
    p.tokens[rows.first + i] = i < plan.w - 1    ? p.drafts[rows.first + i]
                               : i == plan.w - 1 ? token
                                                 : -1;
}

// Parts of a row: enough for two workgroups per CU, each of at least 512 chunks.
int verify_parts(long long rows, int n, int esize, int cus) {
  const long long chunks = ((long long)n * esize + 15) / 16;
  const long long parts = (2LL * cus + rows - 1) / rows, most = (chunks + 511) / 512;
  const long long r = parts < most ? parts : most;
  return (int)(r < 1 ? 1 : r > kVerifyParts ? kVerifyParts : r);
}

hipError_t verify_launch(const VerifyParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)((long long)p.rows * p.parts));
  if (p.f16)
    hipLaunchKernelGGL(verify_rows_kernel<f16>, grid, dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL(verify_rows_kernel<float>, grid, dim3(kThreads), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(verify_sums_kernel, dim3((unsigned)(p.sequences * p.parts2)), dim3(kThreads), 0,
                     stream, p);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(verify_token_kernel, dim3((unsigned)p.sequences), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace aexq
