// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits (gfx950).
#include <math.h>

#include "aexq_device.hpp"
#include "aexq_serving.hpp"

namespace aexq {

// ---------------------------------------------------------------------------
// One pass over a row of logits x with a running reference b:
//   y = log2 e (x - max so far),  Z = sum 2^y,  T = sum 2^y y
//   log p[t] = ln 2 (y[t] - log2 Z),   H = ln 2 (log2 Z - T / Z)
// fp16: b is the rounded log2 e times the maximum and y one fma, x log2 e - b; no
// sum depends on how b was rounded, so large logits lose nothing.  fp32: b is the
// maximum itself, as a logit of the type's lowest value (a mask) times log2 e is
// past the type's range.
// Lanes take 16-byte chunks in turn; what a lane keeps for the alternatives is
// its best chunk (by its largest logit) and the largest logit of the others.
//
// The K best of the row, by logit and then by index: a bound that K of the 256
// lanes' best chunks reach is one that K logits reach, so only chunks that reach
// it are read again (mostly about K of them), and a lane's whole share only where
// its second chunk reaches it too.  Those logits go through a sorted
// list per wave, an entry a lane; the four lists are merged by counting, for
// each entry, the entries above it.
//
// Reading the logits bounds it (HBM): 777 rows of 151936 fp32 logits, 20 alternatives,
// 87 us (5.4 TB/s), 512 rows of fp16 ones 41 (3.8).  Few rows are cut into parts of
// chunks, a workgroup each, whose (m, Z, T, K best) a second launch joins in the same
// way (one row, 5 alternatives: 7.1 and 4.8 us, each a chain of dependent loads).
// ---------------------------------------------------------------------------
typedef unsigned long long u64;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// y of a logit that weighs nothing (-inf among them)
constexpr float kFar = -300.0f;

// Order of the alternatives: the larger logit, then the lower index.  0 is below
// every logit.
__device__ __forceinline__ u64 top_key(float x, int index) {
  return (u64)argmax_ord(x) << 32 | (uint32_t)~index;
}

struct Stats {
  float b, z, t;
};
// The reference for a maximum m, y of logit x, and y's step between references.
template <typename E>
constexpr bool kHalf = sizeof(E) == 2;
template <typename E>
__device__ __forceinline__ float reference(float m) {
  return kHalf<E> ? m * kLog2e : m;
}
template <typename E>
__device__ __forceinline__ float away(float x, float b) {
  return kHalf<E> ? fmaf(x, kLog2e, -b) : (x - b) * kLog2e;
}
template <typename E>
__device__ __forceinline__ float shift(float from, float to) {
  return fmaxf(kHalf<E> ? from - to : (from - to) * kLog2e, kFar);
}
// The sums of two parts on the larger reference; parts of weight 0 add 0.
template <typename E>
__device__ __forceinline__ Stats join(Stats p, Stats q) {
  const float b = fmaxf(p.b, q.b), base = b == -INFINITY ? 0.0f : b;
  const float dp = shift<E>(p.b, base), dq = shift<E>(q.b, base);
  const float fp = __builtin_amdgcn_exp2f(dp), fq = __builtin_amdgcn_exp2f(dq);
  Stats r;
  r.b = b;
  r.z = p.z * fp + q.z * fq;
  r.t = fp * fmaf(p.z, dp, p.t) + fq * fmaf(q.z, dq, q.t);
  return r;
}
template <typename E>
__device__ __forceinline__ Stats join_wave(Stats p) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    Stats q;
    q.b = __shfl_xor(p.b, off, 64);
    q.z = __shfl_xor(p.z, off, 64);
    q.t = __shfl_xor(p.t, off, 64);
    p = join<E>(p, q);
  }
  return p;
}

// A row's outputs by its workgroup: thread r < top has the r-th key.  A row
// whose logits have no finite sum of exponentials (a NaN, a +inf, or only -inf)
// has no probabilities: NaN, and alternatives -1.
template <typename E>
__device__ __forceinline__ void row_outputs(const LogprobParams& p, int row, const E* x, Stats s,
                                            u64 key) {
  const bool sound = s.z > 0.0f && s.z < INFINITY;
  const float log2z = log2f(s.z), nan = __builtin_nanf("");
  auto log_p = [&](float x) {
    return kHalf<E> ? (away<E>(x, s.b) - log2z) * kLn2 : x - s.b - log2z * kLn2;
  };
  if (threadIdx.x == 0) {
    if (p.logprob) {
      const int token = p.tokens[row];
      float v = token == -1 ? 0.0f : nan;
      if (sound && token >= 0 && token < p.n) v = log_p((float)x[token]);
      p.logprob[row] = v;
    }
    if (p.entropy) p.entropy[row] = sound ? (log2z - s.t / s.z) * kLn2 : nan;
  }
  if ((int)threadIdx.x < p.top) {
    const long long at = (long long)row * p.top + threadIdx.x;
    if (p.ids) p.ids[at] = sound ? (int)~(uint32_t)key : -1;
    if (p.values) p.values[at] = sound ? log_p(argmax_unord((uint32_t)(key >> 32))) : nan;
  }
}

// Puts `key` (wave-uniform) into the wave's sorted list, an entry a lane.
__device__ __forceinline__ void list_insert(u64& entry, u64 key) {
  const int at = __popcll(__ballot(entry > key)), lane = threadIdx.x & 63;
  const u64 up = __shfl_up(entry, 1, 64);
  entry = lane < at ? entry : lane == at ? key : up;
}

// A key that at least `top` of the kThreads keys (0: none) reach, and few more:
// bit by bit from above until no more than `top` + 8 reach it.  0 where fewer than
// `top` are there.  By every wave, four keys a lane.
__device__ __forceinline__ u64 top_bound(const u64* keys, int top) {
  const int lane = threadIdx.x & 63;
  u64 k[kThreads / 64];
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) k[i] = keys[i * 64 + lane];
  uint32_t high = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = high | 1u << bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) n += __popcll(__ballot((uint32_t)(k[i] >> 32) >= c));
    if (n < top) continue;
    high = c;
    if (n <= top + 8) return (u64)high << 32;
  }
  uint32_t low = 0;  // many equal logits: by index too
  for (int bit = 31; bit >= 0; --bit) {
    const u64 c = (u64)high << 32 | low | 1u << bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) n += __popcll(__ballot(k[i] >= c));
    if (n >= top) low |= 1u << bit;
  }
  return (u64)high << 32 | low;
}

// STREAM: the logits do not stay in the caches.
template <typename E, bool STREAM>
__global__ __launch_bounds__(kThreads) void logprob_kernel(const LogprobParams p) {
  constexpr int VE = 16 / (int)sizeof(E), U = 3;  // logits of a chunk, chunks in flight
  __shared__ Stats wave_stats[kWaves];
  __shared__ u64 keys[kThreads], sorted[64];
  __shared__ int counts[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const E* x = (const E*)p.x + (long long)row * p.rstride;
  // chunks lie on 16-byte boundaries: chunk c starts at logit c VE - skew
  const int skew = (int)((uintptr_t)x % 16 / sizeof(E));
  const int chunks = (int)(((long long)p.n + skew + VE - 1) / VE);
  const int c0 = min(part * p.cols, chunks), c1 = min(c0 + p.cols, chunks);

  // chunk c; logits before the row's first or past its last read -inf
  typedef E Chunk __attribute__((ext_vector_type(VE)));
  auto read = [&](int c) {
    const int i0 = c * VE - skew;
    Chunk v;
    if (i0 >= 0 && i0 <= p.n - VE) {
      v = STREAM ? __builtin_nontemporal_load((const Chunk*)(x + i0)) : *(const Chunk*)(x + i0);
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        v[i] = (E)-INFINITY;
        if (i0 + i >= 0 && i0 + i < p.n) v[i] = x[i0 + i];
      }
    }
    return v;
  };
  const Chunk none = (Chunk)(E)-INFINITY;

  Stats s = {-INFINITY, 0.0f, 0.0f};
  float best = -INFINITY, second = -INFINITY;
  int best_chunk = c0 + tid;
  Chunk next[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    next[u] = c0 + tid + u * kThreads < c1 ? read(c0 + tid + u * kThreads) : none;
  for (int c = c0 + tid; c < c1; c += U * kThreads) {
    Chunk v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = next[u];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // the next chunks on their way
      const int n = c + (U + u) * kThreads;
      next[u] = n < c1 ? read(n) : none;
    }
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      E t = v[u][0];
#pragma unroll
      for (int i = 1; i < VE; ++i) t = __builtin_elementwise_maxnum(t, v[u][i]);
      const float top = (float)t;
      m = fmaxf(m, top);
      second = fmaxf(second, fminf(best, top));
      best_chunk = top > best ? c + u * kThreads : best_chunk;
      best = fmaxf(best, top);
    }
    const float b = fmaxf(s.b, reference<E>(m)), base = b == -INFINITY ? 0.0f : b;
    const float d = shift<E>(s.b, base), f = __builtin_amdgcn_exp2f(d);
    s.t = f * fmaf(s.z, d, s.t);
    s.z *= f;
    s.b = b;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const float y = away<E>((float)v[u][i], base), e = __builtin_amdgcn_exp2f(y);
        s.z += e;
        s.t = fmaf(e, fmaxf(y, kFar), s.t);
      }
  }
  s = join_wave<E>(s);
  if (lane == 0) wave_stats[wave] = s;

  u64 key = 0;
  if (p.top) {
    const bool any = c0 + tid < c1;
    // some logit of the best chunk is `best`, at the chunk's last index or before
    const u64 mine = any ? top_key(best, min(best_chunk * VE - skew + VE, p.n) - 1) : 0;
    keys[tid] = mine;
    if (tid < 64) sorted[tid] = 0;
    __syncthreads();
    const u64 least = top_bound(keys, p.top);  // 0: fewer chunks than alternatives, so all of them
    const bool all = any && argmax_ord(second) >= (uint32_t)(least >> 32);
    const bool one = any && !all && top_key(best, max(best_chunk * VE - skew, 0)) >= least;
    u64 entry = 0;
    auto take = [&](int c, bool on) {
      const Chunk v = on ? read(c) : none;
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const int at = c * VE - skew + i;
        const float y = (float)v[i];
        const bool in = on && at >= 0 && at < p.n && !__builtin_isnan(y);
        const u64 k = in ? top_key(y, at) : 0;
        for (u64 left = __ballot(in && k >= least); left; left &= left - 1) {
          const int from = __ffsll((unsigned long long)left) - 1;
          const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(k >> 32), from);
          const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)k, from);
          list_insert(entry, (u64)hi << 32 | lo);
        }
      }
    };
    if (__any(one)) take(best_chunk, one);
    for (u64 left = __ballot(all); left; left &= left - 1) {
      // the whole share of one lane, by all lanes
      const int from = __ffsll((unsigned long long)left) - 1;
      for (int c = c0 + wave * 64 + from; c < c1; c += 64 * kThreads) {
        const int at = c + lane * kThreads;
        take(at, at < c1);
      }
    }
    const u64 own = lane < p.top ? entry : 0;
    __syncthreads();
    keys[tid] = own;
    const int held = __popcll(__ballot(own != 0));
    if (lane == 0) counts[wave] = held;
    __syncthreads();
    int above = 0;
    for (int w = 0; w < kWaves; ++w)
      for (int i = 0; i < counts[w]; ++i) above += keys[w * 64 + i] > own;
    if (own && above < p.top) sorted[above] = own;
  }
  __syncthreads();
  if (tid < p.top) key = sorted[tid];
  s = wave_stats[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) s = join<E>(s, wave_stats[w]);
  if (p.parts == 1) {
    row_outputs(p, row, x, s, key);
    return;
  }
  if (tid == 0) {
    float* to = p.stats + 4LL * blockIdx.x;
    to[0] = s.b;
    to[1] = s.z;
    to[2] = s.t;
  }
  if (tid < p.top) p.keys[(long long)blockIdx.x * p.top + tid] = key;
}

// Joins the parts of a row (at most kThreads).
template <typename E>
__global__ __launch_bounds__(kThreads) void logprob_join_kernel(const LogprobParams p) {
  __shared__ Stats wave_stats[kWaves];
  __shared__ u64 first[kThreads], reach[72 * 64], sorted[64];
  __shared__ int count;
  const int row = blockIdx.x, tid = threadIdx.x;
  const u64* keys = p.keys + (long long)row * p.parts * p.top;
  Stats s = {-INFINITY, 0.0f, 0.0f};
  u64 mine = 0;
  if (tid < p.parts) {
    const float* from = p.stats + 4LL * (row * (long long)p.parts + tid);
    s = Stats{from[0], from[1], from[2]};
    if (p.top) mine = keys[(long long)tid * p.top];
  }
  s = join_wave<E>(s);
  if ((tid & 63) == 0) wave_stats[tid >> 6] = s;
  u64 key = 0;
  if (p.top) {
    first[tid] = mine;
    if (tid == 0) count = 0;
    if (tid < 64) sorted[tid] = 0;
    __syncthreads();
    const u64 least = top_bound(first, p.top);
    // keys that reach the bound lie in at most top + 8 parts (fewer than top in all
    // where there is no bound): no more than the buffer holds
    for (int i = tid; i < p.parts * p.top; i += kThreads) {
      const u64 k = keys[i];
      if (!k || k < least) continue;
      const int at = atomicAdd(&count, 1);
      if (at < 72 * 64) reach[at] = k;
    }
    __syncthreads();
    const int n = min(count, 72 * 64);
    for (int i = tid; i < n; i += kThreads) {
      const u64 own = reach[i];
      int above = 0;
      for (int j = 0; j < n; ++j) above += reach[j] > own;
      if (above < p.top) sorted[above] = own;
    }
  }
  __syncthreads();
  if (tid < p.top) key = sorted[tid];
  s = wave_stats[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) s = join<E>(s, wave_stats[w]);
  row_outputs(p, row, (const E*)p.x + (long long)row * p.rstride, s, key);
}

// Parts of a row: enough for two workgroups per CU, each of at least 512 chunks.
int logprob_parts(long long rows, int n, int esize, int cus) {
  const long long chunks = ((long long)n * esize + 15) / 16;
  const long long parts = (2LL * cus + rows - 1) / rows, most = (chunks + 511) / 512;
  const long long r = parts < most ? parts : most;
  return (int)(r < 1 ? 1 : r > kThreads ? kThreads : r);
}

template <typename E>
static hipError_t dispatch(const LogprobParams& p, hipStream_t stream) {
  // Logits of more than the last cache holds are read past the caches (1000 rows of
  // 151936 fp32 logits 118 -> 106 us, 777 101 -> 92); fewer may still be there since
  // the linear that wrote them (512 rows of fp16 ones 45 us past the caches, 41 through
  // them; 300 rows 49 and 46).
  const bool stream_reads = (long long)p.rows * p.n * sizeof(E) > 256LL << 20;
  hipLaunchKernelGGL((stream_reads ? logprob_kernel<E, true> : logprob_kernel<E, false>),
                     dim3((unsigned)(p.rows * p.parts)), dim3(kThreads), 0, stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.parts == 1) return e;
  hipLaunchKernelGGL(logprob_join_kernel<E>, dim3((unsigned)p.rows), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

hipError_t logprob_launch(const LogprobParams& p, hipStream_t stream) {
  return p.f16 ? dispatch<f16>(p, stream) : dispatch<float>(p, stream);
}

}  // namespace aexq
