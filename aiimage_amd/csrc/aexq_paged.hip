// Operators on a paged key/value cache (gfx950): rotary positions with the
// append of packed tokens, and attention of one new token per sequence.
//
// The cache is a pool of fp16 pages [pages][heads_kv][page_size][head_dim]
// for K and one for V; position x of sequence s is row x % page_size of page
// table[s][x / page_size].  Lengths and tables live on the device, so a
// captured launch follows them from step to step.
#include <math.h>

#include "aexq_paged.hpp"

namespace aexq {

// ---------------------------------------------------------------------------
// Rotary positions and append.  One wave per packed token (or four, where there
// are few tokens): the cos and sin of a head's pairs go to its LDS once (pair j
// from the table row of its axis' position), then each lane moves 16-byte pieces,
// several on the way at a time: first those of eight pairs (j, j + rot/2) of a q
// or k head, then eight unrotated elements behind them, then eight of v, so that
// the lanes of a wave mostly do the same.
//   x'[j] = x[j] cos - x[j + rot/2] sin,  x'[j + rot/2] = x[j] sin + x[j + rot/2] cos
// in fp32, rounded once to fp16.  Memory bounds it.  Token t of a sequence with n new tokens and
// length L (after the append) lands at position L - n + (t - first).
// ---------------------------------------------------------------------------
template <int U>  // pieces of a lane on the way
__global__ __launch_bounds__(kThreads) void rope_append_kernel(const RopeAppendParams p) {
  __shared__ float table[kWaves][2][128];
  const int lane = threadIdx.x & 63, wave = sreg((int)threadIdx.x >> 6);
  const int index = blockIdx.x * kWaves + wave;
  const int t = index / p.waves, lead = index % p.waves * 64 + lane, step = 64 * p.waves;
  if (t >= p.tokens) return;  // (waves meet nowhere below)
  float* cs = table[wave][0];
  float* sn = table[wave][1];
  const int d = p.d, half = p.rot / 2;
  const int r8 = half / 8, c8 = (d - p.rot) / 8, heads = p.hq + p.kv.hkv;
  const int turns = heads * r8, copies = heads * c8, log8 = __builtin_ctz(d) - 3;
  const int total = turns + copies + (p.kv.hkv << log8);

  // piece id: its head (q's, then k's, then v's), its first element, and whether
  // that is turned with the one rot/2 behind it
  struct Place {
    int head, at;
    bool turn;
  };
  auto place = [&](int id) {
    Place x;
    x.turn = id < turns;
    if (x.turn) {
      x.head = r8 == 1 ? id : __umulhi(id, p.per_r8);
      x.at = 8 * (id - x.head * r8);
    } else if (id < turns + copies) {
      x.head = __umulhi(id - turns, p.per_c8);
      x.at = p.rot + 8 * (id - turns - x.head * c8);
    } else {
      const int e = id - turns - copies;
      x.head = heads + (e >> log8);
      x.at = 8 * (e & ((1 << log8) - 1));
    }
    return x;
  };
  u32x4 xa[U], xb[U];
  auto load = [&](int id, u32x4& a, u32x4& b) {
    id = min(id, total - 1);  // (a lane without a piece reads the last one)
    const Place x = place(id);
    const int kv = x.head - p.hq;
    const f16* row = kv < 0            ? p.q + (long long)t * p.q_stride + x.head * d
                     : kv < p.kv.hkv ? p.k + (long long)t * p.k_stride + kv * d
                                     : p.v + (long long)t * p.v_stride + (kv - p.kv.hkv) * d;
    a = *(const u32x4*)(row + x.at);
    b = a;
    if (x.turn) b = *(const u32x4*)(row + x.at + half);
  };
#pragma unroll
  for (int u = 0; u < U; ++u)  // before anything else is known of the token
    load(lead + step * u, xa[u], xb[u]);

  // where positions are given, the tables' rows wait for nothing else
  auto turn_by = [&](int pos) {
    for (int j = lane; j < half; j += 64) {
      int axis = 0, end = p.sections[0];
#pragma unroll
      for (int a = 1; a < 4; ++a) {
        if (p.interleaved) {
          if (j % p.axes == a && j < p.axes * p.sections[a]) axis = a;
        } else {
          if (a < p.axes && j >= end) axis = a;
          end += p.sections[a];
        }
      }
      int at = p.positions ? p.positions[(long long)axis * p.tokens + t] : pos;
      at = min(max(at, 0), p.rows - 1);
      cs[j] = p.cos_table[(long long)at * half + j];
      sn[j] = p.sin_table[(long long)at * half + j];
    }
  };
  const PackedRow own = packed_row(p.offsets, p.kv.lengths, p.kv.n, t);
  if (p.positions) turn_by(0);
  if (!own.found) return;  // rows behind the last sequence stay as they were
  // (a length below 0 is 0: its difference to a token does not wrap)
  const int pos = max(own.length, 0) - (own.end - t);
  // where its k and v rows go; nowhere outside the table or the pool
  int page = -1;
  if (pos >= 0 && pos < p.kv.width << p.kv.shift)
    page = p.kv.table[(long long)own.seq * p.kv.width + (pos >> p.kv.shift)];
  const bool keep = page >= 0 && page < p.kv.pages;
  const int row = pos & ((1 << p.kv.shift) - 1);
  if (!p.positions) turn_by(pos);
  // the wave's own LDS: its stores before its loads
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  // (stored past the caches: 46 us for the 214 MB above, 57 through them)
  auto store = [&](int id, const u32x4& xa, const u32x4& xb) {
    const Place x = place(id);
    const int kv = x.head - p.hq;
    if (id >= total || (kv >= 0 && !keep)) return;
    f16* to;
    if (kv < 0)
      to = p.q_out + (long long)t * p.q_out_stride + x.head * d;
    else if (kv < p.kv.hkv)
      to = p.kp + ((((long long)page * p.kv.hkv + kv) << p.kv.shift) + row) * d;
    else
      to = p.vp + ((((long long)page * p.kv.hkv + (kv - p.kv.hkv)) << p.kv.shift) + row) * d;
    to += x.at;
    if (!x.turn) {
      __builtin_nontemporal_store(xa, (u32x4*)to);
      return;
    }
    u32x4 lo, hi;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f16x2 a = as_h2(xa[e]), b = as_h2(xb[e]);
      f16x2 u, w;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float c = cs[x.at + 2 * e + i], z = sn[x.at + 2 * e + i];
        u[i] = (f16)((float)a[i] * c - (float)b[i] * z);
        w[i] = (f16)((float)a[i] * z + (float)b[i] * c);
      }
      lo[e] = as_u(u);
      hi[e] = as_u(w);
    }
    __builtin_nontemporal_store(lo, (u32x4*)to);
    __builtin_nontemporal_store(hi, (u32x4*)(to + half));
  };
  for (int id = lead;;) {
#pragma unroll
    for (int u = 0; u < U; ++u) store(id + step * u, xa[u], xb[u]);
    id += step * U;
    if (id - lead >= total) break;
#pragma unroll
    for (int u = 0; u < U; ++u) load(id + step * u, xa[u], xb[u]);
  }
}

hipError_t rope_append_launch(RopeAppendParams p, hipStream_t stream) {
  // four waves on a token shorten the way of one (4 tokens of 16/4 heads of 128: 3.9
  // us, one wave 5.3); a wave with several tokens' worth of loads on the way keeps
  // memory busy (17383 tokens of 8/2 heads of 256, 214 MB: 46 us, four waves 64; a
  // copy of as many bytes 43)
  p.waves = p.tokens <= 1024 ? kWaves : 1;
  const int r8 = p.rot / 16, c8 = (p.d - p.rot) / 8;
  // n / r8 of any piece is umulhi(n, per_r8): n stays below 2^32 / r8
  p.per_r8 = r8 > 1 ? 0xffffffffu / r8 + 1 : 0;
  p.per_c8 = c8 > 1 ? 0xffffffffu / c8 + 1 : 0;
  const int per = kWaves / p.waves;
  const dim3 grid((p.tokens + per - 1) / per);
  if (p.waves > 1)
    hipLaunchKernelGGL(rope_append_kernel<2>, grid, dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL(rope_append_kernel<6>, grid, dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Attention of one new token per sequence, out = softmax(scale q K^T) V, for
// the up to 16 query heads of a key/value head at a time (more take further
// blocks).  A wave takes 32 positions a step with both products on matrix
// instructions and K and V straight from the cache to registers:
//   S^T = K q^T   16 positions x 16 heads x 32 dims: lane (c = l % 16, g = l / 16)
//                 holds 8 dims of K row c; the result leaves lane (c, g) with
//                 head c's scores of positions 4 g + r (+ 16 in the second half);
//   O^T = V^T P^T those scores' weights are the right operand as they stand, if
//                 its k index 8 g + i is position 4 g + i (i < 4) or 16 + 4 g + i
//                 - 4.  So lane (c, g) loads D/16 consecutive dims of those 8 V
//                 rows (16 lanes cover a row) and v_perm turns the 8 rows x D/16
//                 dims into the left operands: product t has dims (D/16) m + t.
// The waves of a workgroup take steps in turn and meet in LDS at the end.
//
// What bounds it is reading K and V once (HBM): 7 sequences of 309146 positions, 2
// key heads of 256, 633 MB in 112 us (5.7 TB/s); 64 of 56891, 8 of 128, 234 MB in 44
// (5.4; 2.7 us of it to find the piece, and memory serves pieces of one length
// unevenly); one of 300 positions takes 6 us.
//
// Lengths may differ as they like and the host need not know them: where it pays, a
// (sequence, head block) longer than a share of all of them is cut into even pieces
// of kDecodeUnit positions and more, found on the device.  Pieces leave (max, sum,
// acc) rows that a second launch joins.
// ---------------------------------------------------------------------------
constexpr int kDecodeUnit = 128;
constexpr int kDecodeMost = 2048;  // pieces of a (sequence, head block)

// Two numbers that are added up together.
struct Two {
  int a, b;
};
__device__ __forceinline__ Two operator+(Two x, Two y) { return Two{x.a + y.a, x.b + y.b}; }
__device__ __forceinline__ Two operator-(Two x, Two y) { return Two{x.a - y.a, x.b - y.b}; }
__device__ __forceinline__ int shuffle_up(int v, int off) { return __shfl_up(v, off, 64); }
__device__ __forceinline__ Two shuffle_up(Two v, int off) {
  return Two{__shfl_up(v.a, off, 64), __shfl_up(v.b, off, 64)};
}

template <int D>
struct DecodeLds {
  static constexpr int HT = D / 16 < 8 ? D / 16 : 8;  // dims of a lane's run in one pass
  static constexpr int W = 16 * HT;                   // dims of one pass
  alignas(16) float o[kWaves][16][W + 4];
  float m[kWaves][16], l[kWaves][16];
  int seq, base, slot, units[kWaves];
  Two pieces[kWaves];
};

// One (sequence s, head block hb) over positions [p0, p1) of len, by the whole
// workgroup.  `slot` null: the output, else the partial rows.
template <int D>
__device__ __forceinline__ void decode_piece(const DecodePagedParams& p, DecodeLds<D>& lds, int s,
                                             int hb, int len, int p0, int p1, float* slot) {
  constexpr int KS = D / 32, DPL = D / 16, HT = DecodeLds<D>::HT, W = DecodeLds<D>::W;
  const int tid = threadIdx.x, lane = tid & 63, wave = sreg(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int h = hb / p.blocks, first = hb % p.blocks * 16;  // kv head, first query head of it
  const int live = min(16, p.group - first);
  const int mask = (1 << p.kv.shift) - 1;

  f16x8 qf[KS];
  {
    const f16* row = p.q + (long long)s * p.q_stride + (h * p.group + first + min(c, live - 1)) * D;
#pragma unroll
    for (int i = 0; i < KS; ++i)
      qf[i] = c < live ? *(const f16x8*)(row + 32 * i + 8 * g) : f16x8{};
  }
  f32x4 acc[DPL];
#pragma unroll
  for (int i = 0; i < DPL; ++i) acc[i] = f32x4{};
  float m = -INFINITY, l = 0.0f;

  for (int x = p0 + 32 * wave; x < p1; x += 32 * kWaves) {
    // the two blocks of 16 positions; a block past the end repeats the last one
    const int x1 = min(x + 16, (len - 1) & ~15);
    const long long r0 =
        (((long long)sreg(paged_page(p.kv, s, x >> p.kv.shift)) * p.kv.hkv + h) << p.kv.shift) +
        (x & mask);
    const long long r1 =
        (((long long)sreg(paged_page(p.kv, s, x1 >> p.kv.shift)) * p.kv.hkv + h) << p.kv.shift) +
        (x1 & mask);
    f16x8 k0[KS], k1[KS];
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      k0[i] = *(const f16x8*)(p.kv.k + r0 * D + c * D + 8 * g + 32 * i);
      k1[i] = *(const f16x8*)(p.kv.k + r1 * D + c * D + 8 * g + 32 * i);
    }
    uint32_t v[8][DPL / 2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const f16* row = p.kv.v + (i < 4 ? r0 : r1) * D + (4 * g + i % 4) * D + DPL * c;
      // Past the caches, where one load covers whole rows: 256 sequences of 1000 to
      // 3000 positions, 8 key heads of 128, 364 -> 332 us, of 100 to 1000 88 -> 72, 64
      // of 56891 together cold 59 -> 55, warm 48 -> 49.  The two loads of a row of 256
      // dims need its lines twice, as K's do (309146 positions cold 117 -> 120).
      if constexpr (DPL <= 8) {
        typedef uint32_t Run __attribute__((ext_vector_type(DPL / 2)));
        const Run run = __builtin_nontemporal_load((const Run*)row);
        __builtin_memcpy(v[i], &run, sizeof(run));
      } else {
        __builtin_memcpy(v[i], __builtin_assume_aligned(row, 2 * DPL), 2 * DPL);
      }
    }
    f32x4 s0 = f32x4{}, s1 = f32x4{};
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0[i], qf[i], s0, 0, 0, 0);
      s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1[i], qf[i], s1, 0, 0, 0);
    }
    float sc[8];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      sc[r] = s0[r] * p.scale2;
      sc[r + 4] = s1[r] * p.scale2;
    }
    if (x + 32 > len) {
      // rows past the end weigh 0 and, whatever the page holds there, read 0
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = x + (i < 4 ? 0 : 16) + 4 * g + i % 4 < len;
        sc[i] = in ? sc[i] : -INFINITY;
#pragma unroll
        for (int e = 0; e < DPL / 2; ++e) v[i][e] = in ? v[i][e] : 0u;
      }
    }
    float top = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])),
                      fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7])));
    if (__any(top > m + kLag)) {
      const float next = fmaxf(m, rows_max(top));
      const float f = exp2_fast(m - (next == -INFINITY ? 0.0f : next));
      l *= f;
#pragma unroll
      for (int i = 0; i < DPL; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][r] *= f;
      m = next;
    }
    // (where every score so far is -inf the weights are 0, not NaN)
    const float base = (m == -INFINITY ? 0.0f : m) - kLift;
    f16x8 w;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = exp2_fast(sc[i] - base);
      l += e;
      // the weights' one rounding below 32 bits, for products in fp16 (a second product
      // with what is left of them is NaN where v is infinite and nothing is left)
      w[i] = (f16)e;
    }
#pragma unroll
    for (int e = 0; e < DPL / 2; ++e) {
      u32x4 lo, hi;
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        lo[a] = __builtin_amdgcn_perm(v[2 * a + 1][e], v[2 * a][e], 0x05040100u);
        hi[a] = __builtin_amdgcn_perm(v[2 * a + 1][e], v[2 * a][e], 0x07060302u);
      }
      acc[2 * e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, lo), w,
                                                          acc[2 * e], 0, 0, 0);
      acc[2 * e + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, hi), w,
                                                              acc[2 * e + 1], 0, 0, 0);
    }
  }

  // the waves' (max, sum, acc) meet, D / (16 HT) passes of W dims
  l = rows_sum(l);
  if (lane < 16) {
    lds.m[wave][c] = m;
    lds.l[wave][c] = l;
  }
#pragma unroll
  for (int pass = 0; pass < DPL / HT; ++pass) {
    // acc[t][r] is dim DPL (4 g + r) + t of head c
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int t = 0; t < HT; t += 4) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = acc[pass * HT + t + e][r];
        *(f32x4*)&lds.o[wave][c][HT * (4 * g + r) + t] = y;
      }
    __syncthreads();
    for (int i = tid; i < live * (W / 4); i += kThreads) {
      const int q = i / (W / 4), y = i % (W / 4) * 4;
      float top = lds.m[0][q];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) top = fmaxf(top, lds.m[w][q]);
      const float base = top == -INFINITY ? 0.0f : top;
      f32x4 a = f32x4{};
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = exp2_fast(lds.m[w][q] - base);
        sum = fmaf(lds.l[w][q], f, sum);
        const f32x4 b = *(const f32x4*)&lds.o[w][q][y];
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = fmaf(b[e], f, a[e]);
      }
      const int dim = y / HT * DPL + pass * HT + y % HT;
      if (slot) {
        float* to = slot + q * (D + 4);
        *(f32x4*)(to + 4 + dim) = a;
        if (y == 0 && pass == 0) {
          to[0] = top;
          to[1] = sum;
        }
      } else {
        // (a sum of 0: every score was -inf, and the answer is NaN)
        const float inv = 1.0f / sum;
        f16x4 b;
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = average_f16(a[e] * inv);
        *(f16x4*)(p.out + (long long)s * p.out_stride + (h * p.group + first + q) * D + dim) = b;
      }
    }
    __syncthreads();
  }
}

// One workgroup per (head block, sequence), nothing to join.
template <int D>
__global__ __launch_bounds__(kThreads, D == 256 ? 2 : 4) void decode_paged_whole(const DecodePagedParams p) {
  __shared__ DecodeLds<D> lds;
  const int hb = blockIdx.x, s = blockIdx.y;
  const int len = paged_length(p.kv, s);
  if (len > 0) {
    decode_piece<D>(p, lds, s, hb, len, 0, len, nullptr);
    return;
  }
  const int h = hb / p.blocks, first = hb % p.blocks * 16, live = min(16, p.group - first);
  for (int i = threadIdx.x; i < live * D; i += kThreads)
    p.out[(long long)s * p.out_stride + (h * p.group + first) * D + i] = (f16)0.0f;
}

// A (sequence, head block) of `len` positions in even pieces of at most `share`
// units: their number, and the units of each but the last.
struct DecodeCut {
  int pieces, size;
  __device__ DecodeCut(int len, int share) {
    const int units = (len + kDecodeUnit - 1) / kDecodeUnit;
    pieces = (units + share - 1) / share;
    size = pieces ? (units + pieces - 1) / pieces : 0;
    pieces = size ? (units + size - 1) / size : 0;
  }
};

// Sum over the workgroup's threads, and of those before each.
template <typename T>
__device__ __forceinline__ T block_scan(T mine, T* waves, T* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T upto = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T v = shuffle_up(upto, off);
    if (lane >= off) upto = upto + v;
  }
  if (lane == 63) waves[wave] = upto;
  __syncthreads();
  T before = upto - mine, sum = T{};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before = before + waves[w];
    sum = sum + waves[w];
  }
  *total = sum;
  return before;
}

// A piece per workgroup.  plan[0] takes the share of units that is cut, plan[1 +
// s] the first slot of partial rows of sequence s, for the joining launch: only the
// pieces of what is cut have one, fewer than two for each share.  (That the last
// workgroup of a head block joins it in the same launch was slower: its rows then
// go past the L2s.  One sequence of 1000 positions 9.4 -> 12.9 us, 64 sequences of
// 56891 55 -> 63.)
template <int D>
__global__ __launch_bounds__(kThreads, D == 256 ? 2 : 4) void decode_paged_cut(
    const DecodePagedParams p) {
  __shared__ DecodeLds<D> lds;
  const int tid = threadIdx.x, n = p.kv.n, heads = p.kv.hkv * p.blocks;
  // thread t adds up its share of the sequences
  const int each = (n + kThreads - 1) / kThreads;
  const int s0 = min(tid * each, n), s1 = min(s0 + each, n);
  int units = 0, all;
  for (int s = s0; s < s1; ++s)
    units += (paged_length(p.kv, s) + kDecodeUnit - 1) / kDecodeUnit * heads;
  block_scan(units, lds.units, &all);
  const int share = max((all + p.target - 1) / p.target, 1);
  // the pieces of sequence s, and those of them that have a slot
  auto count = [&](int s) {
    const int m = DecodeCut(paged_length(p.kv, s), share).pieces;
    return Two{m * heads, m > 1 ? m * heads : 0};
  };
  Two pieces = {0, 0}, total;
  for (int s = s0; s < s1; ++s) pieces = pieces + count(s);
  const Two before = block_scan(pieces, lds.pieces, &total);
  if (blockIdx.x == 0 && tid == 0) p.plan[0] = share;
  const int at = blockIdx.x;
  if (at >= total.a) return;
  if (before.a <= at && at < before.a + pieces.a) {
    int s = s0;
    Two base = before;
    for (;; ++s) {
      const Two m = count(s);
      if (at < base.a + m.a) break;
      base = base + m;
    }
    lds.seq = s;
    lds.base = base.a;
    lds.slot = base.b;
    if (at == base.a) p.plan[1 + s] = base.b;
  }
  __syncthreads();
  const int s = sreg(lds.seq), len = paged_length(p.kv, s);
  const DecodeCut cut(len, share);
  const int mine = at - sreg(lds.base), hb = mine / cut.pieces, i = mine % cut.pieces;
  // (whatever the lengths do meanwhile, the rows written are the launch's own)
  const int slot = min(sreg(lds.slot) + mine, p.slots - 1);
  decode_piece<D>(p, lds, s, hb, len, i * cut.size * kDecodeUnit,
                  min(len, (i + 1) * cut.size * kDecodeUnit),
                  cut.pieces == 1 ? nullptr : p.part + (long long)slot * p.rows * (D + 4));
}

// Joins the partial rows of the (sequence, head)s that were cut:
// M = max m_i, out = sum acc_i 2^(m_i - M) / sum l_i 2^(m_i - M), the pieces'
// weights first, so that no row waits for another (5.6 us).  Also the zero rows of empty sequences.
template <int D>
__global__ __launch_bounds__(kThreads) void decode_paged_join(const DecodePagedParams p) {
  constexpr int T4 = D / 4, R = kThreads / T4;  // threads along a row, rows at a time
  __shared__ f32x4 sums[R][T4];
  __shared__ float weight[kDecodeMost], sum[kDecodeMost], tops[kWaves], parts[kWaves];
  const int head = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6, y = tid % T4, r = tid / T4;
  const int len = paged_length(p.kv, s), share = p.plan[0], slot = p.plan[1 + s];
  f16* out = p.out + (long long)s * p.out_stride + head * D;
  if (len == 0) {
    if (tid < T4) *(f16x4*)(out + 4 * y) = f16x4{};
    return;
  }
  // (whatever the plan holds, the rows read are the launch's own)
  const int h = head / p.group, q = head % p.group;
  const int pieces = DecodeCut(len, max(share, 1)).pieces;
  if (pieces == 1 || pieces > kDecodeMost) return;
  const long long first = max(slot, 0) + (h * p.blocks + q / 16) * (long long)pieces;
  if (first > p.slots - pieces) return;
  auto row = [&](int i) { return p.part + ((first + i) * p.rows + q % 16) * (D + 4); };
  // the first rows are on their way before the weights are known
  constexpr int U = 4;
  f32x4 o[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    o[u] = f32x4{};
    if (r + u * R < pieces) o[u] = *(const f32x4*)(row(r + u * R) + 4 + 4 * y);
  }
  float m = -INFINITY;
  for (int i = tid; i < pieces; i += kThreads) {
    const float2 ml = *(const float2*)row(i);
    weight[i] = ml.x;
    sum[i] = ml.y;
    m = fmaxf(m, ml.x);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
  if (lane == 0) tops[wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, tops[w]);
  const float base = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  for (int i = tid; i < pieces; i += kThreads) {  // (its own entries again)
    const float f = exp2_fast(weight[i] - base);
    weight[i] = f;
    l = fmaf(sum[i], f, l);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) l += __shfl_xor(l, off, 64);
  if (lane == 0) parts[wave] = l;
  __syncthreads();
  l = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) l += parts[w];
  f32x4 acc = f32x4{};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (r + u * R >= pieces) break;
    const float f = weight[r + u * R];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(o[u][e], f, acc[e]);
  }
#pragma unroll 4
  for (int i = r + U * R; i < pieces; i += R) {
    const f32x4 x = *(const f32x4*)(row(i) + 4 + 4 * y);
    const float f = weight[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(x[e], f, acc[e]);
  }
  sums[r][y] = acc;
  __syncthreads();
  if (r) return;
#pragma unroll
  for (int i = 1; i < R; ++i) {
    const f32x4 o = sums[i][y];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += o[e];
  }
  const float inv = 1.0f / l;
  f16x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = average_f16(acc[e] * inv);
  *(f16x4*)(out + 4 * y) = v;
}

// The cut of a launch over up to `bound` positions of each sequence in `blocks`
// head blocks of sequences: one piece for each `target`-th of all units, so that
// no more than blocks + target are there.  What is cut has more than one share, and
// less than two pieces for each: fewer than 2 target in all.  Nothing is cut (target
// 0) where the steps of a workgroup are few, and where there is a workgroup for every
// CU whose longest way is not much longer.
DecodePlan decode_paged_plan(int head_dim, int cus, long long bound, long long blocks) {
  DecodePlan r;
  r.target = bound <= 512 || (blocks >= cus && bound <= 1024) ? 0 : (head_dim == 256 ? 2 : 3) * cus;
  r.grid = blocks + r.target;
  r.slots = 2 * r.target;
  return r;
}

template <int D>
static hipError_t decode_launch(const DecodePagedParams& p, hipStream_t stream) {
  if (!p.target) {
    hipLaunchKernelGGL(decode_paged_whole<D>, dim3(p.kv.hkv * p.blocks, p.kv.n), dim3(kThreads), 0,
                       stream, p);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(decode_paged_cut<D>, dim3((unsigned)p.grid), dim3(kThreads), 0, stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(decode_paged_join<D>, dim3(p.kv.hkv * p.group, p.kv.n), dim3(kThreads), 0,
                     stream, p);
  return hipGetLastError();
}

hipError_t decode_paged_launch(const DecodePagedParams& p, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 64: return decode_launch<64>(p, stream);
    case 128: return decode_launch<128>(p, stream);
    default: return decode_launch<256>(p, stream);
  }
}

}  // namespace aexq
