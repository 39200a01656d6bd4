// Attention over prompts (gfx950): packed sequences of different lengths,
// grouped heads, causal or over whole sequences, K and V packed like q or in a
// paged cache (whose last rows the queries then are).
#include <math.h>

#include <type_traits>

#include "aexq_paged.hpp"

namespace aexq {

// ---------------------------------------------------------------------------
// out = softmax(scale q K^T over what a row sees) V, in one pass over K and V
// with a running maximum and sum per row.
//
// The rows of a sequence and kv head are its (token, query head of the group)
// pairs, token by token: row r is token r / group, head r % group.  A workgroup
// takes 128 of them, 32 to a wave, so one K/V tile in LDS serves every head of
// the group and short prompts still fill the tile.  Tiles of KT positions are
// fetched LDS-direct, one ahead, 16-byte chunks of a row exchanged by swz() so
// that neither product's reads meet in LDS banks.
//   S^T = K q^T   32 positions x 32 rows x 16 dims a product: q stays in
//                 registers as the right operand; lane (j = l % 32, h = l / 32)
//                 ends with row j's scores of positions 8 (i / 4) + 4 h + i % 4;
//   O^T = V^T P^T takes the weights as they stand as its right operand when its
//                 k index 8 h + i is position 8 (i / 4) + 4 h + i % 4 of 16; the
//                 left operand is V transposed on the way out of LDS
//                 (ds_read_b64_tr_b16), 4 positions of 16 dims per 16 lanes.
// So scores, weights, maximum and sum of a row never leave its two lanes.
//
// What bounds it: the matrix instructions, and what the two waves of a SIMD do not
// cover for each other.  16384 causal tokens of 32/8 heads of 128 take 2015 to 2064 us
// (1.07 PFLOP/s): the matrix units are busy 61% of the time, at 1.66 GHz, where
// products and nothing else keep them busy at 1.39 GHz, the power's limit (1.45
// PFLOP/s).  8192 of 16/4 heads take 290 us (940 TFLOP/s; 64 wide 177 and 256 wide 760
// us).  4 x 512 tokens after 6143 take 231 us; the same products alone, without reads,
// exponentials and loads, 191.  Exponentials put
// between the products of the next tile, and loads between products, were no faster
// for that (254 and 239 us).  Short prompts wait: some 7 us of a workgroup's time go
// to finding its rows, its first tile, the masked tile and its stores.
//
// Where a launch has few 128-row tiles for the part, or tiles of very different
// length, a launch of 5 to 6 us before it lays out its work (prompt_plan): tiles longer
// than a share of the whole are cut along the positions, and the longest pieces
// start first (4 x 512 tokens after up to 16000: 280 -> 126 us).  The pieces of a cut
// tile leave their (max, sum, acc) registers in scratch and are added up in a tree of
// fixed shape.
// Otherwise every workgroup finds its tile from the offsets, last tiles first.
// ---------------------------------------------------------------------------
constexpr int kPromptRows = 128;
constexpr int kPlanThreads = 1024;
constexpr int kPromptLeast = 6;  // units (KT positions) that a cut leaves at least, about
constexpr int kPlanMost = 2048;  // sequences, and tiles of a kv head, that are laid out

// A sequence as the kernels see it, clamped to what the call holds.
struct PromptSeq {
  int q0, rows, queries;  // first query row; (query, head of the group) rows; queries
  int kv0, len;           // first key row (packed), positions
};
__device__ __forceinline__ int prompt_first(const PromptParams& p, int s) {
  return min(max(p.q_offsets[s], 0), p.tokens);
}
__device__ __forceinline__ int prompt_rows(const PromptParams& p, int s) {
  const int a = prompt_first(p, s);
  return (min(max(p.q_offsets[s + 1], a), p.tokens) - a) * p.group;
}
template <bool PAGED>
__device__ __forceinline__ PromptSeq prompt_seq(const PromptParams& p, int s) {
  PromptSeq q;
  q.q0 = prompt_first(p, s);
  q.rows = prompt_rows(p, s);
  q.queries = q.rows / p.group;
  if constexpr (PAGED) {
    q.kv0 = 0;
    q.len = paged_length(p.kv, s);
  } else {
    q.kv0 = min(max(p.kv_offsets[s], 0), p.kv_tokens);
    q.len = min(max(p.kv_offsets[s + 1], q.kv0), p.kv_tokens) - q.kv0;
  }
  return q;
}
// Positions that the token of row r sees.
__device__ __forceinline__ int prompt_seen(const PromptParams& p, const PromptSeq& q, int r) {
  return p.causal ? max(q.len - q.queries + r / p.group + 1, 0) : q.len;
}

// A piece of work: tiles [t0, t1) of positions for a 128-row tile of a sequence.
// pieces > 1: it leaves registers in slot `slot`, those of its tile are in
// slot0 .. slot0 + pieces - 1 (per kv head).
struct PromptPiece {
  int seq, tile, t0, t1, slot, slot0, pieces, pad;
};

// Lays out the pieces of every kv head, one workgroup: plan[0] their number, then
// the pieces from plan + 4 by falling length; and clears the tiles' counters.
template <bool PAGED>
__global__ __launch_bounds__(kPlanThreads) void prompt_plan_kernel(const PromptParams p, int kt) {
  constexpr int kBuckets = 256, kW = kPlanThreads / 64;
  // of each sequence: the tiles before it, its rows, and where its queries start
  // among its positions (causal) or its length
  __shared__ int before[kPlanMost + 1], rows[kPlanMost], from[kPlanMost];
  __shared__ int bucket[kBuckets], waves[kW], tops[kW], slots;
  __shared__ unsigned long long sums[kW];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int carry = 0;
  for (int b = 0; b < p.n; b += kPlanThreads) {
    const int s = b + tid;
    int mine = 0;
    if (s < p.n) {
      const PromptSeq q = prompt_seq<PAGED>(p, s);
      rows[s] = q.rows;
      from[s] = p.causal ? q.len - q.queries : q.len;
      mine = (q.rows + kPromptRows - 1) / kPromptRows;
    }
    int upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(upto, off, 64);
      if (lane >= off) upto += v;
    }
    if (b) __syncthreads();
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      if (w < wave) upto += waves[w];
      sum += waves[w];
    }
    if (s < p.n) before[s] = carry + upto - mine;
    carry += sum;
  }
  for (int i = tid; i < p.slots * p.columns; i += kPlanThreads) p.counters[i] = 0;
  if (tid < kBuckets) bucket[tid] = 0;
  if (tid == 0) slots = 0;
  __syncthreads();
  const int tiles = carry;  // (the first kPlanMost of them: two a thread)
  int seq[2], cost[2] = {0, 0};
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = tid + u * kPlanThreads;
    if (i >= tiles) continue;
    int a = 0, b = p.n;  // the last sequence with before[s] <= i
    while (b - a > 1) {
      const int m = (a + b) / 2;
      if (before[m] <= i) a = m; else b = m;
    }
    const int last = min((i - before[a] + 1) * kPromptRows, rows[a]) - 1;
    const int seen = p.causal ? max(from[a] + last / p.group + 1, 0) : from[a];
    seq[u] = a;
    cost[u] = (seen + kt - 1) / kt;
  }
  unsigned long long units = (unsigned long long)cost[0] + cost[1];
  int longest = max(cost[0], cost[1]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    units += __shfl_xor(units, off, 64);
    longest = max(longest, __shfl_xor(longest, off, 64));
  }
  if (lane == 0) {
    sums[wave] = units;
    tops[wave] = longest;
  }
  __syncthreads();
  units = 0;
#pragma unroll
  for (int w = 0; w < kW; ++w) {
    units += sums[w];
    longest = max(longest, tops[w]);
  }
  // the share of a workgroup, where the part's workgroups all have one
  const int share =
      max(kPromptLeast, (int)min((units * p.columns + p.target - 1) / p.target, 0x7fffffffULL));
  const int most = min(share, max(longest, 1));
  int pieces[2], size[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if (tid + u * kPlanThreads >= tiles) continue;
    pieces[u] = max(1, (cost[u] + share - 1) / share);
    size[u] = max(1, (cost[u] + pieces[u] - 1) / pieces[u]);
    pieces[u] = max(1, (cost[u] + size[u] - 1) / size[u]);
    atomicAdd(&bucket[max(0, kBuckets - 1 - (int)((long long)size[u] * (kBuckets - 1) / most))],
              pieces[u]);
  }
  __syncthreads();
  if (tid < 64) {  // where each bucket's pieces start
    int own[kBuckets / 64], sum = 0;
#pragma unroll
    for (int i = 0; i < kBuckets / 64; ++i) {
      own[i] = sum;
      sum += bucket[tid * (kBuckets / 64) + i];
    }
    int upto = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(upto, off, 64);
      if (lane >= off) upto += v;
    }
#pragma unroll
    for (int i = 0; i < kBuckets / 64; ++i) bucket[tid * (kBuckets / 64) + i] = upto - sum + own[i];
    if (tid == 63) p.plan[0] = upto;
  }
  __syncthreads();
  PromptPiece* out = (PromptPiece*)(p.plan + 4);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = tid + u * kPlanThreads;
    if (i >= tiles) continue;
    int at = atomicAdd(
        &bucket[max(0, kBuckets - 1 - (int)((long long)size[u] * (kBuckets - 1) / most))],
        pieces[u]);
    const int slot = pieces[u] > 1 ? atomicAdd(&slots, pieces[u]) : 0;
    // (offsets that decrease may ask for more than the call's rows need: left out)
    for (int k = 0; k < pieces[u] && at < p.pieces; ++k, ++at)
      out[at] = PromptPiece{seq[u], i - before[seq[u]], k * size[u],
                            min((k + 1) * size[u], cost[u]), slot + k, slot, pieces[u], 0};
  }
}

template <int D>
struct PromptLds {
  static constexpr int KT = D == 256 ? 32 : 64;
  static constexpr int DV = D == 256 ? 128 : D;  // dims of V and of the output it takes
  alignas(1024) f16 k[2][KT * D];
  alignas(1024) f16 v[2][KT * DV];
  int seq, tile, count[kWaves];
  int odd[2][kWaves];  // a V tile holds an infinity or a NaN
};

// Where chunk c of row r of a tile lies: chunk c ^ swz(r) of that row.
template <int D>
__device__ __forceinline__ int swz(int r) {
  if constexpr (D == 64) return (r >> 1 & 1) << 2 | (r >> 2 & 3);
  return (r & 3) << 2 | (r >> 2 & 3);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
// Of each 16 lanes, lane i reads 4 elements at its address; together a 4 x 16
// block, row i / 4, columns 4 (i % 4) ..; lane i gets column i.
__device__ __forceinline__ f16x4 read_transposed(const f16* p) {
  return __builtin_bit_cast(
      f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}

template <int D, bool PAGED>
__global__ __launch_bounds__(kThreads, D == 64 ? 3 : 2) void prompt_kernel(const PromptParams p) {
  constexpr int KT = PromptLds<D>::KT, DV = PromptLds<D>::DV;
  constexpr int KS = D / 16, DB = DV / 32, SB = KT / 32;
  // tile rows of one LDS-direct load, and loads of a wave per tile, of K and of V
  constexpr int RK = 512 / D, NK = KT / 4 / RK, RV = 512 / DV, NV = KT / 4 / RV;
  __shared__ PromptLds<D> lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = sreg(tid >> 6);
  // (DV < D: the heads' output in parts, a workgroup each)
  const int n = p.n, group = p.group, column = blockIdx.x, head = column / (D / DV);
  const int dv0 = column % (D / DV) * DV;

  // 1. the workgroup's sequence, tile and positions
  int seq, tile;
  PromptPiece piece{};
  if (p.plan) {
    if ((int)blockIdx.y >= p.plan[0]) return;
    piece = ((const PromptPiece*)(p.plan + 4))[blockIdx.y];
    // (whatever the plan holds, reads and writes stay within the call's own rows)
    seq = min(max(sreg(piece.seq), 0), n - 1);
    tile = max(sreg(piece.tile), 0);
    if (tile * (long long)kPromptRows >= prompt_rows(p, seq)) return;
    piece.pieces = sreg(piece.pieces);
    piece.slot0 = min(max(sreg(piece.slot0), 0), max(p.slots - piece.pieces, 0));
    if (piece.pieces > p.slots) return;
    piece.slot = min(max(sreg(piece.slot), piece.slot0), piece.slot0 + max(piece.pieces, 1) - 1);
  } else {
    const int share = (n + kThreads - 1) / kThreads;
    const int sa = min(tid * share, n), sb = min(sa + share, n);
    int mine = 0;
    for (int s = sa; s < sb; ++s) mine += (prompt_rows(p, s) + kPromptRows - 1) / kPromptRows;
    int upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(upto, off, 64);
      if (lane >= off) upto += v;
    }
    if (lane == 63) lds.count[wave] = upto;
    __syncthreads();
    int before = upto - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) before += lds.count[w];
      total += lds.count[w];
    }
    const int at = total - 1 - (int)blockIdx.y;
    if (at < 0) return;
    if (before <= at && at < before + mine) {
      int s = sa, base = before;
      for (;; ++s) {
        const int u = (prompt_rows(p, s) + kPromptRows - 1) / kPromptRows;
        if (at < base + u) break;
        base += u;
      }
      lds.seq = s;
      lds.tile = at - base;
    }
    __syncthreads();
    seq = sreg(lds.seq);
    tile = sreg(lds.tile);
  }
  const PromptSeq sq = prompt_seq<PAGED>(p, seq);
  const int q0 = sq.q0, rows = sq.rows, kv0 = sq.kv0, len = sreg(sq.len);
  auto seen = [&](int r) { return prompt_seen(p, sq, r); };

  // 2. q: the lane's row as the right operand of S^T
  const int j = lane & 31, h = lane >> 5;
  const int row = tile * kPromptRows + wave * 32 + j, last = rows - 1;
  const int rr = min(row, last);  // rows past the end repeat the last one, and store nothing
  const long long token = q0 + rr / group;
  const int qh = head * group + rr % group;
  f16x8 qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s)
    qf[s] = *(const f16x8*)(p.q + token * p.q_stride + qh * D + 16 * s + 8 * h);
  const int vis = seen(rr);
  // what the wave's rows see at most, and the workgroup's at least and at most
  const int hi = sreg(seen(min(tile * kPromptRows + wave * 32 + 31, last)));
  const int low = sreg(seen(tile * kPromptRows));
  const int most = sreg(seen(min(tile * kPromptRows + kPromptRows - 1, last)));
  const int begin = max(sreg(piece.t0), 0), all = (most + KT - 1) / KT;
  const int tiles = p.plan ? min(sreg(piece.t1), all) : all;
  const bool live = tile * kPromptRows + wave * 32 <= last;  // the wave has a row

  f32x16 o[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i) o[i] = f32x16{};
  float m = -INFINITY, l = 0.0f;

  // A wave's rows of a tile lie in one block of 16 positions, so in one page: a
  // uniform base and an offset of each lane's own, the same for every tile.  Rows past
  // the sequence's end lie past the resource's and read zeros.
  const int r0 = wave * (KT / 4);
  const int kst = PAGED ? D * 2 : (int)p.k_stride * 2, vst = PAGED ? D * 2 : (int)p.v_stride * 2;
  uint32_t koff[NK], voff[NV];
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const int r = i * RK + lane / (D / 8);
    koff[i] = r * kst + 16 * (lane % (D / 8) ^ swz<D>(r0 + r));
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int r = i * RV + lane / (DV / 8);
    voff[i] = r * vst + 16 * (lane % (DV / 8) ^ swz<DV>(r0 + r));
  }
  const uint32_t lds_base = lds_addr(&lds);
  auto fetch = [&](int t, int b) {
    const int x = min(t * KT + r0, len - 1), keep = min(max(len - t * KT - r0, 0), KT / 4);
    const f16 *kb, *vb;
    if constexpr (PAGED) {
      const long long a =
          ((((long long)sreg(paged_page(p.kv, seq, x >> p.kv.shift)) * p.kv.hkv + head)
            << p.kv.shift) + (x & ((1 << p.kv.shift) - 1))) * D;
      kb = p.kv.k + a;
      vb = p.kv.v + a + dv0;
    } else {
      kb = p.k + (long long)(kv0 + x) * p.k_stride + head * D;
      vb = p.v + (long long)(kv0 + x) * p.v_stride + head * D + dv0;
    }
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)sreg(kb), (short)0, sreg(keep * kst), kBufferRsrcWord3);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)sreg(vb), (short)0, sreg(keep * vst), kBufferRsrcWord3);
    const uint32_t kl = lds_base + (b * KT + r0) * D * 2;
    const uint32_t vl = lds_base + 2 * KT * D * 2 + (b * KT + r0) * DV * 2;
#pragma unroll
    for (int i = 0; i < NK; ++i) dma<16>(kr, kl + i * 1024, koff[i]);
#pragma unroll
    for (int i = 0; i < NV; ++i) dma<16>(vr, vl + i * 1024, voff[i]);
  };

  // Where the lane's operands lie in a tile: step s of K (16 dims), and of V the
  // four positions z of 16 and the 32 dims i (the 16-dim half tg, lane ti of 16).
  // Everything else of an address is the instruction's own offset.
  // (step s + 8 lies 16 chunks behind step s: swz() exchanges the low 4 bits)
  constexpr int KA = KS < 8 ? KS : 8;
  int kat[KA], vat[2][DB];
#pragma unroll
  for (int s = 0; s < KA; ++s) kat[s] = j * D + 8 * ((2 * s + h) ^ swz<D>(j));
#pragma unroll
  for (int z = 0; z < 2; ++z)
#pragma unroll
    for (int i = 0; i < DB; ++i) {
      const int tg = lane >> 4 & 1, ti = lane & 15, r = 8 * z + 4 * h + ti / 4;
      vat[z][i] = r * DV + 8 * ((2 * tg + (ti & 3) / 2) ^ (4 * i) ^ swz<DV>(r)) + 4 * (ti & 1);
    }

  // The arrival of tile t in buffer b, and the next one on its way.  EDGE: some row
  // of the workgroup does not see all of it.
  auto arrive = [&](int t, int b, auto edge) {
    constexpr bool EDGE = decltype(edge)::value;
    // The wave's rows of tile t are there, and its reads of tile t - 1 are done: the
    // compiler may leave a product, and the wait for its operands, behind the
    // barrier, after which the others' next rows overwrite that buffer.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    if constexpr (EDGE) {
      // An infinity or a NaN in V reaches, through 0 * V, the rows that do not
      // see it: each wave looks through the rows it fetched.
      float z = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const u32x4 y =
            *(const u32x4*)((const char*)lds.v[b] + r0 * DV * 2 + i * 1024 + lane * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) z = dot2(y[e], 0u, z);
      }
      const bool odd = __any(z != 0.0f);
      if (lane == 0) lds.odd[b][wave] = odd;
      wait_lgkm0();
    }
    bar();
    if (t + 1 < tiles) fetch(t + 1, b ^ 1);
  };
  // The wave's products with it.  `buf`: its buffer where the code is for one of
  // them, else -1.
  auto take = [&](int t, auto edge, auto buf) {
    constexpr bool EDGE = decltype(edge)::value;
    constexpr int BUF = decltype(buf)::value;
    const int b = BUF >= 0 ? BUF : (t - begin) & 1, x0 = t * KT;
    arrive(t, b, edge);
    if (EDGE && x0 >= hi) return;  // none of the wave's rows sees any of it

    f32x16 sc[SB];
#pragma unroll
    for (int i = 0; i < SB; ++i) sc[i] = f32x16{};
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < SB; ++i) {
        const f16x8 kf = *(const f16x8*)&lds.k[b][32 * i * D + s / KA * 128 + kat[s % KA]];
        sc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[s], sc[i], 0, 0, 0);
      }
    if constexpr (BUF >= 0) {
      // eight K reads ahead of the products that take them
      constexpr int N = KS * SB, AHEAD = N < 8 ? N : 8;
      __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
      for (int i = 0; i < N - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
    }
    if constexpr (EDGE) {
      const int left = vis - x0 - 4 * h;
#pragma unroll
      for (int i = 0; i < SB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          sc[i][r] = 32 * i + 8 * (r / 4) + r % 4 < left ? sc[i][r] : -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < SB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, sc[i][r]);
    top *= p.scale2;
    if (__any(top > m + kLag)) {
      const float next = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
      const float f = exp2_fast(m - (next == -INFINITY ? 0.0f : next));
      l *= f;
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] *= f;
      m = next;
    }
    const float base = (m == -INFINITY ? 0.0f : m) - kLift;
#pragma unroll
    for (int i = 0; i < SB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        sc[i][r] = exp2_fast(fmaf(sc[i][r], p.scale2, -base));
        l += sc[i][r];
      }
    if (EDGE && (lds.odd[b][0] | lds.odd[b][1] | lds.odd[b][2] | lds.odd[b][3])) {
      // position by position, for the rows that see it
      for (int x = 0; x < KT && x0 + x < hi; ++x) {
        float w = 0.0f;
#pragma unroll
        for (int i = 0; i < SB; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (32 * i + 8 * (r / 4) + r % 4 + 4 * h == x) w = sc[i][r];
        // (the half that does not hold position x has 0)
        w += __shfl_xor(w, 32, 64);
        const bool in = x0 + x < vis;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int d = 32 * i + 8 * (r / 4) + 4 * h + r % 4;
            const f16 y = lds.v[b][x * DV + 8 * ((d / 8) ^ swz<DV>(x)) + d % 8];
            o[i][r] = in ? fmaf(w, (float)y, o[i][r]) : o[i][r];
          }
      }
      return;
    }
#pragma unroll
    for (int y = 0; y < KT / 16; ++y) {
      // The weights' one rounding below 32 bits: the products take fp16, and a second one
      // with what is left of the weights would be half as many again, and NaN where v is
      // infinite and nothing is left.
      f16x8 w;
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = (f16)sc[y / 2][8 * (y % 2) + i];
#pragma unroll
      for (int i = 0; i < DB; ++i) {
        f16x4 a[2];
#pragma unroll
        for (int z = 0; z < 2; ++z) a[z] = read_transposed(&lds.v[b][16 * y * DV + vat[z][i]]);
        const f16x8 vf = __builtin_shufflevector(a[0], a[1], 0, 1, 2, 3, 4, 5, 6, 7);
        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, w, o[i], 0, 0, 0);
      }
    }
  };
  if (tiles > begin) fetch(begin, 0);
  wait_vm<0>();  // q too: the loops below then wait for no load but the tiles'
  const int whole = min(low / KT, tiles);
  int t = begin;
  if (live) {
    for (; t + 1 < whole; t += 2) {
      take(t, std::false_type{}, std::integral_constant<int, 0>{});
      take(t + 1, std::false_type{}, std::integral_constant<int, 1>{});
    }
    for (; t < tiles; ++t) take(t, std::true_type{}, std::integral_constant<int, -1>{});
  } else {  // it only fetches its rows
    for (; t + 1 < whole; ++t) arrive(t, (t - begin) & 1, std::false_type{});
    for (; t < tiles; ++t) arrive(t, (t - begin) & 1, std::true_type{});
  }

  if (piece.pieces > 1) {
    // The pieces of a tile meet in pairs, pairs of pairs and so on: of two siblings
    // the second to finish adds the first one's registers, [wave][four of them]
    // [lane] in its slot, and goes on with the sum.  They travel through coherent
    // stores and loads, the stores done before the count.  The sums do not depend
    // on who is second.
    constexpr int REGS = DB * 16 + 4;
    float* slots = p.part + (long long)column * p.slots * (kThreads * REGS);
    auto slot = [&](int i) {
      return __builtin_amdgcn_make_buffer_rsrc(
          (void*)sreg(slots + (long long)((piece.slot0 + i) * kWaves + wave) * (64 * REGS)),
          (short)0, 64 * REGS * 4, kBufferRsrcWord3);
    };
    const int own = piece.slot - piece.slot0;
    for (int step = 1; step < piece.pieces; step *= 2) {
      const int node = own / step, right = (node | 1) * step;
      if (right >= piece.pieces) continue;  // no sibling
      if (live) {
        const __amdgpu_buffer_rsrc_t to = slot(node * step);
#pragma unroll
        for (int i = 0; i < DB * 4; ++i) {
          const f32x4 y = {o[i / 4][i % 4 * 4], o[i / 4][i % 4 * 4 + 1], o[i / 4][i % 4 * 4 + 2],
                           o[i / 4][i % 4 * 4 + 3]};
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), to,
                                                 (i * 64 + lane) * 16, 0, kCoherent);
        }
        const f32x4 y = {m, l, 0.0f, 0.0f};
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), to,
                                               (DB * 4 * 64 + lane) * 16, 0, kCoherent);
      }
      wait_vm<0>();
      __syncthreads();
      if (tid == 0)
        lds.seq = atomicAdd(&p.counters[column * p.slots + piece.slot0 + right], 1);
      __syncthreads();
      if (sreg(lds.seq) == 0) return;
      if (live) {
        const __amdgpu_buffer_rsrc_t from = slot((node ^ 1) * step);
        auto read = [&](int i) {
          return __builtin_bit_cast(
              f32x4,
              __builtin_amdgcn_raw_buffer_load_b128(from, (i * 64 + lane) * 16, 0, kCoherent));
        };
        const f32x4 ml = read(DB * 4);
        f32x4 y[DB * 4];
#pragma unroll
        for (int i = 0; i < DB * 4; ++i) y[i] = read(i);
        const float top = fmaxf(m, ml[0]), base = top == -INFINITY ? 0.0f : top;
        const float f = exp2_fast(m - base), g = exp2_fast(ml[0] - base);
        m = top;
        // the lower half first, whichever of the two this is
        const bool low = !(node & 1);
        auto add = [&](float x, float y) {
          return low ? fmaf(y, g, x * f) : fmaf(x, f, y * g);
        };
        l = add(l, ml[1]);
#pragma unroll
        for (int i = 0; i < DB * 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            o[i / 4][i % 4 * 4 + e] = add(o[i / 4][i % 4 * 4 + e], y[i][e]);
      }
    }
    if (!live) return;
  }

  // 3. the row's two lanes hold half of its sum each; a row that sees nothing is
  // 0, one whose every score was -inf (a sum of 0) NaN
  l += __shfl_xor(l, 32, 64);
  const float inv = vis > 0 ? 1.0f / l : 0.0f;
  if (row > last) return;  // (a row's two lanes both)
  f16* out = p.out + token * p.out_stride + qh * D + dv0;
  // dims 8 r + 4 h .. of a lane become 16 bytes, 8 r .. of even r in the lower lane of
  // the row, of odd r in the upper one
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int r = 0; r < 4; r += 2) {
      f16x4 a, b;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = average_f16(o[i][4 * r + e] * inv);
        b[e] = average_f16(o[i][4 * r + 4 + e] * inv);
      }
      const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
      const auto u = __builtin_amdgcn_permlane32_swap(x.x, y.x, false, false);
      const auto w = __builtin_amdgcn_permlane32_swap(x.y, y.y, false, false);
      const u32x4 z = {u[0], w[0], u[1], w[1]};
      *(u32x4*)(out + 32 * i + 8 * (r + h)) = z;
    }
}

// Tiles that the rows of `tokens` packed tokens in n sequences need at most.
long long prompt_tiles(long long tokens, int n, int group) {
  return tokens * group / kPromptRows + n;
}

// Whether a launch is laid out first, over sequences of up to `bound` positions
// each: not where the layout would find nothing to cut or to order.
bool prompt_planned(long long tiles, int n, long long bound) {
  return n <= kPlanMost && tiles <= kPlanMost && bound > 512;
}
PromptScratch prompt_scratch(long long tiles, int hkv, int head_dim, int cus) {
  PromptScratch r;
  const int dv = head_dim == 256 ? 128 : head_dim;
  r.columns = hkv * (head_dim / dv);
  // A tile of c units is cut into pieces of at least share / 2, share >= units /
  // target: no more than 2 target pieces of cut tiles in all.  Two workgroups have a
  // place on a CU; shares for 1, 5/4, 3/2 and 2 per CU took 139, 135, 131 and 145 us
  // (4 x 512 tokens after up to 16000) and 55.8, 54.4, 55.2 and 58.2 (12 prompts).
  r.target = 3 * cus / 2;
  r.slots = (2 * r.target + r.columns - 1) / r.columns;
  r.pieces = tiles + r.slots;
  r.plan_ints = 4 + r.pieces * (long long)(sizeof(PromptPiece) / 4);
  r.counters = (long long)r.slots * r.columns;
  r.part_floats = r.counters * kThreads * (dv / 2 + 4);
  return r;
}

template <int D, bool PAGED>
static hipError_t prompt_dispatch(const PromptParams& p, unsigned rows, hipStream_t stream) {
  if (p.plan) {
    hipLaunchKernelGGL(prompt_plan_kernel<PAGED>, dim3(1), dim3(kPlanThreads), 0, stream, p,
                       PromptLds<D>::KT);
    // (the next launch would run on the layout and the counters of an earlier call, and
    // clear this error)
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((prompt_kernel<D, PAGED>), dim3(p.hkv * (D / PromptLds<D>::DV), rows),
                     dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

hipError_t prompt_launch(const PromptParams& p, int head_dim, long long pieces,
                         hipStream_t stream) {
  const unsigned rows = (unsigned)pieces;
  const bool paged = p.kv.k;
  switch (head_dim) {
    case 64: return (paged ? prompt_dispatch<64, true> : prompt_dispatch<64, false>)(p, rows, stream);
    case 128: return (paged ? prompt_dispatch<128, true> : prompt_dispatch<128, false>)(p, rows, stream);
    default: return (paged ? prompt_dispatch<256, true> : prompt_dispatch<256, false>)(p, rows, stream);
  }
}

}  // namespace aexq
