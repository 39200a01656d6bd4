// Host/device definitions of the operators for many sequences (not part of the ABI).
#pragma once

#include "aexq_internal.hpp"

namespace aexq {

// ---- a paged key/value cache (aexq_paged.hip, aexq_prompt.hip)
struct PagedView {
  const _Float16 *k, *v;    // [pages][hkv][1 << shift][head_dim]
  const int32_t* table;     // [n][width]
  const int32_t* lengths;   // [n]
  int pages, shift, width, n, hkv;
};
// rotary positions of packed q and k rows, k and v rows into their pages
struct RopeAppendParams {
  PagedView kv;
  _Float16 *kp, *vp;  // the pools, for writing
  const int32_t* offsets;
  int tokens, hq, d;
  const _Float16 *q, *k, *v;
  _Float16* q_out;
  long long q_stride, k_stride, v_stride, q_out_stride;
  const float *cos_table, *sin_table;  // [rows][rot / 2]
  const int32_t* positions;            // [axes][tokens]; null: the cache positions
  int rows, rot, axes, interleaved, sections[4];
  // set by the launch: waves of a token, and 2^32 over the pieces of a head
  int waves;
  uint32_t per_r8, per_c8;
};
hipError_t rope_append_launch(RopeAppendParams p, hipStream_t stream);
// attention of one row per sequence; heads go in blocks of up to 16 of a group
struct DecodePagedParams {
  PagedView kv;
  const _Float16* q;
  _Float16* out;
  long long q_stride, out_stride;
  int group, blocks;  // query heads per kv head, and their blocks of 16
  float scale2;       // scale * log2(e)
  int target;         // shares of the work that is cut; 0: nothing is cut
  int grid;           // pieces at most
  int slots, rows;    // of those of what is cut, and query heads of a block at most
  float* part;        // a slot's partial rows, each of head_dim + 4 floats
  int* plan;          // 1 + n ints
};
struct DecodePlan {
  int target, slots;
  long long grid;
};
DecodePlan decode_paged_plan(int head_dim, int cus, long long bound, long long blocks);
hipError_t decode_paged_launch(const DecodePagedParams& p, int head_dim, hipStream_t stream);
// attention of packed rows over packed (kv.k null) or paged keys and values
struct PromptParams {
  PagedView kv;
  const _Float16 *q, *k, *v;
  _Float16* out;
  long long q_stride, k_stride, v_stride, out_stride;
  const int32_t *q_offsets, *kv_offsets;  // [n + 1]
  int n, tokens, kv_tokens, hkv, group, causal;
  float scale2;
  // where the launch is laid out first (else plan is null): its pieces, and the
  // registers of cut tiles, `slots` for each column (kv head, or part of one)
  int* plan;
  float* part;
  int* counters;
  int target, columns, slots, pieces;
};
// what that takes: pieces of a kv head at most, and scratch
struct PromptScratch {
  int target, columns, slots;
  long long pieces, plan_ints, counters, part_floats;
};
long long prompt_tiles(long long tokens, int n, int group);
bool prompt_planned(long long tiles, int n, long long bound);
PromptScratch prompt_scratch(long long tiles, int hkv, int head_dim, int cus);
// `pieces`: workgroups of a kv head
hipError_t prompt_launch(const PromptParams& p, int head_dim, long long pieces,
                         hipStream_t stream);
// ---- log probabilities of tokens (aexq_logprobs.hip)
struct LogprobParams {
  const void* x;  // [rows][rstride] logits, n of each row
  int f16;
  long long rows, rstride;
  int n;
  const int32_t* tokens;    // [rows]
  float *logprob, *entropy;  // [rows], each may be null
  int top;                  // alternatives, at most 64
  int32_t* ids;             // [rows][top]
  float* values;            // [rows][top]
  int parts, cols;          // workgroups a row, 16-byte chunks of each
  float* stats;             // parts > 1: 4 floats and top keys per (row, part)
  unsigned long long* keys;
};
int logprob_parts(long long rows, int n, int esize, int cus);
hipError_t logprob_launch(const LogprobParams& p, hipStream_t stream);

}  // namespace aexq
