// Host/device definitions of the recurrent layers and of drafted tokens (not part of
// the ABI).
#pragma once

#include "aexq_internal.hpp"

namespace aexq {

// The sequences of a call and their states (aexq_slots).
struct SlotsView {
  const int32_t *slot, *lengths, *counts;  // [n], each may be null
  int count, n, store;
};
// ---- short causal convolution (aexq_mixer.hip)
struct ShortConvParams {
  SlotsView slots;
  _Float16* state;  // [count][width - 1][channels]
  const int32_t* offsets;
  int tokens, channels, width, silu;
  const _Float16* x;
  _Float16* out;  // may be null
  long long x_stride, out_stride;
  const float *weight, *bias;  // [channels][width], [channels] or null
};
long long conv_groups(int tokens, int sequences, int channels);  // workgroups at most
hipError_t short_conv_launch(const ShortConvParams& p, hipStream_t stream);
// ---- root-mean-square norm of heads, gated by silu (aexq_mixer.hip)
struct GatedNormParams {
  const _Float16 *x, *z;
  _Float16* out;
  long long x_stride, z_stride, out_stride;
  const float* gamma;  // [dim] or null
  long long rows;      // tokens * heads
  int heads, dim;
  float eps;
};
long long gated_norm_groups(long long rows, int dim);  // workgroups
hipError_t gated_norm_launch(const GatedNormParams& p, hipStream_t stream);
// ---- the gated delta rule (aexq_delta.hip)
struct DeltaParams {
  SlotsView slots;
  float* state;            // [count][hv][dk][dv]
  const int32_t* offsets;  // null: row s is sequence s
  int tokens, hk, hv, group, dk, dv;
  const _Float16 *q, *k, *v, *a, *b;
  _Float16* out;  // may be null
  long long q_stride, k_stride, v_stride, a_stride, b_stride, out_stride;
  const float *a_log, *dt_bias;
  float scale, eps;
  // of each block of 64 rows (aexq_rows.hpp), scratch: per value head the matrices
  // T and P and the rows' factors, per key head keys, queries and the keys transposed
  char* heads;
  char* keys;
  int* longs;  // sequences of more than 16 rows, their number first; null: not apart
};
// Scratch of a block and value head: six (16 rows, 32 columns) pieces of T and as many of
// P, each in two fp16 parts of 1 KB; four factors a row and the block's decay.  Of a block
// and key head: three times its rows.
constexpr int kDeltaRows = 64;
constexpr int kDeltaEnd = 16;  // rows of a last block that go through one row tile
constexpr int kDeltaFactors = 24 * 1024;
constexpr int kDeltaHead = kDeltaFactors + 4 * kDeltaRows * 4 + 64;
constexpr int delta_key_bytes(int dk) { return 3 * dk * kDeltaRows * 2; }
bool delta_splits(const DeltaParams& p, int cus);
hipError_t delta_prompt_launch(const DeltaParams& p, hipStream_t stream);
hipError_t delta_decode_launch(const DeltaParams& p, int cus, hipStream_t stream);
// ---- drafted tokens against the target's probabilities (aexq_verify.hip)
constexpr int kVerifyParts = 64;   // parts of a row at most: a lane each
constexpr int kVerifyRuns = 256;   // runs of a sampled row at most: a thread each
// The draft behind a row, its logit, and what its probability has to pass (+inf where it
// is none).
struct VerifyDraft {
  double need;
  float x;
  int token;
};
struct VerifyParams {
  const void* x;  // [rows][rstride] logits, n of each row
  int f16;
  long long rstride;
  int rows, n;
  const int32_t* offsets;
  int sequences;
  const int32_t* drafts;     // [rows]
  const float* probs;        // [rows][probs_stride], or null
  long long probs_stride;
  const float* temperature;  // [sequences] or null
  const float *accept_u, *sample_u;
  int32_t *counts, *tokens;
  int parts, cols;    // parts of a row in the first pass, 16-byte chunks of each
  int runs, run;      // runs of a sampled row, and values of each
  int blocks;         // workgroups that sum the runs of a sequence
  // scratch: of each (row, part) the sum of weights, the largest logit and its
  // index; of each row its draft; of each sequence's sampled row the runs' sums, all
  // of it and without the draft's probabilities; what was decided
  double* z;
  float* m;
  int* at;
  VerifyDraft* draft;
  double2* sums;  // [sequences][runs]
  int4* plan;    // row, mode, greedy token, accepted rows
  double2* norm; // largest logit and sum of weights of the sampled row
};
int verify_parts(long long rows, int n, int esize, int cus);
int verify_runs(int n);
int verify_blocks(int sequences, int runs, int cus);
hipError_t verify_launch(const VerifyParams& p, hipStream_t stream);

}  // namespace aexq
