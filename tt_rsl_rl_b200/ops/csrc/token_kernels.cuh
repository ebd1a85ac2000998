// Row-wise operators over the logits of a token policy: log-probabilities and entropies, the clipped policy loss with a
// KL term, the preference loss over pairs of sequences, and their gradients to the logits.
//
// With z a row of V logits, k = log2(e) / T, m = max z and s = sum_j 2^((z_j - m) k):
//   log p_j = (z_j - m) / T - ln s,   H = ln s - (sum_j 2^((z_j - m) k) (z_j - m) / T) / s.
// The maximum and the sums are held in fp32 and rescaled as the maximum grows, so a row is read once.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace rlb {

enum TokenDtype : int { kTokF32 = 0, kTokBF16 = 1, kTokF16 = 2 };
enum KlKind : int { kKl1 = 1, kKl2 = 2, kKl3 = 3 };
enum PrefKind : int { kPrefSigmoid = 0, kPrefHinge = 1, kPrefIpo = 2 };

// Rows of logits: row r starts at base + (r / inner) * stride_outer + (r % inner) * stride_inner elements.
struct TokenRows {
  void* base;
  int64_t inner, stride_outer, stride_inner;
};

// Tokens and weights of the rows. A row counts if its token lies in [0, V) and its weight is not zero; no other row's
// logits are read.
struct TokenIndex {
  const void* tokens;
  int tokens_i64;
  const void* mask;  // null: every weight is 1
  int mask_kind;     // 1: one byte (bool), 2: fp32 weights
};

struct PolicyTerms {
  const float *old_logp, *adv, *ref_logp;  // ref_logp may be null
  float clip_lo, clip_hi, kl_coef, entropy_coef;
  int kl_kind;
};

struct TokenStatsArgs {
  int dtype;
  int64_t rows, vocab;
  TokenRows z;
  TokenIndex idx;
  double inv_temp;
  float* logp;      // [rows]
  float* entropy;   // [rows]; null: not computed
  float2* ml;       // [rows] what token_grad needs; null: not stored
  const PolicyTerms* policy;  // null: log-probabilities only (host pointer, copied into the launch)
  float4* terms;    // [rows] weighted (surrogate, kl, entropy, clipped) with `policy`
  float2* coef;     // [rows] (dL/dlogp, dL/dH) times the row's weight, before division by the sum of weights
};
cudaError_t token_stats(const TokenStatsArgs& a, cudaStream_t stream);
// The statistics with `policy` and the gradient times scale (times *scale_device) in one pass; with `mean` the gradient is
// divided by the sum of the weights. `grad` rows start at the same places within 16 bytes as the logits' rows. Writes logp
// and terms. weight_sum: room for one number.
cudaError_t token_policy(const TokenStatsArgs& a, const TokenRows& grad, float scale, const float* scale_device, int mean,
                         double* weight_sum, cudaStream_t stream);

struct TokenGradArgs {
  int dtype;
  int64_t rows, vocab;
  TokenRows z, out;
  TokenIndex idx;
  double inv_temp;
  const float2* ml;
  const float* entropy;  // needed where b is given
  const float *a, *b;    // dL/dlogp and dL/dH of row r at a[r * a_stride], weights included; b may be null (no entropy term)
  int64_t a_stride, b_stride;
  float scale;
  const float *scale_a, *scale_b;  // optional factors on the device
};
cudaError_t token_grad(const TokenGradArgs& a, cudaStream_t stream);

// loss[0]; out[0..4] = surrogate, kl, entropy, clip fraction, factor that the gradients carry (1 / sum of weights, or 1).
struct PolicyFinishArgs {
  int64_t rows;
  const float4* terms;
  TokenIndex idx;
  int64_t vocab;
  float kl_coef, entropy_coef;
  int mean;
  float *loss, *out;
};
cudaError_t policy_finish(const PolicyFinishArgs& a, cudaStream_t stream);

struct PreferenceArgs {
  int64_t rows, vocab, seqs;  // sequences 2 k (chosen) and 2 k + 1 (rejected) form a pair
  const void* offsets;        // [seqs + 1] first row of each sequence; null: sequences of `length` rows
  int offsets_i64;
  int64_t length;
  TokenIndex idx;
  const float* logp;
  const float* ref;  // [seqs] or null (no reference)
  float beta, smoothing;
  int kind, average;
  float* loss;        // [1]
  float* seq_logp;    // [seqs]
  float* rewards;     // [2, seqs / 2]: of the chosen, of the rejected sequences
  float* coef;        // [rows] dL/dlogp; zero outside the sequences
};
cudaError_t preference_pairs(const PreferenceArgs& a, cudaStream_t stream);

}  // namespace rlb
