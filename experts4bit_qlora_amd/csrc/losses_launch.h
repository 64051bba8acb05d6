// Launch-side view of the losses over the vocabulary's logits (losses.h), instantiated in losses.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/e4b_amd.h"

namespace e4b {

constexpr int kLossMaxTop = 1024;
constexpr int64_t kLossMaxSeqs = int64_t(1) << 21;
constexpr int64_t kLossMaxVocab = int64_t(1) << 30;  // a row's indexes stay in 32 bits

constexpr int kPartValues = 8192;  // of a split row
// What a part of a row leaves in the workspace: s 2^n the sum of its exponentials (kStats; the others' sums are fp32 alone).
struct LossPart {
  double s;
  float n;
};

// Parts of a row in the forward: 0 (a workgroup takes the whole) or the workgroups that share it.
int loss_parts(const e4b_logits& z);

// What a token's loss is made of.
// kScore: log-probabilities that no backward follows; kStats: the same, in 64 bits and into stats alone.
enum LossKind { kStats = 0, kLogprobs = 1, kPolicy = 2, kDistill = 3, kScore = 4 };

struct LossArgs {
  e4b_logits z;
  float2 k;         // log2(e) / temperature, its high and low part
  int parts;        // loss_parts(z)
  float* logps;     // [R] log-probabilities of the labels, 0 where a token does not count (kLogprobs, kScore, kPolicy)
  // [R] (reference, sum of the row's exponentials against it, label's log-probability in two parts: the second for kStats only);
  // (0, -1, 0, 0) where a token does not count
  float4* stats;
  // kPolicy
  const float* old_logps;   // [R]
  const float* advantages;  // [seqs] or [R]
  int adv_per_token;
  const float* ref_logps;  // [R] or NULL
  float clip_lo, clip_hi, kl_coef;
  // kDistill
  const void* teacher;  // [R, top] in teacher_dtype
  int teacher_dtype;
  const int64_t* index;  // [R, top]
  int top;
  float* share;  // [R, top] the teacher's probabilities
  // kPolicy, kDistill
  float* token_loss;  // [R]
  float* coef;        // [R] dloss_t / dlogp_t (kPolicy)
};
void launch_loss_rows(LossKind kind, const LossArgs& a, hipStream_t s);

// loss[i] = mean of token_loss over the counted tokens of group i, inv[i] = 1 / their number (0 where none counts)
struct MeanArgs {
  const float* token_loss;
  const float4* stats;
  int64_t groups, per;  // groups of `per` consecutive tokens
  float* loss;
  float* inv;
};
void launch_loss_mean(const MeanArgs& a, hipStream_t s);

struct PairArgs {
  int64_t seqs, tokens;  // the first half of the sequences are the chosen ones
  const float4* stats;
  const void* ref;  // [R], [seqs] or NULL
  int ref_kind;     // e4b_reference
  int kind;  // e4b_preference
  float beta, smoothing;
  int average;
  float* loss;     // [seqs / 2]
  float* rewards;  // [seqs]
  float* coef;     // [seqs] dloss / d(a token's log-probability)
};
void launch_pairs(const PairArgs& a, hipStream_t s);

struct LossBackwardArgs {
  e4b_logits z;
  float2 k;
  const float4* stats;
  // a token's derivative: grad_loss[n, t] * coef[n, t] * inv[n], each at its own strides; coef and inv may be NULL
  const float* grad_loss;
  int64_t grad_seqs, grad_ns, grad_ts;  // sequence n has that of n mod grad_seqs
  const float* coef;
  int64_t coef_ns, coef_ts;
  const float* inv;
  int64_t inv_ns;
  float slope;            // times this: 1 / temperature, for the teacher's -temperature
  const int64_t* index;   // teacher: [R, top]; NULL: one label a token
  const float* share;     // [R, top]
  int top;
  void* grad;  // [R, vocab] in the logits' dtype
};
void launch_loss_backward(const LossBackwardArgs& a, hipStream_t s);

}  // namespace e4b
