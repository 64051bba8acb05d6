// Launch-side view of the router kernels (gate.h), instantiated in gate.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace e4b {

constexpr int kGateMaxExperts = 1024;
constexpr int kGateMaxK = 64;

struct GateArgs {
  const void* logits;  // [T, E]
  int dtype;
  int64_t T;
  int E, k;
  int over_chosen;  // the softmax runs over the chosen logits only
  int64_t* index;   // [T, k]: written by the forward, read by the backward
  void* weights;    // [T, k] in wdtype: written by the forward; the backward's dL/dweights
  int wdtype;
  void* grad;       // backward: dL/dlogits [T, E] in dtype
};
void launch_gate(const GateArgs& a, hipStream_t s);
void launch_gate_backward(const GateArgs& a, hipStream_t s);

struct BalanceArgs {
  const void* logits;  // [L, T, E]
  int dtype;
  int64_t T;
  int L, E, k;
  const int64_t* index;  // [L, T, k]
  const uint8_t* mask;   // token t of layer l is valid iff mask[l * mask_stride + t] (NULL: all are)
  int64_t mask_stride;
  int chunks;            // token chunks per layer, a workgroup each
  float* part;           // [L, chunks, E] sums of the probabilities
  int32_t* part_counts;  // [L, chunks, E + 1] counts, then the valid tokens
  float* loss;           // [L]
  int64_t* counts;       // [L, E]
  int64_t* kept;         // [L, E], NULL without tokens: the same, in the workspace
  int64_t* valid;        // [L] valid tokens
  const float* grad_loss;  // backward: [L]
  void* grad;              // backward: [L, T, E] in dtype
};
int balance_chunks(int64_t T, int L, int E);
void launch_balance(const BalanceArgs& a, hipStream_t s);
void launch_balance_backward(const BalanceArgs& a, hipStream_t s);

}  // namespace e4b
