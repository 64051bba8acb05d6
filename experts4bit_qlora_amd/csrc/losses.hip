// Launchers of the losses over the vocabulary's logits (losses.h).
#include "losses.h"

#include <algorithm>

namespace e4b {

namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// f(first row, rows) for all rows in order: a launch holds fewer than 2^32 work items, `per` workgroups of `threads` a row.
template <class F>
void by_launch(int64_t rows, int64_t per, int threads, F&& f) {
  const int64_t most = std::max<int64_t>(1, ((int64_t(1) << 32) - 1) / threads / per);
  for (int64_t first = 0; first < rows; first += most) f(first, std::min(most, rows - first));
}

template <int KIND, int DT>
void rows_of(const LossArgs& a, hipStream_t s) {
  if (a.parts) {
    const unsigned rows = static_cast<unsigned>(a.z.seqs * a.z.tokens);
    hipLaunchKernelGGL((loss_parts_kernel<KIND, DT>), dim3(rows * a.parts), dim3(kPartThreads), 0, s, a);
    hipLaunchKernelGGL((loss_rows_kernel<KIND, DT, 512, kRowUnroll, true>), dim3(rows), dim3(512), 0, s, a, int64_t(0));
    return;
  }
  const auto with = [&](auto nt) {
    by_launch(a.z.seqs * a.z.tokens, 1, nt(), [&](int64_t first, int64_t rows) {
      hipLaunchKernelGGL((loss_rows_kernel<KIND, DT, nt(), kRowUnroll, false>), dim3(static_cast<unsigned>(rows)), dim3(nt()), 0, s, a,
                         first);
    });
  };
  // Threads a row by its bytes, us by 128 / 256 / 512 / 1,024 threads: 5,500 rows of 1,000 bf16 logits 7.3 / 9.8 / 15 / 27; of
  // 8,000 23 / 23.5 / 28 / 45; of 32,000 76 / 69 / 69 / 85; of 50,257 114 / 109 / 106 / 105; of 128,000 283 / 269 / 268 / 253. 37
  // rows of 50,257: - / 7.4 / 6.3 / 6.4, of 128,000: - / 13.6 / 11.5 / 10.6.
  using std::integral_constant;
  const int64_t bytes = a.z.vocab * Piece<DT>::kBytes;
  if (bytes <= 4096) return with(integral_constant<int, 128>{});
  if (bytes <= 32768) return with(integral_constant<int, 256>{});
  if (bytes < 128000) return with(integral_constant<int, 512>{});
  with(integral_constant<int, 1024>{});
}

template <int KIND>
void rows_of(const LossArgs& a, hipStream_t s) {
  switch (a.z.dtype) {
    case E4B_FP32: return rows_of<KIND, E4B_FP32>(a, s);
    case E4B_BF16: return rows_of<KIND, E4B_BF16>(a, s);
    default: return rows_of<KIND, E4B_FP16>(a, s);
  }
}

template <int DT, bool TEACHER>
void backward_of(const LossBackwardArgs& a, hipStream_t s) {
  const int64_t parts = std::max<int64_t>(1, cdiv(a.z.vocab, int64_t(kBackThreads) * kBackUnroll * Piece<DT>::kCount));
  by_launch(a.z.seqs * a.z.tokens, parts, kBackThreads, [&](int64_t first, int64_t rows) {
    hipLaunchKernelGGL((loss_backward_kernel<DT, TEACHER>), dim3(static_cast<unsigned>(rows * parts)), dim3(kBackThreads),
                       0, s, a, first, static_cast<int>(parts));
  });
}

template <bool TEACHER>
void backward_of(const LossBackwardArgs& a, hipStream_t s) {
  switch (a.z.dtype) {
    case E4B_FP32: return backward_of<E4B_FP32, TEACHER>(a, s);
    case E4B_BF16: return backward_of<E4B_BF16, TEACHER>(a, s);
    default: return backward_of<E4B_FP16, TEACHER>(a, s);
  }
}

}  // namespace

// One CU takes ~7 us over the exponentials of 128,000 logits, so few long rows are shared by a workgroup per 8,192 logits and
// joined in a second launch, which costs the host 2.4 us with its workspace: rows where the GPU gains as much. Whole / split, us
// on the GPU: 1 row of 100,003 bf16 7.6 / 7.1, of 128,000 9.5 / 6.9 (a call: 8.4 / 10.7), of 152,000 10.3 / 6.9; 64 of 128,000
// 11.1 / 8.5, of 152,000 11.9 / 9.5; 128 of 152,000 12.4 / 12.4. fp32: 1 row of 50,257 5.8 / 5.6, of 80,000 8.1 / 5.8, of 128,000
// 10.7 / 5.7; 64 of 80,000 10.7 / 10.0, of 128,000 14.1 / 11.2; 128 of 128,000 16.2 / 16.6.
int loss_parts(const e4b_logits& z) {
  const int64_t bytes = z.vocab * (z.dtype == E4B_FP32 ? 4 : 2);
  return z.seqs * z.tokens <= 64 && bytes >= 300000 ? static_cast<int>(cdiv(z.vocab, kPartValues)) : 0;
}

void launch_loss_rows(LossKind kind, const LossArgs& a, hipStream_t s) {
  switch (kind) {
    case kStats: return rows_of<kStats>(a, s);
    case kScore: return rows_of<kScore>(a, s);
    case kLogprobs: return rows_of<kLogprobs>(a, s);
    case kPolicy: return rows_of<kPolicy>(a, s);
    default: return rows_of<kDistill>(a, s);
  }
}

// Both: groups and pairs number at most 2^21 (kLossMaxSeqs), so one launch holds their workgroups.
void launch_loss_mean(const MeanArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(loss_mean_kernel, dim3(static_cast<unsigned>(a.groups)), dim3(kJoin), 0, s, a);
}

void launch_pairs(const PairArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(pairs_kernel, dim3(static_cast<unsigned>(a.seqs / 2)), dim3(kJoin), 0, s, a);
}

void launch_loss_backward(const LossBackwardArgs& a, hipStream_t s) {
  if (a.index) return backward_of<true>(a, s);
  return backward_of<false>(a, s);
}

}  // namespace e4b
