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
  // Threads a row by its bytes, us by 128 / 256 / 512 / 1,024 threads for 1,000 rows and for 5,500, bf16 logits read from
  // memory (log-probabilities that a backward follows):
  //     4,096 bytes   4.1 /  4.3 /  4.8 /  6.9     9.1 / 10.9 / 18.8 / 30.9
  //     6,000         4.7 /  4.7 /  5.1 /  7.2    11.4 / 13.1 / 20.2 / 33.0
  //    32,768         8.8 /  8.8 /  9.0 / 11.6    34.7 / 32.1 / 32.5 / 54.3
  //    48,000        12.3 / 12.3 / 11.9 / 13.9    50.1 / 47.7 / 46.1 / 62.9
  //   114,688        22.3 / 22.9 / 22.6 / 24.1     112 /  107 /  106 /  103
  //   144,000        27.8 / 28.2 / 27.3 / 27.3     140 /  135 /  132 /  127
  //   256,000        46.3 / 47.8 / 46.7 / 46.1     246 /  235 /  232 /  224
  // fp32 rows of 114,688 bytes 21.8 / 22.1 / 22.0 / 22.8 and 109 / 106 / 105 / 102, of 128,000 25.0 / 24.8 / 24.4 / 25.4 and 123 /
  // 119 / 116 / 112 (a training call over 2,400 of them, what the caches hold read from there: 156 by 512, 153 by 1,024), of
  // 160,000 30.0 / 30.2 / 30.0 / 29.1 and 152 / 148 / 145 / 140; a preference's statistics, bf16, 114,688 bytes 23.6 / 24.5 / 25.7 /
  // 26.8 and 118 / 112 / 110 / 120, 128,000 27.4 / 27.4 / 28.4 / 29.6 and 132 / 125 / 122 / 130, 160,000 32.6 / 34.2 / 34.9 / 33.8
  // and 163 / 155 / 153 / 147. 37 rows of 100,514 bytes 10.0 / 6.9 / 5.6 / 5.9, of 256,000 19.3 / 12.2 / 10.0 / 9.5. Up to 300 rows
  // 512 threads gain 0.6 us at 16,000 bytes already (5.4 -> 4.7), where 5,500 rows lose 6 (21.7 -> 27.6).
  using std::integral_constant;
  const int64_t bytes = a.z.vocab * Piece<DT>::kBytes;
  if (bytes <= 4096) return with(integral_constant<int, 128>{});
  if (bytes <= 32768) return with(integral_constant<int, 256>{});
  if (bytes < 122880) return with(integral_constant<int, 512>{});
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

// One CU takes ~7 us over the exponentials of 100,000 logits, so few long rows are shared by a workgroup per 8,192 logits and
// joined in a second launch, which with its workspace costs the host as much as the GPU gains on rows below this border. Whole /
// split, us on the GPU, 1 / 37 / 64 rows: bf16 of 80,000 6.8 / 6.4, 7.2 / 7.9, 7.8 / 8.7; of 128,000 8.9 / 6.2, 10.4 / 8.0, 10.6 /
// 8.5; of 152,000 9.7 / 6.5, 11.1 / 8.4, 11.1 / 9.5; fp32 of 80,000 7.6 / 6.2, 9.9 / 8.3, 10.4 / 9.7; of 100,003 7.9 / 6.3, 10.6 /
// 8.2, 11.3 / 10.1; of 128,000 9.6 / 6.3, 12.9 / 9.2, 13.9 / 11.2; 128 rows gain nothing below 262,144 logits. A call whose rows
// are split takes 10.2 us of host time, so for 1 / 8 / 37 / 64 rows a call takes at bf16 of 149,999 (whole) 9.3 / 9.5 / 9.6 / 10.0
// and of 150,000 (split) 9.8 / 10.2 / 9.8 / 9.9; at fp32 of 99,999 (whole) 7.9 / 8.2 / 9.1 / 9.3 and of 100,000 (split) 9.7 / 10.1 /
// 9.9 / 9.8, while of 75,000 split ones took 10.2 / 10.3 / 10.1 / 10.0 and whole ones 6.8 / 7.2 / 7.4 / 7.4: fp32 rows, half as
// many logits to the byte, are split from 400,000 bytes on. A captured call, which waits for the GPU alone, would gain from
// 200,000 on.
int loss_parts(const e4b_logits& z) {
  const bool wide = z.dtype == E4B_FP32;
  const int64_t bytes = z.vocab * (wide ? 4 : 2);
  return z.seqs * z.tokens <= 64 && bytes >= (wide ? 400000 : 300000) ? static_cast<int>(cdiv(z.vocab, kPartValues)) : 0;
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
