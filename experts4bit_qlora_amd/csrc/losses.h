// Losses over the vocabulary: log-probabilities of labels, preference pairs, the clipped policy loss, distillation
// from a teacher's top logits, forward and backward.
//
// A row of logits z [V] at temperature tau: y = z / tau, m = max z, s = sum_j exp((z_j - m) / tau),
// q_j = exp((z_j - m) / tau) / s, and for its label l
//   lp = (z_l - m) / tau - log s,                    dlp / dz_j = ([j = l] - q_j) / tau.
// Policy, r = exp(lp - old):  loss = -min(r A, clip(r) A) + kl (e^x - x - 1), x = ref - lp,
//   dloss / dlp = -A r [r A <= clip(r) A] + kl (1 - e^x).
// Teacher with probabilities p_k at the indices i_k:  loss = tau^2 sum_k p_k (log p_k - log q_{i_k}),
//   dloss / dz_j = tau (q_j - sum of p_k with i_k = j).
// With rest = sum over j != l of exp((z_j - z_l) / tau), lp = -log(1 + rest) keeps its precision where the label is nearly
// certain, and so does the label's derivative 1 - q_l = 1 - e^lp: the label is left out of its row's sum.
// Preference, S = sum of a sequence's lp (or their mean), d = (S_c - r_c) - (S_r - r_r):  a loss of d, whose slope is
// every chosen token's dloss / dlp and, negated, every rejected one's.
//
// One workgroup takes a row: its threads sum over 16-byte pieces, the sums are joined; a row's logits are read once in the
// forward and once in the backward, tokens that do not count are not read.
//
// Bound by HBM from a few hundred rows on: 5,369 counted of 8,192 rows of 128,000 bf16 logits take 222 us forward (6.2 TB/s,
// the vector units 80 % busy) and 575-585 us backward (1.4 GB in, 2.1 GB out: 6.0 TB/s, where a copy reaches 4.9). Computing
// the gradient while the forward holds the row would save the second read, but what the loss is multiplied by is known only in
// the backward: a third fewer bytes where that is exactly one, a third more where it is not.
#pragma once

#include "common.h"
#include "losses_launch.h"

namespace e4b {

constexpr float kLowest = -3.402823466e38f;

// ---- 16-byte pieces of a row

template <int DT>
struct Piece {
  static constexpr int kBytes = DT == E4B_FP32 ? 4 : 2;
  static constexpr int kCount = 16 / kBytes;
  using T = std::conditional_t<DT == E4B_FP32, float, uint16_t>;

  static E4B_DEV float one(T v) {
    if constexpr (DT == E4B_FP32) return v;
    else return to_f<DT>(v);
  }
  static E4B_DEV T round(float f) {
    if constexpr (DT == E4B_FP32) return f;
    else return from_f<DT>(f);
  }
  static E4B_DEV void unpack(const uint4& v, float (&f)[kCount]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == E4B_FP32) {
        f[i] = __uint_as_float(w[i]);
      } else {
        f[2 * i] = lo_f<DT>(w[i]);
        f[2 * i + 1] = hi_f<DT>(w[i]);
      }
    }
  }
  static E4B_DEV uint4 pack(const float (&f)[kCount]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == E4B_FP32) w[i] = __float_as_uint(f[i]);
      else w[i] = pack2(from_f<DT>(f[2 * i]), from_f<DT>(f[2 * i + 1]));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// A row as `head` single values up to the first 16-byte address, `pieces` whole pieces, and what is left.
template <int DT>
struct Split {
  int head, pieces, tail;  // tail: index of the first value behind the pieces
  E4B_DEV Split(const void* p, int n) {
    constexpr int C = Piece<DT>::kCount;
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15) / Piece<DT>::kBytes;
    head = min(n, (C - off) & (C - 1));
    pieces = (n - head) / C;
    tail = head + pieces * C;
  }
};

// 16 bytes at any address that the type's values may have, and to an aligned one, past the caches: logits that are read for the
// last time, gradients, which are as large. Backward of 1,500 x 128,000 bf16: 143 -> 122 us (the stores alone 125), of
// 5,500 x 50,257 184 -> 185, of 252 x 50,257 13.7 -> 12.2. A forward that no backward follows: 5,500 x 128,000 232 -> 214, 252 x
// 50,257 9.6 -> 10.0; one that a backward follows leaves it what the caches hold (both, 5,500 x 128,000: 668 -> 682).
E4B_DEV uint4 load16_once(const void* p) {
  typedef uint32_t Any __attribute__((ext_vector_type(4), aligned(2)));
  const Any v = __builtin_nontemporal_load(static_cast<const Any*>(p));
  return make_uint4(v.x, v.y, v.z, v.w);
}
E4B_DEV void store16_once(uint4* p, const uint4& v) {
  typedef uint32_t Vec __attribute__((ext_vector_type(4)));
  __builtin_nontemporal_store(Vec{v.x, v.y, v.z, v.w}, reinterpret_cast<Vec*>(p));
}

// ---- sums over a row

// k = log2(e) / temperature in two parts: with one, the exponents of all rows are off the same way by 2^-25 or so of
// their size, which a sequence's sum of log-probabilities adds up (820 tokens: 2e-4). The first has 12 bits, so that what the
// second adds to x k.x - n is not below that's last bit: rounded away, it would be missing as if there were one part.
E4B_DEV float times(float d, float2 k) { return __builtin_fmaf(d, k.x, d * k.y); }
E4B_DEV float exp_of(float d, float2 k) { return __builtin_amdgcn_exp2f(times(d, k)); }

constexpr int kRowUnroll = 4;  // pieces in flight per thread
constexpr int kPartThreads = 256;
template <int DT>
constexpr int kPartPieces = kPartValues / Piece<DT>::kCount;

// f(values) over a row, without its element `skip` if SKIP, by NT threads, of its pieces [begin, end) alone where it is
// split (the first of the parts takes the single values at the row's ends); -inf in the place of what is skipped. ready() is
// called once the first pieces are on their way.
template <int DT, int NT, int U, bool ONCE, bool SKIP, class G, class F>
E4B_DEV void over_row(const void* row, int V, int skip, int begin, int end, G&& ready, F&& f) {
  using P = Piece<DT>;
  const typename P::T* p = static_cast<const typename P::T*>(row);
  const Split<DT> at(row, V);
  const int tid = threadIdx.x;
  // the skipped element's piece (one that no thread takes where it is none) and its place there
  const int skip_at = skip < at.head ? -1 : (skip - at.head) / P::kCount, skip_off = (skip - at.head) % P::kCount;
  auto take = [&](const uint4& w, int i) {
    float x[P::kCount];
    P::unpack(w, x);
    if (SKIP && __any(i == skip_at)) {  // a branch of the wave: under a lane's mask the selections would cost every piece
#pragma unroll
      for (int c = 0; c < P::kCount; ++c)
        if (i == skip_at && c == skip_off) x[c] = -__builtin_inff();
    }
    f(x);
  };
  const uint4* v = reinterpret_cast<const uint4*>(p + at.head);
  const int last = min(end, at.pieces);
  int i = begin + tid;
  uint4 w[U];
  auto load = [&] {
    const bool all = i + (U - 1) * NT < last;
    if (all) {
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = ONCE ? load16_once(v + i + u * NT) : v[i + u * NT];
    }
    return all;
  };
  bool more = load();
  ready();
  while (more) {
#pragma unroll
    for (int u = 0; u < U; ++u) take(w[u], i + u * NT);
    i += U * NT;
    more = load();
  }
  for (; i < last; i += NT) take(v[i], i);
  if (begin == 0) {
    float edge[2] = {-__builtin_inff(), -__builtin_inff()};
    if (tid < at.head && !(SKIP && tid == skip)) edge[0] = P::one(p[tid]);
    if (tid < V - at.tail && !(SKIP && at.tail + tid == skip)) edge[1] = P::one(p[at.tail + tid]);
    f(edge);
  }
}

E4B_DEV float wave_sum(float v) {
#pragma unroll
  for (int off = 1; off < kWave; off *= 2) v += __shfl_xor(v, off);
  return v;
}

// sum_j exp((z_j - ref) / tau) by the whole workgroup, in every lane; ref is the row's element `first`, which
// is left out if SKIP: a logit that is likely among the largest, not the maximum. fp32 has 2^126 of room on either side, so a
// maximum kept while the sum runs, with a rescaling at every step, is only needed where a row leaves that room (Run). It
// costs two multiply-adds a value, x k.x - ref k and x k.y added to it; the rounding of ref k is taken out of the sum. With a
// running maximum / so, us, before the label's selection became a branch: 5,500 rows of 128,000 bf16 logits 268 / 253, of 50,257
// 111 / 106; 37 rows of 128,000 13.6 / 10.6, of 50,257 7.8 / 6.3 (the reference is loaded behind a row's first pieces: before
// them 5 % more).
template <int DT, int NT, int U, bool ONCE, bool SKIP>
E4B_DEV float row_sum(const void* row, int V, int first, float& ref, float2 k, int begin = 0, int end = 0x7fffffff) {
  float at, s = 0.0f;
  const auto ready = [&] {
    ref = Piece<DT>::one(static_cast<const typename Piece<DT>::T*>(row)[first]);
    at = times(ref, k);
  };
  over_row<DT, NT, U, ONCE, SKIP>(row, V, first, begin, end, ready, [&](const auto& x) {
    float sum = 0.0f;
    for (float v : x) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(v, k.y, __builtin_fmaf(v, k.x, -at)));
    s += sum;
  });
  s = wave_sum(s * __builtin_amdgcn_exp2f(-__builtin_fmaf(ref, k.y, __builtin_fmaf(ref, k.x, -at))));
  if constexpr (NT > kWave) {
    constexpr int W = NT / kWave;
    __shared__ float part[W];
    if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = s;
    __syncthreads();
    s = part[threadIdx.x & (W - 1)];
#pragma unroll
    for (int off = 1; off < W; off *= 2) s += __shfl_xor(s, off);
  }
  return s;
}

// Whether a row's reference, scaled, and its sum kept to that room (a NaN does not). Up to this reference the two parts of a
// product, 2^-11 of it, are added to within 1e-6; up to this sum the backward's quotient by it is a normal number.
E4B_DEV bool in_room(float ref, float2 k, float sum) { return fabsf(ref * k.x) < 65536.0f && sum < 1e18f; }

// A sum s of 2^(x k - n) whose reference n is the running maximum of x k rounded up to a whole number: the largest terms' exponents
// are the smallest, and so are their roundings, and a change of the reference is exact. Sequences' sums are made of these
// (kStats): a rescaling by a rounded exponential is 3e-9 too small in the mean, and a row's ten of them added up over 2,048
// tokens to 3e-6 of their ratio; the label as reference rounds the largest terms (60 tokens: 1.4e-6). Lanes, waves and a split
// row's parts are joined in 64 bits: in 32 a part's 8,192 logits lose up to 3e-8 of their sum. 8,192 rows of 128,000: 229 us,
// against 222 with row_sum and 240 with a running maximum that is no power of two.
constexpr float kNoPower = -1e30f;  // nothing summed yet
template <class S>
struct PowerOf {
  float n = kNoPower;
  S s = 0;
  static E4B_DEV S scaled(S v, float by) {  // by: a whole number, not positive
    const int e = static_cast<int>(fmaxf(by, -2000.0f));
    if constexpr (sizeof(S) == 8) return __builtin_amdgcn_ldexp(v, e);
    else return __builtin_amdgcn_ldexpf(v, e);
  }
  E4B_DEV void join(float on, S os) {
    const float to = fmaxf(n, on);
    s = scaled(s, n - to) + scaled(os, on - to);
    n = to;
  }
  E4B_DEV void join_lanes(int lanes) {
    for (int off = 1; off < lanes; off *= 2) join(__shfl_xor(n, off), __shfl_xor(s, off));
  }
  template <int N>
  E4B_DEV void add(const float (&x)[N], float2 k) {
    float most = x[0], sum = 0.0f;
    for (float v : x) most = fmaxf(most, v);
    const float to = fmaxf(n, __builtin_ceilf(times(most, k)));
    for (float v : x) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(v, k.y, __builtin_fmaf(v, k.x, -to)));
    s = scaled(s, n - to) + sum;
    n = to;
  }
};

// A value of each of a workgroup's waves to every lane: lane l has those of wave l mod (NT / 64).
template <int NT, class R>
E4B_DEV R of_waves(const R& mine) {
  constexpr int W = NT / kWave;
  __shared__ decltype(R::n) part_n[W];
  __shared__ decltype(R::s) part_s[W];
  if ((threadIdx.x & (kWave - 1)) == 0) {
    part_n[threadIdx.x / kWave] = mine.n;
    part_s[threadIdx.x / kWave] = mine.s;
  }
  __syncthreads();
  R r;
  r.n = part_n[threadIdx.x & (W - 1)];
  r.s = part_s[threadIdx.x & (W - 1)];
  return r;
}

template <int DT, int NT>
E4B_DEV PowerOf<double> row_power(const void* row, int V, int skip, float2 k, int begin = 0, int end = 0x7fffffff) {
  PowerOf<float> r;
  over_row<DT, NT, kRowUnroll, false, true>(row, V, skip, begin, end, [] {}, [&](const auto& x) { r.add(x, k); });
  PowerOf<double> all;
  all.n = r.n;
  all.s = r.s;
  all.join_lanes(kWave);
  all = of_waves<NT>(all);
  all.join_lanes(NT / kWave);
  return all;
}

// The same for any finite logits: running maximum n and sum s of exp((x - n) / tau). Differences to the maximum are taken before
// they are scaled, and the type's lowest value stays finite.
struct Run {
  float n = kLowest, s = 0.0f;
  E4B_DEV void join(float on, float os, float2 k) {
    const float to = fmaxf(n, on);
    s = s * exp_of(n - to, k) + os * exp_of(on - to, k);
    n = to;
  }
  E4B_DEV void join_lanes(int lanes, float2 k) {
    for (int off = 1; off < lanes; off *= 2) join(__shfl_xor(n, off), __shfl_xor(s, off), k);
  }
  template <int N>
  E4B_DEV void add(const float (&x)[N], float2 k) {
    float to = n, sum = 0.0f;
    for (float v : x) to = fmaxf(to, v);
    for (float v : x) sum += exp_of(v - to, k);
    s = s * exp_of(n - to, k) + sum;
    n = to;
  }
};

template <int DT, int NT, bool SKIP>
E4B_DEV Run row_run(const void* row, int V, int skip, float2 k) {
  Run r;
  over_row<DT, NT, kRowUnroll, false, SKIP>(row, V, skip, 0, 0x7fffffff, [] {}, [&](const auto& x) { r.add(x, k); });
  r.join_lanes(kWave, k);
  r = of_waves<NT>(r);
  r.join_lanes(NT / kWave, k);
  return r;
}

E4B_DEV float any_float(const void* p, int dtype, int64_t i) {
  if (dtype == E4B_FP32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return dtype == E4B_BF16 ? to_f<E4B_BF16>(v) : to_f<E4B_FP16>(v);
}

E4B_DEV float wave_max(float v) {
#pragma unroll
  for (int off = 1; off < kWave; off *= 2) v = fmaxf(v, __shfl_xor(v, off));
  return v;
}
// The row of token `at`, and whether the token counts.
struct Token {
  const char* row;
  int64_t n, t, label;
  bool counts;
  E4B_DEV Token(const e4b_logits& z, int64_t at, int bytes) {
    n = at / z.tokens;
    t = at - n * z.tokens;
    row = static_cast<const char*>(z.logits) + (n * z.seq_stride + t * z.row_stride) * bytes;
    label = z.labels ? z.labels[at] : 0;
    counts = (!z.mask || z.mask[n * z.mask_stride + t]) && label >= 0 && label < z.vocab;
  }
};

// Entry k of a token's teacher: an index inside the vocabulary and its value, or -1 and -inf.
struct Entry {
  int64_t j = -1;
  float w = -__builtin_inff();
  E4B_DEV Entry(const LossArgs& a, int64_t at, int k) {
    if (k >= a.top) return;
    j = a.index[at * a.top + k];
    const float v = any_float(a.teacher, a.teacher_dtype, at * a.top + k);
    if (j >= 0 && j < a.z.vocab) w = v;
    else j = -1;
  }
};

// The teacher's part of a row, by the first wave: probabilities over its usable entries (an index inside the
// vocabulary, a value above -inf) and tau^2 sum_k p_k (log p_k - log q_k); zero where no entry is usable. `own`: entry
// `lane`; the others are loaded in each pass.
template <int DT>
E4B_DEV float teacher_loss(const LossArgs& a, int64_t at, const typename Piece<DT>::T* row, const Entry& own, Run& r) {
  const float tau = a.z.temperature, per = 1.0f / tau;
  const int lane = threadIdx.x;
  auto entry = [&](int k) { return k == lane ? own : Entry(a, at, k); };
  float most = own.w;
  bool bad = own.w != own.w;
  for (int k = lane + kWave; k < a.top; k += kWave) {
    const float w = entry(k).w;
    most = fmaxf(most, w);
    bad |= w != w;
  }
  most = wave_max(most);
  const bool none = most == -__builtin_inff() && !__any(bad);
  float norm = 0.0f;
  if (!none)
    for (int k = lane; k < a.top; k += kWave) {
      const Entry e = entry(k);
      if (e.j >= 0) norm += expf((e.w - most) * per);
    }
  norm = wave_sum(norm);
  const float log_norm = logf(norm), log_s = logf(r.s), inv = 1.0f / norm;
  float sum = 0.0f;
  for (int k = lane; k < a.top; k += kWave) {
    const Entry e = entry(k);
    float p = 0.0f;
    if (!none && e.j >= 0) {
      const float w = (e.w - most) * per;
      p = expf(w) * inv;
      // log p - log q; an entry without probability adds nothing, whatever the student holds there
      const float lq = r.s == 0.0f ? -__builtin_inff() : (Piece<DT>::one(row[e.j]) - r.n) * per - log_s;
      if (!(p == 0.0f)) sum += p * ((w - log_norm) - lq);
    }
    a.share[at * a.top + k] = p;
  }
  if (none) r.s = 0.0f;         // nothing to differentiate
  if (norm != norm) r.s = norm;  // a teacher without a number: nor has any of the row's gradient one
  return tau * tau * wave_sum(sum);
}

// The logit that a row's exponentials refer to: the label's; the student's at the teacher's first entry.
template <int KIND>
E4B_DEV int64_t reference_of(const LossArgs& a, int64_t at, const Token& tok) {
  if (KIND != kDistill) return tok.label;
  const int64_t j = a.index[at * a.top];
  return j >= 0 && j < a.z.vocab ? j : 0;
}

// A workgroup per part of a row, where there are few rows.
template <int KIND, int DT>
__global__ __launch_bounds__(kPartThreads) void loss_parts_kernel(LossArgs a) {
  using P = Piece<DT>;
  const int64_t at = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts, step = kPartPieces<DT>;
  const Token tok(a.z, at, P::kBytes);
  if (!tok.counts) return;
  const int V = static_cast<int>(a.z.vocab), own = static_cast<int>(reference_of<KIND>(a, at, tok));
  const int begin = part * step;
  if constexpr (KIND == kStats) {
    const PowerOf<double> r = row_power<DT, kPartThreads>(tok.row, V, own, a.k, begin, begin + step);
    if (threadIdx.x == 0) static_cast<LossPart*>(a.z.workspace)[blockIdx.x] = {r.s, r.n};
  } else {
    float ref;
    const float s = row_sum<DT, kPartThreads, kRowUnroll, KIND == kScore, KIND != kDistill>(tok.row, V, own, ref, a.k, begin,
                                                                                             begin + step);
    if (threadIdx.x == 0) static_cast<float*>(a.z.workspace)[blockIdx.x] = s;
  }
}

// A label's log-probability from its logit and the running sum of the others, with the statistics (m, s) of the whole row.
E4B_DEV float join_label(float own, const Run& r, const LossArgs& a, float& m, float& s) {
  m = fmaxf(r.n, own);
  const float rest = r.s * exp_of(r.n - m, a.k);
  s = rest + exp_of(own - m, a.k);
  // the sum is 0 where every logit is -inf: each label has probability 0
  if (s == 0.0f) return -__builtin_inff();
  return (own - m) / a.z.temperature - (own == m ? log1pf(rest) : logf(s));  // the first also where it is 0, for a label of +inf
}

// A workgroup per row; SPLIT: one that joins a split row's parts, each wave for itself.
template <int KIND, int DT, int NT, int U, bool SPLIT>
__global__ __launch_bounds__(NT) void loss_rows_kernel(LossArgs a, int64_t begin) {
  using P = Piece<DT>;
  const int64_t at = begin + blockIdx.x;
  const Token tok(a.z, at, P::kBytes);
  const bool lead = threadIdx.x == 0;
  if (!tok.counts) {
    if (lead) {
      if (KIND != kScore) a.stats[at] = make_float4(0.0f, -1.0f, 0.0f, 0.0f);
      if (KIND == kLogprobs || KIND == kScore || KIND == kPolicy) a.logps[at] = 0.0f;
      if (KIND == kPolicy || KIND == kDistill) a.token_loss[at] = 0.0f;
      if (KIND == kPolicy) a.coef[at] = 0.0f;
    }
    return;
  }
  const typename P::T* row = reinterpret_cast<const typename P::T*>(tok.row);
  const int V = static_cast<int>(a.z.vocab), first = static_cast<int>(reference_of<KIND>(a, at, tok));
  // On their way while the row is read, by scalar loads: as vector loads, in front of the row's own, 230 -> 250 us (8,192 rows of
  // 128,000).
  float adv = 0.0f, old = 0.0f, ref = 0.0f;
  if constexpr (KIND == kPolicy) {
    const int64_t u = __builtin_amdgcn_readfirstlane(static_cast<int>(at));  // rows are below 2^31
    adv = a.advantages[a.adv_per_token ? u : __builtin_amdgcn_readfirstlane(static_cast<int>(tok.n))];
    old = a.old_logps[u];
    if (a.ref_logps) ref = a.ref_logps[u];
  }
  float own, sum = 0.0f;  // sum of the others' exponentials against own (a teacher: of all)
  PowerOf<double> power;
  const Entry teacher(a, at, KIND == kDistill ? static_cast<int>(threadIdx.x) : a.top);
  const int lane = threadIdx.x & (kWave - 1);
  if constexpr (KIND == kStats) {
    own = P::one(row[first]);
    if constexpr (SPLIT) {
      const LossPart* parts = static_cast<const LossPart*>(a.z.workspace) + at * a.parts;
      for (int i = lane; i < a.parts; i += kWave) power.join(parts[i].n, parts[i].s);
      power.join_lanes(kWave);
    } else {
      power = row_power<DT, NT>(row, V, first, a.k);
    }
    // nothing summed: row_run decides
    sum = power.n == kNoPower ? __builtin_nanf("")
                              : static_cast<float>(power.s) * __builtin_amdgcn_exp2f(power.n - times(own, a.k));
  } else if constexpr (SPLIT) {
    own = P::one(row[first]);
    for (int i = lane; i < a.parts; i += kWave) sum += static_cast<const float*>(a.z.workspace)[at * a.parts + i];
    sum = wave_sum(sum);
  } else {
    sum = row_sum<DT, NT, U, KIND == kScore, KIND != kDistill>(row, V, first, own, a.k);
  }
  Run r;
  r.n = own;
  r.s = sum;
  // rows of -inf, labels less likely than 1e-18: read once more, from the caches (all of 8,192 rows of 128,000: 321 -> 605 us,
  // of 64 10 -> 18, of 800 of 50,257 16 -> 31)
  const bool again = !in_room(own, a.k, sum);
  if (again) r = row_run<DT, NT, KIND != kDistill>(row, V, first, a.k);
  if (threadIdx.x >= kWave) return;
  if constexpr (KIND == kDistill) {
    const float loss = teacher_loss<DT>(a, at, row, teacher, r);
    if (lead) a.token_loss[at] = loss;
    if (lead) a.stats[at] = make_float4(r.n, r.s, 0.0f, 0.0f);
    return;
  }
  float m = own, s = 1.0f + sum, lp, low = 0.0f;
  if (again) {
    lp = join_label(own, r, a, m, s);
  } else if constexpr (KIND == kStats) {
    const double rest = power.s * exp2(power.n - own * (static_cast<double>(a.k.x) + a.k.y)), l = -log1p(rest);
    s = static_cast<float>(1.0 + rest);
    lp = static_cast<float>(l);
    low = static_cast<float>(l - lp);
  } else {
    lp = -log1pf(sum);
  }
  if (lead) {
    if (KIND != kStats) a.logps[at] = lp;
    if (KIND != kScore) a.stats[at] = make_float4(m, s, lp, low);
    if constexpr (KIND == kPolicy) {
      const float ratio = expf(lp - old);
      const float clipped = fminf(fmaxf(ratio, a.clip_lo), a.clip_hi);
      const float free_gain = ratio * adv, held = clipped * adv;
      const bool bad = free_gain != free_gain;
      float loss = bad ? free_gain : -fminf(free_gain, held);
      float slope = bad ? free_gain : free_gain <= held ? -free_gain : 0.0f;
      if (a.ref_logps) {
        const float x = ref - lp, e = expm1f(x);
        loss += a.kl_coef * (e == __builtin_inff() ? e : e - x);
        slope -= a.kl_coef * e;
      }
      a.token_loss[at] = loss;
      a.coef[at] = slope;
    }
  }
}

// ---- joins over tokens

constexpr int kJoin = 1024;

// The sums of N values over the workgroup, in the first thread.
template <int N>
E4B_DEV void block_sums(double (&v)[N]) {
  constexpr int W = kJoin / kWave;
  __shared__ double part[W][N];
#pragma unroll
  for (int off = 1; off < kWave; off *= 2) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], off);
  }
  const int lane = threadIdx.x & (kWave - 1);
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) part[threadIdx.x / kWave][i] = v[i];
  }
  __syncthreads();
  if (threadIdx.x >= kWave) return;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = part[lane & (W - 1)][i];
#pragma unroll
  for (int off = 1; off < W; off *= 2) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], off);
  }
}

// A workgroup per group; sums in 64 bits, in an order that the sizes alone decide. One workgroup for a mean over all tokens costs
// 0.7 to 0.9 ns a row: a policy forward over 8,192 / 65,536 / 262,144 / 1,048,576 rows of 1,000 bf16 logits takes 17 / 94 / 420 /
// 1,842 us with it and 11 / 57 / 237 / 916 without (a mean for each of 16 sequences: 14 / 62 / 250 / 979).
__global__ __launch_bounds__(kJoin) void loss_mean_kernel(MeanArgs a) {
  const int64_t first = blockIdx.x * a.per;
  double v[2] = {0.0, 0.0};
  for (int64_t t = threadIdx.x; t < a.per; t += kJoin)
    if (!(a.stats[first + t].y < 0.0f)) {
      v[0] += a.token_loss[first + t];
      v[1] += 1.0;
    }
  block_sums(v);
  if (threadIdx.x == 0) {
    const double sum = v[0], n = v[1];
    a.loss[blockIdx.x] = n > 0.0 ? static_cast<float>(sum / n) : 0.0f;
    a.inv[blockIdx.x] = n > 0.0 ? static_cast<float>(1.0 / n) : 0.0f;
  }
}

// A workgroup per pair. The tokens' log-probabilities and their sums are in 64 bits: the sums are long, their
// differences short.
__global__ __launch_bounds__(kJoin) void pairs_kernel(PairArgs a) {
  const int64_t half = a.seqs / 2, b = blockIdx.x;
  const bool ref_of_tokens = a.ref_kind == E4B_REF_TOKEN || a.ref_kind == E4B_REF_TOKEN_FP64;
  // in the type that they come in: of two sums of thousands the difference is left
  auto ref = [&](int64_t i) -> double {
    return a.ref_kind >= E4B_REF_SEQUENCE_FP64 ? static_cast<const double*>(a.ref)[i] : static_cast<const float*>(a.ref)[i];
  };
  double v[4] = {0.0, 0.0, 0.0, 0.0};  // sum of lp - ref over the counted tokens, their number; of both sequences
  for (int64_t i = threadIdx.x; i < 2 * a.tokens; i += kJoin) {
    const bool second = i >= a.tokens;
    const int64_t at = second ? (b + half) * a.tokens + i - a.tokens : b * a.tokens + i;
    const float4 st = a.stats[at];
    if (st.y < 0.0f) continue;
    double lp = static_cast<double>(st.z) + st.w;
    if (a.ref && ref_of_tokens) lp -= ref(at);
    v[0] += second ? 0.0 : lp;
    v[1] += second ? 0.0 : 1.0;
    v[2] += second ? lp : 0.0;
    v[3] += second ? 1.0 : 0.0;
  }
  block_sums(v);
  if (threadIdx.x != 0) return;
  const double2 c = make_double2(v[0], v[1]), r = make_double2(v[2], v[3]);
  double each[2] = {1.0, 1.0}, ratio[2] = {c.x, r.x};
  for (int i = 0; i < 2; ++i) {
    const double n = i ? r.y : c.y;
    if (a.average && n > 0.0) {
      each[i] = 1.0 / n;
      ratio[i] *= each[i];
    }
    if (a.ref && !ref_of_tokens) ratio[i] -= ref(b + i * half);
    a.rewards[b + i * half] = static_cast<float>(a.beta * ratio[i]);
  }
  const double d = ratio[0] - ratio[1], beta = a.beta, h = beta * d, eps = a.smoothing;
  double loss, slope;
  if (a.kind == E4B_PREFERENCE_SIGMOID) {
    // log(1 + e^-|h|) once: -log sigmoid(h) = log1p + max(-h, 0), -log sigmoid(-h) = log1p + max(h, 0)
    const double e = exp(-fabs(h)), soft = log1p(e), small = e / (1.0 + e), large = 1.0 / (1.0 + e);
    loss = soft + (h < 0.0 ? (1.0 - eps) * -h : eps == 0.0 ? 0.0 : eps * h);
    slope = beta * (eps * (h < 0.0 ? small : large) - (1.0 - eps) * (h < 0.0 ? large : small));
  } else if (a.kind == E4B_PREFERENCE_HINGE) {
    loss = h < 1.0 ? 1.0 - h : h != h ? h : 0.0;
    slope = h < 1.0 ? -beta : h != h ? h : 0.0;
  } else {
    const double off = d - 0.5 / beta;
    loss = off * off;
    slope = 2.0 * off;
  }
  a.loss[b] = static_cast<float>(loss);
  a.coef[b] = static_cast<float>(slope * each[0]);
  a.coef[b + half] = static_cast<float>(-slope * each[1]);
}

// ---- backward

constexpr int kBackThreads = 256;
// Pieces a thread, 1 / 2 / 4 / 8, us: 5,500 x 128,000 bf16 480 / 459 / 519 / 521, 5,500 x 50,257 196 / 180 / 195 / 222, 1,000 x
// 32,000 26.7 / 23.3 / 25.7 / 25.3, 250 x 50,257 12.1 / 11.7 / 11.1 / 14.0; fp32 5,500 x 128,000 910 / 935 / 1,055 / 1,040, 5,500 x
// 50,257 378 / 368 / 421 / 438.
constexpr int kBackUnroll = 2;

// A workgroup takes kBackThreads * kBackUnroll pieces of one row's gradient: A q_j - A p_k at the row's entries (a label:
// one entry with p = 1, A = -derivative / tau; a teacher: p_k, A = derivative * tau). Entries inside the workgroup's part are
// listed in LDS in the order of k, and each thread takes those in its pieces before it rounds: it walks the part's list, in the
// order that decides the sum. 4,096 rows by 8 / 64 / 256 / 1,024 entries: of 2,000 bf16 logits 30 / 34 / 98 / 392 us, of 32,000 93 /
// 107 / 217 / 673; of 128,000 by 64 / 1,024 356 / 1,199.
template <int DT, bool TEACHER>
__global__ __launch_bounds__(kBackThreads) void loss_backward_kernel(LossBackwardArgs a, int64_t begin, int parts) {
  using P = Piece<DT>;
  constexpr int C = P::kCount;
  const int64_t at = begin + blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const int V = static_cast<int>(a.z.vocab), tid = threadIdx.x;
  typename P::T* out = static_cast<typename P::T*>(a.grad) + at * V;
  const int64_t n = at / a.z.tokens, t = at - n * a.z.tokens;
  const float4 st = a.stats[at];
  float A = 0.0f;
  if (st.y > 0.0f || st.y != st.y) {
    A = a.grad_loss[n % a.grad_seqs * a.grad_ns + t * a.grad_ts] * a.slope;
    if (a.coef) A *= a.coef[n * a.coef_ns + t * a.coef_ts];
    if (a.inv) A *= a.inv[n * a.inv_ns];
  }
  const Split<DT> sp(out, V);
  const int first = part * kBackThreads * kBackUnroll;
  uint4* dst = reinterpret_cast<uint4*>(out + sp.head);
  if (A == 0.0f) {  // nothing to differentiate: the logits are not read
#pragma unroll
    for (int u = 0; u < kBackUnroll; ++u) {
      const int i = first + u * kBackThreads + tid;
      if (i < sp.pieces) store16_once(dst + i, make_uint4(0, 0, 0, 0));
    }
    if (part == 0) {
      if (tid < sp.head) out[tid] = P::round(0.0f);
      if (tid < V - sp.tail) out[sp.tail + tid] = P::round(0.0f);
    }
    return;
  }
  const typename P::T* row = static_cast<const typename P::T*>(a.z.logits) + n * a.z.seq_stride + t * a.z.row_stride;
  const typename P::T* body = row + sp.head;
  uint4 w[kBackUnroll];
#pragma unroll
  for (int u = 0; u < kBackUnroll; ++u) {
    const int i = first + u * kBackThreads + tid;
    if (i < sp.pieces) w[u] = load16_once(body + static_cast<int64_t>(i) * C);
  }
  // the entries of this part: positions relative to its first value, head and tail among them in part 0
  const int lo = sp.head + first * C, hi = min(sp.tail, lo + kBackThreads * kBackUnroll * C);
  auto mine = [&](int64_t j) {
    return (j >= lo && j < hi) || (part == 0 && ((j >= 0 && j < sp.head) || (j >= sp.tail && j < V)));
  };
  __shared__ int where[TEACHER ? kLossMaxTop : 1];
  __shared__ float what[TEACHER ? kLossMaxTop : 1];
  __shared__ int listed;
  int count = 0, label = -1;
  if constexpr (TEACHER) {
    if (tid < kWave) {
      int have = 0;
      for (int k0 = 0; k0 < a.top; k0 += kWave) {
        const int k = k0 + tid;
        int64_t j = -1;
        if (k < a.top) j = a.index[at * a.top + k];
        const bool keep = mine(j);
        const uint64_t held = __ballot(keep);
        if (keep) {
          const int slot = have + __popcll(held & ((uint64_t(1) << tid) - 1));
          where[slot] = static_cast<int>(j);
          what[slot] = A * a.share[at * a.top + k];
        }
        have += __popcll(held);
      }
      if (tid == 0) listed = have;
    }
    __syncthreads();
    count = __builtin_amdgcn_readfirstlane(listed);
  } else {
    const int64_t j = a.z.labels[at];
    if (mine(j)) label = static_cast<int>(j), count = 1;
  }
  auto entry = [&](int e) { return TEACHER ? where[e] : label; };
  const float rest = TEACHER ? 0.0f : A * expm1f(st.z);  // the label's A (q_l - 1)
  const float A_s = A / st.y;
  auto value = [&](float z) { return A_s * exp_of(z - st.x, a.k); };
#pragma unroll
  for (int u = 0; u < kBackUnroll; ++u) {
    const int i = first + u * kBackThreads + tid;
    if (i >= sp.pieces) continue;
    float x[C];
    P::unpack(w[u], x);
#pragma unroll
    for (int c = 0; c < C; ++c) x[c] = value(x[c]);
    const int j0 = sp.head + i * C;
    for (int e = 0; e < count; ++e) {
      const int off = entry(e) - j0;
      if (off >= 0 && off < C) {
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (c == off) x[c] = TEACHER ? x[c] - what[e] : rest;
      }
    }
    store16_once(dst + i, P::pack(x));
  }
  if (part == 0) {
    for (int side = 0; side < 2; ++side) {
      const int j = side ? sp.tail + tid : tid;
      if (side ? j >= V : j >= sp.head) continue;
      float x = value(P::one(row[j]));
      for (int e = 0; e < count; ++e)
        if (entry(e) == j) x = TEACHER ? x - what[e] : rest;
      out[j] = P::round(x);
    }
  }
}

}  // namespace e4b
