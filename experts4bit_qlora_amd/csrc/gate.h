// The router: top-k gate and load-balance loss over logits [T, E], forward and backward.
//
// Gate: S = the k largest logits of a row (ties to the lower index, a NaN above everything), and the
// weights w_s = softmax(z)_s over all logits, or the softmax over the chosen ones (the same as
// renormalising the first over S). Backward with g = dL/dw:
//   over all:    dz_j = p_j (g_j [j in S] - sum_S g_s p_s)
//   over chosen: dz_j = w_j (g_j - sum_S g_s w_s) on S, 0 off S.
// Balance: N valid tokens, c_e their choices of expert e, S_e their summed probabilities,
//   loss = E sum_e (c_e / N)(S_e / N),   dz_tj = E / N^2 p_tj (c_j - sum_e c_e p_te)
// (the counts are constants to the gradient). A row whose logits are all -inf has no probabilities:
// its weights and gradients are zero.
//
// GL lanes hold one row, VPL consecutive logits each, so a row is one or two 16-byte loads per lane and
// its sums and maxima are a few cross-lane steps; a row's logits are read once per pass. Bound by
// latency (launches, one memory round trip, k dependent selection steps) up to tens of thousands of
// rows, then by the logits' bytes.
#pragma once

#include "common.h"
#include "gate_launch.h"

namespace e4b {

constexpr int kGateThreads = 256;

// ---- a row over GL lanes

template <int GL>
E4B_DEV int lanes_max(int v) {
  if constexpr (GL >= 2) v = max(v, __builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, false));   // quad: lane ^ 1
  if constexpr (GL >= 4) v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, false));   // quad: lane ^ 2
  if constexpr (GL >= 8) v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false));  // mirrored eight
  if constexpr (GL >= 16) v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, false)); // mirrored row
  if constexpr (GL >= 32) v = max(v, __shfl_xor(v, 16));
  if constexpr (GL >= 64) v = max(v, __shfl_xor(v, 32));
  return v;
}

template <int CTRL>
E4B_DEV float dpp_f(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}

template <int GL>
E4B_DEV float lanes_sum(float v) {
  if constexpr (GL >= 2) v += dpp_f<0xb1>(v);
  if constexpr (GL >= 4) v += dpp_f<0x4e>(v);
  if constexpr (GL >= 8) v += dpp_f<0x141>(v);
  if constexpr (GL >= 16) v += dpp_f<0x140>(v);
  if constexpr (GL >= 32) v += __shfl_xor(v, 16);
  if constexpr (GL >= 64) v += __shfl_xor(v, 32);
  return v;
}

constexpr float kNoLogit = -__builtin_inff();

// Logits VPL gl .. + VPL - 1 of a row, as fp32; past the row's end -inf. vec: rows are whole 16-byte
// pieces at 16-byte addresses.
template <int DT, int VPL>
E4B_DEV void load_logits(const void* logits, int64_t row, int E, int gl, bool vec, float (&z)[VPL]) {
  const int first = VPL * gl;
  const int64_t at = row * E + first;
  if (vec) {
    constexpr int PER = DT == E4B_FP32 ? 4 : 8;  // values per 16 bytes
#pragma unroll
    for (int i = 0; i < VPL / PER; ++i) {
      if (first + PER * i < E) {
        if constexpr (DT == E4B_FP32) {
          const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(logits) + at + 4 * i);
          z[4 * i] = v.x; z[4 * i + 1] = v.y; z[4 * i + 2] = v.z; z[4 * i + 3] = v.w;
        } else {
          const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(logits) + at + 8 * i);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            z[8 * i + 2 * j] = lo_f<DT>(w[j]);
            z[8 * i + 2 * j + 1] = hi_f<DT>(w[j]);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) z[PER * i + j] = kNoLogit;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      z[j] = kNoLogit;
      if (first + j < E) {
        if constexpr (DT == E4B_FP32) z[j] = static_cast<const float*>(logits)[at + j];
        else z[j] = to_f<DT>(static_cast<const uint16_t*>(logits)[at + j]);
      }
    }
  }
}

template <int DT, int VPL>
E4B_DEV void store_row(void* out, int64_t row, int E, int gl, bool vec, const float (&d)[VPL]) {
  const int first = VPL * gl;
  const int64_t at = row * E + first;
  if (vec) {
    constexpr int PER = DT == E4B_FP32 ? 4 : 8;
#pragma unroll
    for (int i = 0; i < VPL / PER; ++i) {
      if (first + PER * i < E) {
        if constexpr (DT == E4B_FP32) {
          *reinterpret_cast<float4*>(static_cast<float*>(out) + at + 4 * i) =
              make_float4(d[4 * i], d[4 * i + 1], d[4 * i + 2], d[4 * i + 3]);
        } else {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = pack2(from_f<DT>(d[8 * i + 2 * j]), from_f<DT>(d[8 * i + 2 * j + 1]));
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at + 8 * i) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      if (first + j < E) {
        if constexpr (DT == E4B_FP32) static_cast<float*>(out)[at + j] = d[j];
        else static_cast<uint16_t*>(out)[at + j] = from_f<DT>(d[j]);
      }
    }
  }
}

E4B_DEV float load_dt(const void* p, int dt, int64_t i) {
  if (dt == E4B_FP32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return dt == E4B_BF16 ? to_f<E4B_BF16>(v) : to_f<E4B_FP16>(v);
}
E4B_DEV void store_dt(void* p, int dt, int64_t i, float v) {
  if (dt == E4B_FP32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = dt == E4B_BF16 ? from_f<E4B_BF16>(v) : from_f<E4B_FP16>(v);
}

// Order-preserving key of a logit: signed integers compare as the values do, -0 as 0, any NaN above
// infinity. INT_MIN is below every value's key.
E4B_DEV int logit_key(float z) {
  const int b = __builtin_bit_cast(int, z + 0.0f);
  return z != z ? 0x7fffffff : b ^ ((b >> 31) & 0x7fffffff);
}
E4B_DEV float key_logit(int k) {
  return k == 0x7fffffff ? __builtin_nanf("") : __builtin_bit_cast(float, k ^ ((k >> 31) & 0x7fffffff));
}
constexpr int kTaken = -0x7fffffff - 1;

// exp(z - m) of a row's logits and their sum over the row; zeros for a row without probabilities (m =
// -inf). A NaN or +inf makes the row NaN, as in torch's softmax.
template <int GL, int VPL>
E4B_DEV float row_exp(const float (&z)[VPL], float m, float (&e)[VPL]) {
  const float base = m == kNoLogit ? 0.0f : m;
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    e[j] = expf(z[j] - base);
    sum += e[j];
  }
  return lanes_sum<GL>(sum);
}

// The largest logit; NaN are passed over as long as a lane has another (row_exp finds them).
template <int GL, int VPL>
E4B_DEV float row_max(const float (&z)[VPL]) {
  float m = z[0];
#pragma unroll
  for (int j = 1; j < VPL; ++j) m = fmaxf(m, z[j]);
  return key_logit(lanes_max<GL>(logit_key(m)));
}
// 1 / the sum of a row's exponentials, 0 for a row without probabilities (any other row's sum is 1 at least).
E4B_DEV float row_inv(float sum) { return sum == 0.0f ? 0.0f : 1.0f / sum; }

// ---- gate

// The k largest of a row one after the other: each step takes the largest key left (a maximum over the
// lane's VPL keys and the row's GL lanes); the lowest lane that holds it, which has the lowest index,
// strikes its first occurrence out. Choice s stays with lane s % GL. Bound by the dependent steps: 1 row of 32
// experts 3.0 us, 1,531 rows of 64 (top 8, fp32) 5.1, 8,192 of 128 (top 8, bf16) 5.9.
template <int DT, int GL, int VPL>
__global__ void __launch_bounds__(kGateThreads) gate_kernel(GateArgs p, int vec) {
  const int lane = threadIdx.x & (kWave - 1);
  const int gl = lane & (GL - 1);
  const int64_t row = int64_t(blockIdx.x) * (kGateThreads / GL) + threadIdx.x / GL;
  const bool live = row < p.T;
  float z[VPL];
  load_logits<DT, VPL>(p.logits, live ? row : p.T - 1, p.E, gl, vec, z);
  int key[VPL];
#pragma unroll
  for (int j = 0; j < VPL; ++j) key[j] = VPL * gl + j < p.E ? logit_key(z[j]) : kTaken;
  const uint64_t group = (GL == 64 ? ~0ull : (1ull << (GL & 63)) - 1) << (lane & ~(GL - 1));
  int mine[VPL], at[VPL];  // keys and indices of choices s = GL i + gl (k <= E <= GL VPL)
  for (int s = 0; s < p.k; ++s) {
    int best = key[0], slot = 0;
#pragma unroll
    for (int j = 1; j < VPL; ++j) {
      const bool up = key[j] > best;
      best = up ? key[j] : best;
      slot = up ? j : slot;
    }
    const int top = lanes_max<GL>(best);
    const int owner = __builtin_ctzll(__ballot(best == top) & group);
    const int index = VPL * (owner & (GL - 1)) + __shfl(slot, owner);
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      key[j] = index == VPL * gl + j ? kTaken : key[j];
      const bool here = s == GL * j + gl;
      mine[j] = here ? top : mine[j];
      at[j] = here ? index : at[j];
    }
  }
  const float m = key_logit(__shfl(mine[0], lane & ~(GL - 1)));
  float w[VPL], sum = 0.0f;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    w[j] = GL * j + gl < p.k && m != kNoLogit ? expf(key_logit(mine[j]) - m) : 0.0f;
    sum += w[j];
  }
  if (p.over_chosen) {
    sum = lanes_sum<GL>(sum);
  } else {
    float e[VPL];
    sum = row_exp<GL, VPL>(z, m, e);
  }
  if (m == kNoLogit) sum = 1.0f;
  if (!live) return;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int s = GL * j + gl;
    if (s < p.k) {
      p.index[row * p.k + s] = at[j];
      store_dt(p.weights, p.wdtype, row * p.k + s, w[j] / sum);
    }
  }
}

// (8,192 rows of 128 experts, top 8, bf16: 5.4 us.)
template <int DT, int GL, int VPL>
__global__ void __launch_bounds__(kGateThreads) gate_backward_kernel(GateArgs p, int vec) {
  const int gl = threadIdx.x & (GL - 1);
  const int64_t row = int64_t(blockIdx.x) * (kGateThreads / GL) + threadIdx.x / GL;
  const bool live = row < p.T;
  const int64_t r = live ? row : p.T - 1;
  float z[VPL], e[VPL], g[VPL];
  load_logits<DT, VPL>(p.logits, r, p.E, gl, vec, z);
  uint32_t chosen = 0;
#pragma unroll
  for (int j = 0; j < VPL; ++j) g[j] = 0.0f;
  for (int s = 0; s < p.k; ++s) {
    const int i = static_cast<int>(p.index[r * p.k + s]) - VPL * gl;
    const float gs = load_dt(p.weights, p.wdtype, r * p.k + s);
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      g[j] = i == j ? gs : g[j];
      chosen |= i == j ? 1u << j : 0u;
    }
  }
  const float m = row_max<GL, VPL>(z);
  float sum = row_exp<GL, VPL>(z, m, e);
  if (p.over_chosen) {
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      e[j] = (chosen >> j) & 1 ? e[j] : 0.0f;
      sum += e[j];
    }
    sum = lanes_sum<GL>(sum);
  }
  const float inv = row_inv(sum);
  float mean = 0.0f;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    e[j] *= inv;
    mean += (chosen >> j) & 1 ? g[j] * e[j] : 0.0f;
  }
  mean = lanes_sum<GL>(mean);
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const bool zero = p.over_chosen && !((chosen >> j) & 1);
    e[j] = zero ? 0.0f : e[j] * (g[j] - mean);
  }
  if (live) store_row<DT, VPL>(p.grad, row, p.E, gl, vec, e);
}

// ---- balance loss

// One chunk of a layer's tokens: the summed probabilities of its valid tokens and the counts of their
// choices. A lane keeps its VPL experts' sums over the rows its group takes; the groups' sums join in
// LDS in order, so the result does not depend on scheduling (the counts are integer sums). 16 layers of
// 8,192 rows, 64 experts, top 8, bf16 (25 MB): 11.0 us (8.9 with the hardware's short exponential, which is a few
// units less exact).
template <int DT, int GL, int VPL>
__global__ void __launch_bounds__(kGateThreads) balance_kernel(BalanceArgs p, int vec, int64_t chunk_rows) {
  constexpr int NG = kGateThreads / GL;  // rows at a time
  extern __shared__ float sums[];        // [NG, GL * VPL]
  __shared__ int cnt[kGateMaxExperts + 1];
  const int tid = threadIdx.x;
  const int gl = tid & (GL - 1), slot = tid / GL;
  const int layer = blockIdx.y;
  for (int i = tid; i <= p.E; i += kGateThreads) cnt[i] = 0;
  __syncthreads();
  const int64_t t0 = blockIdx.x * chunk_rows, t1 = min(t0 + chunk_rows, p.T);
  float acc[VPL];
#pragma unroll
  for (int j = 0; j < VPL; ++j) acc[j] = 0.0f;
  for (int64_t t = t0 + slot; t < t1; t += NG) {
    const int64_t row = layer * p.T + t;
    float z[VPL], e[VPL];
    load_logits<DT, VPL>(p.logits, row, p.E, gl, vec, z);
    const bool valid = !p.mask || p.mask[layer * p.mask_stride + t];
    for (int s = gl; s < p.k; s += GL) {
      const int64_t i = p.index[row * p.k + s];
      if (valid && i >= 0 && i < p.E) atomicAdd(&cnt[i], 1);
    }
    if (valid && gl == 0) atomicAdd(&cnt[p.E], 1);
    const float m = row_max<GL, VPL>(z);
    const float sum = row_exp<GL, VPL>(z, m, e);
    const float inv = row_inv(sum);
#pragma unroll
    for (int j = 0; j < VPL; ++j) acc[j] = valid ? acc[j] + e[j] * inv : acc[j];
  }
#pragma unroll
  for (int j = 0; j < VPL; ++j) sums[slot * (GL * VPL) + VPL * gl + j] = acc[j];
  __syncthreads();
  const int64_t part = int64_t(layer) * p.chunks + blockIdx.x;
  for (int i = tid; i <= p.E; i += kGateThreads) {
    p.part_counts[part * (p.E + 1) + i] = cnt[i];
    if (i == p.E) continue;
    float s = 0.0f;
    for (int g = 0; g < NG; ++g) s += sums[g * (GL * VPL) + i];
    p.part[part * p.E + i] = s;
  }
}

// A layer's chunks joined, in a fixed order and 64 bits: counts, valid tokens, loss. Bound by the latency of
// its loads: `lanes` threads (a power of two from 32, the layer's experts or 1,024 of them) per part of the chunks, every
// 1024 / lanes'th, so that a thread's serial loads are few (64 chunks of 64 experts in 16 layers: 4.7 us; one
// thread per expert over all chunks 34).
constexpr int kJoinThreads = 1024;
E4B_DEV double wave_sum(double v) {
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__global__ void __launch_bounds__(kJoinThreads) balance_join_kernel(BalanceArgs p, int lanes) {
  __shared__ double part[kJoinThreads];
  __shared__ int count[kJoinThreads];
  const int tid = threadIdx.x, layer = blockIdx.x;
  const int e = tid & (lanes - 1), from = tid / lanes, step = kJoinThreads / lanes;
  const float* sums = p.part + int64_t(layer) * p.chunks * p.E + e;
  const int32_t* counts = p.part_counts + int64_t(layer) * p.chunks * (p.E + 1);
  double s = 0.0;
  int n = 0, valid = 0;  // at most T * k of them: 32 bits
  if (e < p.E) {
#pragma unroll 8
    for (int c = from; c < p.chunks; c += step) {
      s += sums[int64_t(c) * p.E];
      n += counts[int64_t(c) * (p.E + 1) + e];
    }
  }
  for (int c = tid; c < p.chunks; c += kJoinThreads) valid += counts[int64_t(c) * (p.E + 1) + p.E];
  part[tid] = s;
  count[tid] = n;
  __syncthreads();
  double mine = 0.0;
  if (tid < p.E) {  // (lanes >= E: its parts are tid + lanes * i)
    for (int i = 1; i < step; ++i) {
      s += part[tid + lanes * i];
      n += count[tid + lanes * i];
    }
    p.counts[int64_t(layer) * p.E + tid] = n;
    if (p.kept) p.kept[int64_t(layer) * p.E + tid] = n;
    mine = static_cast<double>(n) * s;
  }
  __syncthreads();
  mine = wave_sum(mine);
  const double all = wave_sum(static_cast<double>(valid));  // exact: at most 2^31
  double* const valids = part + kJoinThreads / kWave;
  if (tid % kWave == 0) {
    part[tid / kWave] = mine;
    valids[tid / kWave] = all;
  }
  __syncthreads();
  if (tid == 0) {
    double terms = 0.0, tokens = 0.0;
    for (int i = 0; i < kJoinThreads / kWave; ++i) {
      terms += part[i];
      tokens += valids[i];
    }
    p.valid[layer] = static_cast<int64_t>(tokens);
    p.loss[layer] = tokens > 0.0 ? static_cast<float>(terms * p.E / (tokens * tokens)) : 0.0f;
  }
}

// dL/dz[t, e] = f P[t, e] (c[e] - sum_i c[i] P[t, i]), f = dL/dloss E / N^2. A workgroup takes every gridDim.x'th
// group of rows, so that a lane reads its experts' counts once. 16 layers of 8,192 rows, 64 experts, bf16 (34
// MB): 13.9 us, about half of it the exponentials and the rest the bytes.
template <int DT, int GL, int VPL>
__global__ void __launch_bounds__(kGateThreads) balance_backward_kernel(BalanceArgs p, int vec) {
  constexpr int NG = kGateThreads / GL;
  const int gl = threadIdx.x & (GL - 1);
  const int layer = blockIdx.y;
  float c[VPL];  // (counts of at most T * k choices: 32 bits)
#pragma unroll
  for (int j = 0; j < VPL; ++j)
    c[j] = VPL * gl + j < p.E ? static_cast<float>(static_cast<int>(p.counts[int64_t(layer) * p.E + VPL * gl + j])) : 0.0f;
  // the factor in two divisions: N^2 passes fp32's 24 bits long before N does (N = 0: no row is valid)
  const float n = static_cast<float>(p.valid[layer]);
  const float f = p.grad_loss[layer] * (static_cast<float>(p.E) / n) / n;
  for (int64_t t = int64_t(blockIdx.x) * NG + threadIdx.x / GL; t < p.T; t += int64_t(gridDim.x) * NG) {
    const int64_t row = layer * p.T + t;
    float z[VPL], e[VPL];
    load_logits<DT, VPL>(p.logits, row, p.E, gl, vec, z);
    const bool valid = !p.mask || p.mask[layer * p.mask_stride + t];
    const float m = row_max<GL, VPL>(z);
    const float inv = row_inv(row_exp<GL, VPL>(z, m, e));
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      e[j] *= inv;
      dot += VPL * gl + j < p.E ? c[j] * e[j] : 0.0f;
    }
    dot = lanes_sum<GL>(dot);
#pragma unroll
    for (int j = 0; j < VPL; ++j) e[j] = valid ? f * e[j] * (c[j] - dot) : 0.0f;
    store_row<DT, VPL>(p.grad, row, p.E, gl, vec, e);
  }
}

}  // namespace e4b
