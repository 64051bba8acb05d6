// Launchers of the router kernels: lanes per row by the number of experts.
#include "gate.h"

#include <algorithm>

namespace e4b {

namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Lanes per row: eight logits each, a power of two (sixteen logits above 512 experts).
int lanes_of(int E) {
  int gl = 1;
  while (gl < 64 && 8 * gl < E) gl *= 2;
  return gl;
}

int dtype_bytes(int dtype) { return dtype == E4B_FP32 ? 4 : 2; }

int vec_rows(const void* p, int dtype, int E) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (int64_t(E) * dtype_bytes(dtype)) % 16 == 0;
}

// f(dtype, lanes, logits per lane) with all three known at compile time
template <int DT, class F>
void by_lanes(int E, F&& f) {
  using std::integral_constant;
  integral_constant<int, DT> d;
  integral_constant<int, 8> v8;
  if (E > 512) return f(d, integral_constant<int, 64>{}, integral_constant<int, 16>{});
  switch (lanes_of(E)) {
    case 1: return f(d, integral_constant<int, 1>{}, v8);
    case 2: return f(d, integral_constant<int, 2>{}, v8);
    case 4: return f(d, integral_constant<int, 4>{}, v8);
    case 8: return f(d, integral_constant<int, 8>{}, v8);
    case 16: return f(d, integral_constant<int, 16>{}, v8);
    case 32: return f(d, integral_constant<int, 32>{}, v8);
    default: return f(d, integral_constant<int, 64>{}, v8);
  }
}
template <class F>
void by_shape(int dtype, int E, F&& f) {
  switch (dtype) {
    case E4B_FP32: return by_lanes<E4B_FP32>(E, f);
    case E4B_BF16: return by_lanes<E4B_BF16>(E, f);
    default: return by_lanes<E4B_FP16>(E, f);
  }
}

// f(arguments of the rows, grid) for all rows in order, `per` a workgroup. A launch holds fewer than 2^32 work items
// (2^26 rows of more than 256 experts are as many), so it takes 2^23 workgroups at most.
template <class F>
void by_rows(const GateArgs& a, int per, F&& f) {
  const int64_t most = (int64_t(1) << 23) * per;
  for (int64_t first = 0; first < a.T; first += most) {
    GateArgs p = a;
    p.T = std::min(most, a.T - first);
    p.logits = static_cast<const char*>(a.logits) + first * a.E * dtype_bytes(a.dtype);
    p.index = a.index + first * a.k;
    p.weights = static_cast<char*>(a.weights) + first * a.k * dtype_bytes(a.wdtype);
    if (a.grad) p.grad = static_cast<char*>(a.grad) + first * a.E * dtype_bytes(a.dtype);
    f(p, dim3(static_cast<unsigned>(cdiv(p.T, per))));
  }
}

}  // namespace

void launch_gate(const GateArgs& a, hipStream_t s) {
  by_shape(a.dtype, a.E, [&](auto dt, auto gl, auto vpl) {
    by_rows(a, kGateThreads / gl(), [&](const GateArgs& p, dim3 grid) {
      hipLaunchKernelGGL((gate_kernel<dt(), gl(), vpl()>), grid, dim3(kGateThreads), 0, s, p,
                         vec_rows(p.logits, p.dtype, p.E));
    });
  });
}

void launch_gate_backward(const GateArgs& a, hipStream_t s) {
  by_shape(a.dtype, a.E, [&](auto dt, auto gl, auto vpl) {
    by_rows(a, kGateThreads / gl(), [&](const GateArgs& p, dim3 grid) {
      hipLaunchKernelGGL((gate_backward_kernel<dt(), gl(), vpl()>), grid, dim3(kGateThreads), 0, s, p,
                         vec_rows(p.logits, p.dtype, p.E) && vec_rows(p.grad, p.dtype, p.E));
    });
  });
}

// About two rows per row slot of a workgroup, up to 1,024 workgroups over all layers.
int balance_chunks(int64_t T, int L, int E) {
  const int slots = kGateThreads / lanes_of(E);
  const int64_t most = std::max<int64_t>(1, 1024 / L);
  return static_cast<int>(std::max<int64_t>(1, std::min(most, cdiv(T, 2 * slots))));
}

void launch_balance(const BalanceArgs& a, hipStream_t s) {
  if (a.chunks) by_shape(a.dtype, a.E, [&](auto dt, auto gl, auto vpl) {
    const dim3 grid(static_cast<unsigned>(a.chunks), static_cast<unsigned>(a.L));
    hipLaunchKernelGGL((balance_kernel<dt(), gl(), vpl()>), grid, dim3(kGateThreads),
                       sizeof(float) * kGateThreads * vpl(), s, a, vec_rows(a.logits, a.dtype, a.E),
                       cdiv(a.T, a.chunks));
  });
  int lanes = 32;
  while (lanes < a.E) lanes *= 2;
  hipLaunchKernelGGL(balance_join_kernel, dim3(static_cast<unsigned>(a.L)), dim3(kJoinThreads), 0, s, a, lanes);
}

constexpr int kBackwardGroups = 1024;  // over all layers (16 of 8,192 rows, 64 experts: 13.9 us; one row a lane group 16.8)
void launch_balance_backward(const BalanceArgs& a, hipStream_t s) {
  by_shape(a.dtype, a.E, [&](auto dt, auto gl, auto vpl) {
    const int64_t groups = cdiv(a.T, kGateThreads / gl()), most = std::max(1, kBackwardGroups / a.L);
    const dim3 grid(static_cast<unsigned>(std::min(groups, most)), static_cast<unsigned>(a.L));
    hipLaunchKernelGGL((balance_backward_kernel<dt(), gl(), vpl()>), grid, dim3(kGateThreads), 0, s, a,
                       vec_rows(a.logits, a.dtype, a.E) && vec_rows(a.grad, a.dtype, a.E));
  });
}

}  // namespace e4b
