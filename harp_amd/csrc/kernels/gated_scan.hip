// The gated linear recurrence h_t = a_t h_(t-1) + x_t over [batch, time, width], and its gradients.
#include "elements.hpp"

namespace eh {
namespace {

template <int DT> __device__ inline float at(const Sequences& s, int64_t b, int64_t t, int d) {
  return Elem<DT>::get(static_cast<const typename Elem<DT>::T*>(s.p)[b * s.batch + t * s.step + d]);
}
template <int DT> __device__ inline void put(const Sequences& s, int64_t b, int64_t t, int d, float v) {
  static_cast<typename Elem<DT>::T*>(s.p)[b * s.batch + t * s.step + d] = Elem<DT>::put(v);
}

// A thread for each channel of each sequence, step by step.
template <int DT> __global__ __launch_bounds__(64) void scan_steps(ScanArgs a) {
  const int blocks = (a.width + 63) / 64;
  const int64_t b = blockIdx.x / blocks;
  const int d = static_cast<int>(blockIdx.x % blocks) * 64 + static_cast<int>(threadIdx.x);
  if (d >= a.width) return;
  int64_t n = a.time;
  if (a.lengths) n = min(n, max(static_cast<int64_t>(a.lengths[b]), int64_t{0}));
  float h = a.state ? a.state[b * a.width + d] : 0.f;
  for (int64_t t = 0; t < n; ++t) {
    float g = at<DT>(a.gate, b, t, d);
    if (a.log_gate) g = exp2_hw(g * kLog2e);
    h = __builtin_fmaf(g, h, at<DT>(a.x, b, t, d));
    put<DT>(a.out, b, t, d, h);
  }
  if (a.final_state) a.final_state[b * a.width + d] = h;
}

// lambda_t = g_t + a_(t+1) lambda_(t+1);  dx_t = lambda_t, da_t = lambda_t h_(t-1), d(log a_t) = da_t a_t.
template <int DT> __global__ __launch_bounds__(64) void scan_grad_steps(ScanArgs a) {
  const int blocks = (a.width + 63) / 64;
  const int64_t b = blockIdx.x / blocks;
  const int d = static_cast<int>(blockIdx.x % blocks) * 64 + static_cast<int>(threadIdx.x);
  if (d >= a.width) return;
  int64_t n = a.time;
  if (a.lengths) n = min(n, max(static_cast<int64_t>(a.lengths[b]), int64_t{0}));
  float carry = a.grad_final ? a.grad_final[b * a.width + d] : 0.f;        // a_(t+1) lambda_(t+1)
  for (int64_t t = n; t-- > 0;) {
    float g = at<DT>(a.gate, b, t, d);
    if (a.log_gate) g = exp2_hw(g * kLog2e);
    const float l = at<DT>(a.out, b, t, d) + carry;
    const float before = t ? at<DT>(a.x, b, t - 1, d) : a.state ? a.state[b * a.width + d] : 0.f;
    put<DT>(a.grad_x, b, t, d, l);
    put<DT>(a.grad_gate, b, t, d, a.log_gate ? l * before * g : l * before);
    carry = g * l;
  }
  if (a.final_state) a.final_state[b * a.width + d] = carry;
}

template <class F> hipError_t by_type(int dtype, F&& f) {
  switch (dtype) {
    case kF32: return f(std::integral_constant<int, kF32>{});
    case kBF16: return f(std::integral_constant<int, kBF16>{});
    default: return f(std::integral_constant<int, kF16>{});
  }
}

}  // namespace

size_t scan_workspace(const ScanArgs&, int) { return 0; }

hipError_t launch_scan(const ScanArgs& a, int, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.batch * ((a.width + 63) / 64)));
  return by_type(a.dtype, [&](auto dt) {
    scan_steps<dt.value><<<grid, 64, 0, stream>>>(a);
    return hipGetLastError();
  });
}

hipError_t launch_scan_grad(const ScanArgs& a, int, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.batch * ((a.width + 63) / 64)));
  return by_type(a.dtype, [&](auto dt) {
    scan_grad_steps<dt.value><<<grid, 64, 0, stream>>>(a);
    return hipGetLastError();
  });
}

}  // namespace eh
