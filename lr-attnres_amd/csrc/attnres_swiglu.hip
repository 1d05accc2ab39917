// Gated feed-forward projections: dispatch of the products by type, and the passes
// around them -- the activation's gradient, copies of operands that the products
// cannot address as they are.
#include "attnres_swiglu.h"

namespace attnres {

hipError_t launch_swiglu_gemm_bf16(int form, int tile, const SwGemmParams& p, hipStream_t st);
hipError_t launch_swiglu_gemm_f16(int form, int tile, const SwGemmParams& p, hipStream_t st);
hipError_t launch_swiglu_gemm_f32(int form, int tile, const SwGemmParams& p, hipStream_t st);

hipError_t launch_swiglu_gemm(int dtype, int form, int tile, const SwGemmParams& p, hipStream_t st) {
  if (dtype == BF16::kCode) return launch_swiglu_gemm_bf16(form, tile, p, st);
  if (dtype == F16::kCode) return launch_swiglu_gemm_f16(form, tile, p, st);
  return launch_swiglu_gemm_f32(form, tile, p, st);
}

namespace {

constexpr int kThreads = 256;

// du = dh silu(z), dz = dh u silu'(z), silu'(z) = s + z s (1 - s), s = 1 / (1 + exp(-z)).
// Both products of the backward read [du dz], each of them several times; it is
// rounded to the dtype as they take it.  Bound by memory (10 bytes a hidden value
// in 16 bits).
template <class DT>
__global__ __launch_bounds__(kThreads) void swiglu_grad_kernel(SwGradParams p) {
  using S = typename DT::S;
  constexpr int V = 16 / (int)sizeof(S);
  const int64_t chunks = p.Fp / V;
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (at >= p.n * chunks) return;
  const int64_t t = at / chunks;
  const int f = (int)(at - t * chunks) * V;
  S* du = (S*)p.d + t * 2 * p.Fp + f;
  float g[V], u[V], z[V], a[V], b[V];
  const S* dh = (const S*)p.dh + t * p.dh_stride + f;
  if (f < p.F) {
    if (p.vec && f + V <= p.F) {
      load_vec<DT, V, true>(dh, g);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) g[e] = f + e < p.F ? DT::load1(dh + e) : 0.f;
    }
    load_vec<DT, V, true>((const S*)p.saved + t * p.Fp + f, u);
    load_vec<DT, V, true>((const S*)p.saved + (p.n + t) * p.Fp + f, z);
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float s;
    if constexpr (DT::kCode == 0) s = 1.f / (1.f + expf(-z[e]));
    else s = __builtin_amdgcn_rcpf(1.f + __expf(-z[e]));
    const float act = z[e] * s;
    a[e] = f + e < p.F ? g[e] * act : 0.f;
    b[e] = f + e < p.F ? g[e] * u[e] * (s + act * (1.f - s)) : 0.f;
  }
  store_vec<DT, V>(du, a);
  store_vec<DT, V>(du + p.Fp, b);
}

// Small against the products that follow (a value copied once, multiplied by a
// whole row); single values, since a row may start anywhere.
template <class DT>
__global__ __launch_bounds__(kThreads) void swiglu_pack_kernel(SwPackParams p) {
  using S = typename DT::S;
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t r = at / p.to_stride;
  const int c = (int)(at - r * p.to_stride);
  if (r >= p.rows) return;
  ((S*)p.to)[at] = c < p.cols ? ((const S*)p.from)[r * p.from_stride + c] : (S)0;
}

template <class DT>
__global__ __launch_bounds__(kThreads) void swiglu_clear_kernel(typename DT::S* to, int64_t n) {
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (at < n) to[at] = (typename DT::S)0;
}

bool grid_of(int64_t n, dim3* grid) {
  const int64_t g = (n + kThreads - 1) / kThreads;
  if (g > INT32_MAX) return false;
  *grid = dim3((unsigned)g);
  return true;
}

template <class DT>
hipError_t run_grad(const SwGradParams& p, hipStream_t st) {
  dim3 grid;
  if (!grid_of(p.n * (p.Fp / (16 / (int)sizeof(typename DT::S))), &grid)) return hipErrorInvalidValue;
  swiglu_grad_kernel<DT><<<grid, dim3(kThreads), 0, st>>>(p);
  return hipGetLastError();
}
template <class DT>
hipError_t run_pack(const SwPackParams& p, hipStream_t st) {
  dim3 grid;
  if (!grid_of(p.rows * p.to_stride, &grid)) return hipErrorInvalidValue;
  swiglu_pack_kernel<DT><<<grid, dim3(kThreads), 0, st>>>(p);
  return hipGetLastError();
}
template <class DT>
hipError_t run_clear(void* to, int64_t n, hipStream_t st) {
  dim3 grid;
  if (!grid_of(n, &grid)) return hipErrorInvalidValue;
  swiglu_clear_kernel<DT><<<grid, dim3(kThreads), 0, st>>>((typename DT::S*)to, n);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_swiglu_grad(int dtype, const SwGradParams& p, hipStream_t st) {
  if (dtype == F32::kCode) return run_grad<F32>(p, st);
  return dtype == BF16::kCode ? run_grad<BF16>(p, st) : run_grad<F16>(p, st);
}
hipError_t launch_swiglu_pack(int dtype, const SwPackParams& p, hipStream_t st) {
  return dtype == F32::kCode ? run_pack<F32>(p, st) : run_pack<BF16>(p, st);  // (bits only)
}
hipError_t launch_swiglu_clear(int dtype, void* to, int64_t values, hipStream_t st) {
  return dtype == F32::kCode ? run_clear<F32>(to, values, st) : run_clear<BF16>(to, values, st);
}

}  // namespace attnres
