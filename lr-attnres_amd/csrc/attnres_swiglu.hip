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
constexpr int64_t kMaxGrid = (1 << 24) - 1;  // fewer than 2^32 threads

// du = dh silu(z), dz = dh u silu'(z), silu'(z) = s + z s (1 - s), s = 1 / (1 + exp(-z)).
// Both products of the backward read [du dz], each of them several times; it is
// rounded to the dtype as they take it: in 16 bits dx and dweight are 1.4 times as far from the
// 64-bit result (0.00235 of it by norm in bf16) as their own rounding (0.00166), and a chain that
// rounds u, z, their activation and product too is at 0.0034.  Bound by memory: 11 bytes a hidden value in
// bf16 (2 of dh, 5 of u and z, 4 of du and dz), 12 in fp16; 16384 tokens of hidden 4096, bf16, 738 MB:
// 124-128 us, 5.8-6 TB/s.  A workgroup takes 16 tokens of four neighbouring blocks, so that every
// array is read and written in whole lines.
template <class DT>
__global__ __launch_bounds__(kThreads) void swiglu_grad_kernel(SwGradParams p) {
  using S = typename DT::S;
  constexpr int V = 16 / (int)sizeof(S), kStep = SwElem<DT>::kStep, L = SwPlanes<DT>::kLow;
  const int blocks = p.Fp / kStep, across = (blocks + 3) / 4;
  const int64_t group = (int64_t)blockIdx.x / across;
  const int b = (int)(blockIdx.x - group * across) * 4 + threadIdx.x / 64;
  const int64_t t = group * 16 + threadIdx.x % 64 / 4;
  const int c = threadIdx.x % 4;
  if (b >= blocks || t >= p.n) return;
  const int f = b * kStep + c * V;
  const int64_t at = ((int64_t)b * p.n + t) * kStep + c * V;
  const SwPlaneAddress from = sw_planes<DT>(p.saved, p.n, p.Fp);
  const S* dh = (const S*)p.dh + t * p.dh_stride + f;
  float g[V], u[V], z[V], a[V], d[V];
  if (f < p.F && p.vec && f + V <= p.F) {
    load_vec<DT, V, true>(dh, g);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) g[e] = f + e < p.F ? DT::load1(dh + e) : 0.f;
  }
  if constexpr (L == 0) {
    load_vec<DT, V, true>((const S*)from.u + at, u);
    load_vec<DT, V, true>((const S*)from.z + at, z);
  } else {
    const u32x4 uh = __builtin_nontemporal_load((const u32x4*)((const S*)from.u + at));
    const u32x4 zh = __builtin_nontemporal_load((const u32x4*)((const S*)from.z + at));
    uint32_t low[V];  // u's low bits at L, z's above them
    if constexpr (L == 4) {
      const u32x2 w = __builtin_nontemporal_load((const u32x2*)(from.low + at));
#pragma unroll
      for (int e = 0; e < V; ++e) low[e] = w[e / 4] >> (8 * (e % 4));
    } else {
      const u32x4 w = __builtin_nontemporal_load((const u32x4*)(from.low + at * 2));
#pragma unroll
      for (int e = 0; e < V; ++e) low[e] = w[e / 2] >> (16 * (e % 2));
    }
    constexpr uint32_t kMask = (1u << L) - 1;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const uint32_t uw = e % 2 ? uh[e / 2] & 0xffff0000u : uh[e / 2] << 16;
      const uint32_t zw = e % 2 ? zh[e / 2] & 0xffff0000u : zh[e / 2] << 16;
      u[e] = __uint_as_float(uw | (low[e] & kMask) << (16 - L));
      z[e] = __uint_as_float(zw | (low[e] >> L & kMask) << (16 - L));
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float s;
    if constexpr (DT::kCode == 0) s = 1.f / (1.f + expf(-z[e]));
    else s = __builtin_amdgcn_rcpf(1.f + __expf(-z[e]));
    const float act = z[e] * s;
    a[e] = f + e < p.F ? g[e] * act : 0.f;
    d[e] = f + e < p.F ? g[e] * u[e] * (s + act * (1.f - s)) : 0.f;
  }
  store_vec<DT, V>((S*)p.d + at, a);
  store_vec<DT, V>((S*)p.d + (int64_t)p.Fp * p.n + at, d);
}

// Small against the products that follow (a value copied once, multiplied by a whole
// row).  A thread writes a chunk of 16 bytes; it reads single values, since a row may
// start anywhere.
template <class DT>
__global__ __launch_bounds__(kThreads) void swiglu_pack_kernel(SwPackParams p, int64_t first) {
  using S = typename DT::S;
  constexpr int V = 16 / (int)sizeof(S);
  int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;  // chunk
  const bool second = at >= first;
  const SwPack& k = p.part[second];
  if (second) at -= first;
  const int chunks = p.to_stride / V;
  const int64_t r = at / chunks;
  const int c = (int)(at - r * chunks) * V;
  if (r >= k.to_rows * k.blocks || (second && p.parts < 2)) return;
  const int64_t block = r / k.to_rows, row = r - block * k.to_rows;
  const S* from = (const S*)k.from + (block * k.rows + row) * k.from_stride + c;
  u32x4 v = {0, 0, 0, 0};
  if (row < k.rows) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (c + e >= p.cols) break;
      if constexpr (V == 8) v[e / 2] |= (uint32_t)from[e] << (16 * (e & 1));
      else v[e] = __float_as_uint(from[e]);
    }
  }
  *(u32x4*)((S*)k.to + r * p.to_stride + c) = v;
}

template <class DT>
__global__ __launch_bounds__(kThreads) void swiglu_clear_kernel(typename DT::S* to, int64_t n) {
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (at < n) to[at] = (typename DT::S)0;
}

bool grid_of(int64_t n, dim3* grid) {
  const int64_t g = (n + kThreads - 1) / kThreads;
  if (g > kMaxGrid) return false;
  *grid = dim3((unsigned)g);
  return true;
}

template <class DT>
hipError_t run_grad(const SwGradParams& p, hipStream_t st) {
  const int64_t grid = (p.n + 15) / 16 * ((p.Fp / SwElem<DT>::kStep + 3) / 4);
  if (grid > kMaxGrid) return hipErrorInvalidValue;
  swiglu_grad_kernel<DT><<<dim3((unsigned)grid), dim3(kThreads), 0, st>>>(p);
  return hipGetLastError();
}
template <class DT>
hipError_t run_pack(const SwPackParams& p, hipStream_t st) {
  int64_t n[2] = {0, 0};
  for (int i = 0; i < p.parts; ++i) n[i] = p.part[i].to_rows * p.part[i].blocks * (p.to_stride / (16 / (int)sizeof(typename DT::S)));
  dim3 grid;
  if (!grid_of(n[0] + n[1], &grid)) return hipErrorInvalidValue;
  swiglu_pack_kernel<DT><<<grid, dim3(kThreads), 0, st>>>(p, n[0]);
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
