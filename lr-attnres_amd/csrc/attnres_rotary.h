// Shared by the rotary kernels (attnres_qkv_rotary.hip, attnres_cache_append.hip).
#pragma once

#include "attnres_device.h"

namespace attnres {

constexpr int kRotWaves = 4;   // waves of a workgroup

template <class DT, int E>
__device__ __forceinline__ void store_raw(typename DT::S* p, const Raw<DT, E>& r) {
  constexpr int kBytes = Vec<DT, E>::kBytes;
  if constexpr (kBytes == 16) *(u32x4*)p = u32x4{r.w[0], r.w[1], r.w[2], r.w[3]};
  else if constexpr (kBytes == 8) *(u32x2*)p = u32x2{r.w[0], r.w[1]};
  else *(uint32_t*)p = r.w[0];
}

// A launch dimension holds fewer than 2^32 threads; narrow heads of many tokens are more,
// so workgroups continue in a second one.
__device__ __forceinline__ int64_t rot_wave() {
  return ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kRotWaves + threadIdx.x / kWave;
}
inline bool rot_grid(int64_t waves, dim3* grid) {
  constexpr int64_t kMax = ((int64_t)1 << 32) / (kRotWaves * kWave) - 1;
  const int64_t n = (waves + kRotWaves - 1) / kRotWaves, rows = (n + kMax - 1) / kMax;
  if (rows > 65535) return false;
  *grid = dim3((unsigned)((n + rows - 1) / rows), (unsigned)rows);
  return true;
}

}  // namespace attnres
