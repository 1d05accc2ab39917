// Attention of the newest tokens over the paged cache.
//   p_j = softmax_j(scale <q, k_j>),   out = sum_j p_j v_j
// One pass with the running maximum and sum.
#include "attnres_cache.h"
#include "attnres_device.h"

namespace attnres {

namespace {

constexpr int kWaves = 4;
constexpr int kPer = 4;  // values of a row a lane holds, 64 apart

// tokens that query t of sequence b sees; 0: a query that is not there or sees nothing, -1: bad counts
__device__ __forceinline__ int seen_by(const CacheAttendParams& p, int b, int t) {
  const int fresh = p.c.fresh ? p.c.fresh[b] : p.tokens;
  const int have = p.c.cached[b];
  if (have < 0 || fresh < 0 || have + (int64_t)min(fresh, p.tokens) > p.c.room) return -1;
  return t < fresh ? have + t + 1 : 0;
}

template <class DT>
__device__ __forceinline__ float score(const CacheAttendParams& p, const float (&q)[kPer], int b, int h, int j, int lane,
                                       int64_t* row) {
  using S = typename DT::S;
  const int page = cache_page(p.c, b, j);
  *row = page < 0 ? -1 : page * p.c.page_stride + h * p.c.head_stride + (j % p.c.page_size) * p.c.slot_stride;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int d = lane + i * kWave;
    if (page >= 0 && d < p.c.head_dim) s += q[i] * DT::load1((const S*)p.c.k + *row + d);
  }
  return page < 0 ? __builtin_nanf("") : wave_sum(s) * p.scale;
}

template <class DT>
__device__ __forceinline__ void load_q(const CacheAttendParams& p, int b, int hq, int t, int lane, float (&q)[kPer]) {
  using S = typename DT::S;
  const S* src = (const S*)p.q + b * p.q_b_stride + hq * p.q_h_stride + t * p.q_t_stride;
#pragma unroll
  for (int i = 0; i < kPer; ++i) q[i] = lane + i * kWave < p.c.head_dim ? DT::load1(src + lane + i * kWave) : 0.f;
}

template <class DT>
__global__ __launch_bounds__(kWaves* kWave) void attend_kernel(CacheAttendParams p) {
  using S = typename DT::S;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int hq = blockIdx.x % p.q_heads, bt = blockIdx.x / p.q_heads;
  const int t = bt % p.tokens, b = bt / p.tokens;
  const int h = hq / (p.q_heads / p.c.kv_heads), Dh = p.c.head_dim;
  const int n = seen_by(p, b, t);
  float q[kPer];
  load_q<DT>(p, b, hq, t, lane, q);
  float m = -INFINITY, l = 0.f, o[kPer] = {};
  for (int j = wave; j < n; j += kWaves) {
    int64_t row;
    const float s = score<DT>(p, q, b, h, j, lane, &row);
    const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
    const float was = __builtin_amdgcn_exp2f(m - base), e = __builtin_amdgcn_exp2f(s - base);
    l = l * was + e;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int d = lane + i * kWave;
      if (row >= 0 && d < Dh) o[i] = o[i] * was + e * DT::load1((const S*)p.c.v + row + d);
    }
    m = top;
  }
  __shared__ float sm[kWaves], sl[kWaves], so[kWaves][kPer * kWave];
  if (lane == 0) sm[wave] = m, sl[wave] = l;
#pragma unroll
  for (int i = 0; i < kPer; ++i) so[wave][lane + i * kWave] = o[i];
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, sm[w]);
  for (int w = 0; w < kWaves; ++w) sum += sm[w] == -INFINITY ? 0.f * sl[w] : __builtin_amdgcn_exp2f(sm[w] - top) * sl[w];
  S* out = (S*)p.out + ((int64_t)bt * p.q_heads + hq) * Dh;
  for (int d = threadIdx.x; d < Dh; d += kWaves * kWave) {
    float x = 0.f;
    for (int w = 0; w < kWaves; ++w) x += sm[w] == -INFINITY ? 0.f * so[w][d] : __builtin_amdgcn_exp2f(sm[w] - top) * so[w][d];
    DT::store1(out + d, n == 0 ? 0.f : n < 0 ? __builtin_nanf("") : x / sum);
  }
  if (p.lse && threadIdx.x == 0) p.lse[b * p.q_heads + hq] = top + log2f(sum);
}

template <class DT>
__global__ __launch_bounds__(kWaves* kWave) void weights_kernel(CacheAttendParams p) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int h = blockIdx.x % p.c.kv_heads, b = blockIdx.x / p.c.kv_heads;
  const int group = p.q_heads / p.c.kv_heads, n = seen_by(p, b, 0);
  for (int j = wave; j < n; j += kWaves) {
    float sum = 0.f;
    for (int g = 0; g < group; ++g) {
      float q[kPer];
      int64_t row;
      load_q<DT>(p, b, h * group + g, 0, lane, q);
      sum += __builtin_amdgcn_exp2f(score<DT>(p, q, b, h, j, lane, &row) - p.lse[b * p.q_heads + h * group + g]);
    }
    const int page = cache_page(p.c, b, j);
    if (page < 0 || lane) continue;
    float* w = p.c.w + page * p.c.w_page_stride + h * p.c.w_head_stride + j % p.c.page_size;
    *w = p.decay == 0.f ? sum : p.decay * *w + sum;
  }
}

template <class DT>
hipError_t run(const CacheAttendParams& p, hipStream_t st) {
  attend_kernel<DT><<<dim3((unsigned)(p.c.batch * p.tokens * p.q_heads)), dim3(kWaves * kWave), 0, st>>>(p);
  if (p.c.w) weights_kernel<DT><<<dim3((unsigned)(p.c.batch * p.c.kv_heads)), dim3(kWaves * kWave), 0, st>>>(p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_cache_attend(int dtype, const CacheAttendParams& p, hipStream_t st) {
  if (dtype == F32::kCode) return run<F32>(p, st);
  if (dtype == BF16::kCode) return run<BF16>(p, st);
  return run<F16>(p, st);
}

}  // namespace attnres
