// What each cached token received of a step's attention: with the scores x as the
// attention left them (base-2 logarithms) and each row's logarithm of the sum,
//   w_j <- decay w_j + sum over the head's queries of 2^(x_j - lse).
// Bound by memory: the scores of a group's heads read, the weights read and written, 4
// bytes each.  Tokens are dealt to workgroups as attention's units are.
#include "attnres_cache_attend.h"

namespace attnres {

namespace {

__global__ __launch_bounds__(kAttUnit) void cache_weights_kernel(CacheAttendParams p, int wgs) {
  const int segs = p.c.kv_heads;
  const Deal d = deal(p, segs, wgs);
  int x = deal_start(d, blockIdx.x);
  const int x1 = deal_start(d, blockIdx.x + 1);
  int b = 0, b_start = 0, b_end = 0, units = 1, n = 0;
  for (; x < x1; ++x) {
    if (x >= b_end) {
      find_unit(p, segs, x, &b, &b_start, &units);
      b_end = b_start + segs * units;
      n = seq_len(p, b);
    }
    const int h = (x - b_start) / units, j = (x - b_start - h * units) * kAttUnit + threadIdx.x;
    if (j >= n) continue;
    const int page = cache_page(p.c, b, j);
    if (page < 0) continue;
    float* w = p.c.w + page * p.c.w_page_stride + h * p.c.w_head_stride + j % p.c.page_size;
    const int64_t hq = (int64_t)b * p.q_heads + h * p.group;
    float sum = 0.f;
    for (int g = 0; g < p.group; ++g) sum += __builtin_amdgcn_exp2f(p.logits[(hq + g) * p.logit_stride + j] - p.lse[hq + g]);
    *w = p.decay == 0.f ? sum : p.decay * *w + sum;
  }
}

}  // namespace

hipError_t launch_cache_weights(const CacheAttendParams& p, hipStream_t st) {
  const int wgs = 2048;
  cache_weights_kernel<<<dim3(wgs), dim3(kAttUnit), 0, st>>>(p, wgs);
  return hipGetLastError();
}

}  // namespace attnres
