// The paged cache reduced to a budget: per key / value head the most attended and the
// last tokens, copied in their order to other pages.
//
// Choice (one workgroup a head).  Weights become keys whose unsigned order is theirs (a NaN
// below all); the budget-th largest is found in four rounds of eight bits, counted in LDS,
// and one ordered pass marks what lies above it and, of what equals it, the first ones.
// Copy.  Places are independent: every kept row is read and written once by the lanes of
// its own, so nothing is ordered and nothing waits.
#include "attnres_cache.h"
#include "attnres_device.h"

namespace attnres {

namespace {

constexpr int kSelThreads = 1024;

__device__ __forceinline__ uint32_t weight_key(float w) {
  if (!(w == w)) return 0;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t token_key(const CachePages& c, int b, int h, int j) {
  const int page = cache_page(c, b, j);
  return page < 0 ? 0 : weight_key(c.w[page * c.w_page_stride + h * c.w_head_stride + j % c.page_size]);
}

__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(CacheEvictParams p) {
  const CachePages& c = p.c;
  const int b = blockIdx.x / c.kv_heads, h = blockIdx.x % c.kv_heads;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  constexpr int kWaves = kSelThreads / kWave;
  __shared__ int hist[256];
  __shared__ uint32_t s_digit;
  __shared__ int s_want;
  __shared__ int s_above[kWaves], s_equal[kWaves];
  int n = cache_count(c, b);
  if (n < 0) n = 0;
  const int budget = p.budget;
  int32_t* kept = p.kept + (int64_t)blockIdx.x * budget;
  if (h == 0 && tid == 0) p.left[b] = min(n, budget);
  if (n <= budget) {
    for (int i = tid; i < budget; i += kSelThreads) kept[i] = i < n ? i : -1;
    return;
  }
  const int early = n - p.recent;       // the tokens to choose from
  int want = budget - p.recent;         // and how many of them; want < early
  uint32_t prefix = 0, mask = 0;
  if (want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int j = tid; j < early; j += kSelThreads) {
        const uint32_t k = token_key(c, b, h, j);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int d = 255, w = want;
        while (d > 0 && hist[d] < w) w -= hist[d--];
        s_digit = d;
        s_want = w;
      }
      __syncthreads();
      prefix |= s_digit << shift;
      mask |= 255u << shift;
      want = s_want;
      __syncthreads();
    }
  }
  // above: keys larger than prefix; of those equal to it the first `want`
  int above = 0, equal = 0;  // seen in the tokens before this round's
  const bool any = budget > p.recent;
  for (int j0 = 0; j0 < early && any; j0 += kSelThreads) {
    const int j = j0 + tid;
    const uint32_t k = j < early ? token_key(c, b, h, j) : 0;
    const bool is_above = j < early && k > prefix, is_equal = j < early && k == prefix;
    const uint64_t ma = __ballot(is_above), me = __ballot(is_equal), below = (1ull << lane) - 1;
    if (lane == 0) {
      s_above[wave] = __popcll(ma);
      s_equal[wave] = __popcll(me);
    }
    __syncthreads();
    int a = above + __popcll(ma & below), e = equal + __popcll(me & below);
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) a += s_above[w], e += s_equal[w];
      above += s_above[w];
      equal += s_equal[w];
    }
    if (is_above) kept[a + min(e, want)] = j;
    else if (is_equal && e < want) kept[a + e] = j;
    __syncthreads();
  }
  for (int i = tid; i < p.recent; i += kSelThreads) kept[budget - p.recent + i] = early + i;
}

// lanes: of a row (its 16-byte vectors, or single values)
template <class V>
__global__ __launch_bounds__(256) void evict_copy_kernel(CacheEvictParams p, int lanes, int per, int64_t rows) {
  const CachePages& c = p.c;
  const int here = 256 / lanes, col = threadIdx.x % lanes;
  if ((int)threadIdx.x / lanes >= here) return;
  for (int64_t row = (int64_t)blockIdx.x * here + threadIdx.x / lanes; row < rows; row += (int64_t)gridDim.x * here) {
    const int bh = (int)(row / p.budget), i = (int)(row - (int64_t)bh * p.budget);
    const int b = bh / c.kv_heads, h = bh % c.kv_heads;
    const int j = p.kept[row];
    if (j < 0) continue;
    const int from = cache_page(c, b, j), to = p.new_table[b * p.new_stride + i / c.page_size];
    if (from < 0 || (unsigned)to >= (unsigned)c.pages) continue;
    const int slot = j % c.page_size, slot_to = i % c.page_size;
    if (from == to && slot == slot_to) continue;
    const int64_t src = from * c.page_stride + h * c.head_stride + slot * c.slot_stride;
    const int64_t dst = to * c.page_stride + h * c.head_stride + slot_to * c.slot_stride;
    for (int x = col; x < per; x += lanes) {
      const V k = ((const V*)((const char*)c.k + src * p.es))[x], v = ((const V*)((const char*)c.v + src * p.es))[x];
      ((V*)((char*)c.k + dst * p.es))[x] = k;
      ((V*)((char*)c.v + dst * p.es))[x] = v;
    }
    if (col == 0)
      c.w[to * c.w_page_stride + h * c.w_head_stride + slot_to] = c.w[from * c.w_page_stride + h * c.w_head_stride + slot];
  }
}

}  // namespace

hipError_t launch_cache_evict(const CacheEvictParams& p, hipStream_t st) {
  const int64_t heads = (int64_t)p.c.batch * p.c.kv_heads;
  evict_select_kernel<<<dim3((unsigned)heads), dim3(kSelThreads), 0, st>>>(p);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  const int size = p.vec ? 16 : p.es, per = p.c.head_dim * p.es / size;
  const int lanes = per < 64 ? per : 64;
  const int64_t rows = heads * p.budget, blocks = (rows + 256 / lanes - 1) / (256 / lanes);
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20));
  if (size == 16) evict_copy_kernel<u32x4><<<grid, dim3(256), 0, st>>>(p, lanes, per, rows);
  else if (size == 4) evict_copy_kernel<uint32_t><<<grid, dim3(256), 0, st>>>(p, lanes, per, rows);
  else evict_copy_kernel<uint16_t><<<grid, dim3(256), 0, st>>>(p, lanes, per, rows);
  return hipGetLastError();
}

}  // namespace attnres
