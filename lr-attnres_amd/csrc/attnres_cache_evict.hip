// The paged cache reduced to a budget: per key / value head the most attended and the
// last tokens, copied in their order to other pages.
//
// Choice (one workgroup a head).  Weights become keys whose unsigned order is theirs (a NaN
// below all), held in registers; the budget-th largest is found in three rounds of 12, 10 and 10
// bits counted in LDS (twelve first: weights lie in few octaves, and lanes that count into one
// place wait for each other), fewer where a round leaves nothing open.  What lies above it and, of
// what equals it, the first ones are kept: their places come from counts a wave and 64 tokens,
// scanned once.  Bound by the latency of its rounds and barriers.
// Copy.  Places are independent: every kept row is read and written once by the lanes of
// its own, so nothing is ordered and nothing waits.  Bound by memory.
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

__device__ __forceinline__ int wave_scan(int x) {  // inclusive
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int y = __shfl_up(x, o, kWave);
    if (lane >= o) x += y;
  }
  return x;
}

// x summed over the workgroup's threads up to and with this one; `sums`: one place a wave
__device__ __forceinline__ int block_scan(int x, int* sums) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  x = wave_scan(x);
  if (lane == kWave - 1) sums[wave] = x;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelThreads / kWave; ++w)
    if (w < wave) x += sums[w];
  return x;
}

// R: keys that a thread holds; longer caches are read again, R * 1024 tokens at a time, in every round
template <int R>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(CacheEvictParams p) {
  const CachePages& c = p.c;
  const int b = blockIdx.x / c.kv_heads, h = blockIdx.x % c.kv_heads;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  constexpr int kWaves = kSelThreads / kWave, kBlock = R * kSelThreads;
  constexpr int kBins = 4096, kMine = kBins / kSelThreads;
  __shared__ int hist[kBins];
  __shared__ int sums[2][kWaves];
  __shared__ int s_digit, s_want, s_open;
  __shared__ int s_above[R * kWaves], s_equal[R * kWaves];
  int n = cache_count(c, b);
  if (n < 0) n = 0;
  const int budget = p.budget;
  int32_t* kept = p.kept + (int64_t)blockIdx.x * budget;
  if (h == 0 && tid == 0) p.left[b] = min(n, budget);
  if (n <= budget) {
    for (int i = tid; i < budget; i += kSelThreads) kept[i] = i < n ? i : -1;
    return;
  }
  const int early = n - p.recent;  // the tokens to choose from
  int want = budget - p.recent;    // and how many of them; want < early
  for (int i = tid; i < p.recent; i += kSelThreads) kept[budget - p.recent + i] = early + i;
  if (want == 0) return;

  uint32_t key[R];
  auto load = [&](int j0) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int j = j0 + i * kSelThreads + tid;
      key[i] = j < early ? token_key(c, b, h, j) : 0;
    }
  };
  load(0);
  uint32_t prefix = 0, mask = 0;
  for (int round = 0, bits = 12, shift = 20; round < 3; ++round, bits = 10, shift -= 10) {
    for (int i = tid; i < 1 << bits; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int j0 = 0; j0 < early; j0 += kBlock) {
      if (early > kBlock) load(j0);
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (j0 + i * kSelThreads + tid < early && (key[i] & mask) == prefix)
          atomicAdd(&hist[(key[i] >> shift) & ((1 << bits) - 1)], 1);
    }
    __syncthreads();
    // from the largest digit down: a thread's places, and what lies above them
    const int mine = round == 0 ? kMine : 1, first = (1 << bits) - 1 - tid * mine;
    int sum = 0;
    for (int i = 0; i < mine; ++i) sum += hist[first - i];
    int upto = block_scan(sum, sums[0]);
    if (upto >= want && upto - sum < want) {
      int left = want - (upto - sum), i = 0;
      while (hist[first - i] < left) left -= hist[first - i++];
      s_digit = first - i;
      s_want = left;
      s_open = hist[first - i] > left;
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit << shift;
    mask |= ((1u << bits) - 1) << shift;
    want = s_want;
    if (!s_open) break;  // all that have these digits are kept
  }
  // kept: what lies above prefix, and of what equals it the first `want`
  int above = 0, equal = 0;  // in the blocks before
  for (int j0 = 0; j0 < early; j0 += kBlock) {
    if (early > kBlock) load(j0);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const bool in = j0 + i * kSelThreads + tid < early;
      const uint64_t a = __ballot(in && (key[i] & mask) > prefix), e = __ballot(in && (key[i] & mask) == prefix);
      if (lane == 0) {
        s_above[i * kWaves + wave] = __popcll(a);
        s_equal[i * kWaves + wave] = __popcll(e);
      }
    }
    __syncthreads();
    const int a0 = tid < R * kWaves ? s_above[tid] : 0, e0 = tid < R * kWaves ? s_equal[tid] : 0;
    const int a1 = block_scan(a0, sums[0]), e1 = block_scan(e0, sums[1]);
    if (tid < R * kWaves) {
      s_above[tid] = above + a1 - a0;
      s_equal[tid] = equal + e1 - e0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int j = j0 + i * kSelThreads + tid;
      const bool is_above = j < early && (key[i] & mask) > prefix, is_equal = j < early && (key[i] & mask) == prefix;
      const uint64_t below = (1ull << lane) - 1;
      const int a = s_above[i * kWaves + wave] + __popcll(__ballot(is_above) & below);
      const int e = s_equal[i * kWaves + wave] + __popcll(__ballot(is_equal) & below);
      if (is_above || (is_equal && e < want)) kept[a + min(e, want)] = j;
    }
#pragma unroll
    for (int w = 0; w < kWaves; ++w) above += sums[0][w], equal += sums[1][w];
  }
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
  // keys of the longest table in registers, where 64 a thread are enough
  const dim3 sel((unsigned)heads), wg(kSelThreads);
  if (p.c.room <= 4 * kSelThreads) evict_select_kernel<4><<<sel, wg, 0, st>>>(p);
  else if (p.c.room <= 16 * kSelThreads) evict_select_kernel<16><<<sel, wg, 0, st>>>(p);
  else evict_select_kernel<64><<<sel, wg, 0, st>>>(p);
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
