// The paged cache reduced to a budget: per key / value head the most attended and the
// last tokens, copied in their order to other pages.
//
// Choice.  Weights become keys whose unsigned order is theirs (a NaN below all), held in
// registers; the budget-th largest is found in three rounds of 12, 10 and 10 bits (256 threads:
// 11, 11 and 10) counted in LDS, fewer where a round leaves nothing open.  The first round takes most
// bits: weights lie in few octaves, and lanes that count into one place wait for each other (four
// copies of the counts, a quarter of the lanes each, were no faster).  What lies above the found key and, of what equals
// it, the first ones are kept: their places come from counts a wave and 64 tokens, scanned once.
// One workgroup a head, of 256 threads for tables of up to 2048 tokens (16 x 12 heads: 7.4 us; 1024 threads
// 8.4) and of 1024 up to 16384; longer tables are shared by one for each 8192 tokens, a launch a round
// (16 heads of up to 65536: 6 to 8 us each, 7.3 to place them).  Bound by latency: a launch, the chain
// of count, page and weight, and the rounds' barriers.
//
// Copy.  Places are independent: every kept row is read and written once by lanes of
// its own, so nothing is ordered and nothing waits.  Bound by memory: 102 MB of rows of 128 bytes in 20.7 us
// (4.9 TB/s), 139 MB of rows of 256 in 30.6 (4.5; they are gathered from caches eight times as large).  Two
// and four rows a thread at once: 22 and 27 us, 32 and 40.
#include "attnres_cache.h"
#include "attnres_device.h"

namespace attnres {

namespace {

__device__ __forceinline__ uint32_t weight_key(float w) {
  if (!(w == w)) return 0;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// TH: threads of a workgroup, 1024 or 256.  Places of a round's counts: 2^12, 2^10, 2^10, or 2^11, 2^11, 2^10.
constexpr int kBig = 1024, kFew = 256;
constexpr int kSlice = kEvictSlice, kR = kSlice / kBig;  // tokens of a workgroup, keys a thread
static_assert(kR * kBig == kSlice, "whole keys a thread");
template <int TH>
constexpr int kBins = TH == kBig ? 4096 : 2048;

template <int TH>
__device__ __forceinline__ int round_bits(int round) { return TH == kBig ? (round == 0 ? 12 : 10) : round == 2 ? 10 : 11; }
template <int TH>
__device__ __forceinline__ int round_shift(int round) { return TH == kBig ? 20 - 10 * round : round == 0 ? 21 : round == 1 ? 10 : 0; }

// x summed over the workgroup's threads up to and with this one; `sums`: one place a wave
template <int TH>
__device__ __forceinline__ int block_scan(int x, int* sums) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  x = wave_scan(x);
  if (lane == kWave - 1) sums[wave] = x;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < TH / kWave; ++w)
    if (w < wave) x += sums[w];
  return x;
}

// What the rounds so far have found: kept are the keys above prefix in the bits of mask, and `want` of those equal.
struct Found {
  uint32_t prefix, mask;
  int want;
  bool open;  // more are equal than wanted
};

template <int R, int TH>
struct SelectShared {
  int sums[2][TH / kWave];
  int digit, want, open, before_above, before_equal;
  int above[R * TH / kWave], equal[R * TH / kWave];
};

// The next digit of the want-th largest key from the counts of its places, 2^bits of them: count(low, n, before) of the
// thread's, low .. , backwards; `before` being those of n that lie in slices before this one.  In s.before_*: keys of
// theirs that are above the digit and equal to it.
template <bool SLICES, int R, int TH, class F>
__device__ __forceinline__ void next_digit(int round, Found& f, SelectShared<R, TH>& s, F count) {
  const int bits = round_bits<TH>(round), mine = (1 << bits) / TH;
  // from the largest place down
  const int first = (1 << bits) - 1 - (int)threadIdx.x * mine;
  int n[kBins<TH> / TH], before[kBins<TH> / TH], sum = 0, sum_before = 0;
#pragma unroll
  for (int i = 0; i < kBins<TH> / TH; ++i) n[i] = before[i] = 0;
  count(first - (mine - 1), n, before);
#pragma unroll
  for (int i = 0; i < kBins<TH> / TH; ++i) {
    sum += n[i];
    sum_before += before[i];
  }
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  int upto = wave_scan(sum), upto_before = SLICES ? wave_scan(sum_before) : 0;
  if (lane == kWave - 1) s.sums[0][wave] = upto, s.sums[1][wave] = upto_before;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < (TH / kWave); ++w)
    if (w < wave) {
      upto += s.sums[0][w];
      if (SLICES) upto_before += s.sums[1][w];
    }
  if (upto >= f.want && upto - sum < f.want) {
    int left = f.want - (upto - sum), above = upto_before - sum_before;
#pragma unroll
    for (int i = 0; i < kBins<TH> / TH; ++i) {
      if (left > 0 && left <= n[i]) {
        s.digit = first - i;
        s.want = left;
        s.open = n[i] > left;
        s.before_above = above;
        s.before_equal = before[i];
      }
      left -= n[i];
      above += before[i];
    }
  }
  __syncthreads();
  f.prefix |= (uint32_t)s.digit << round_shift<TH>(round);
  f.mask |= ((1u << bits) - 1) << round_shift<TH>(round);
  f.want = s.want;
  f.open = s.open;
}

// The tokens j0 .. of a head: what is kept of them goes to its places, `above` and `equal` of the tokens before them
// being above the found prefix and equal to it.
template <int R, int TH>
__device__ __forceinline__ void place(const uint32_t (&key)[R], int j0, int early, const Found& f, int above, int equal,
                                      int32_t* kept, SelectShared<R, TH>& s) {
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const bool in = j0 + i * TH + tid < early;
    const uint64_t a = __ballot(in && (key[i] & f.mask) > f.prefix), e = __ballot(in && (key[i] & f.mask) == f.prefix);
    if (lane == 0) {
      s.above[i * (TH / kWave) + wave] = __popcll(a);
      s.equal[i * (TH / kWave) + wave] = __popcll(e);
    }
  }
  __syncthreads();
  const int a0 = tid < R * TH / kWave ? s.above[tid] : 0, e0 = tid < R * TH / kWave ? s.equal[tid] : 0;
  const int a1 = block_scan<TH>(a0, s.sums[0]), e1 = block_scan<TH>(e0, s.sums[1]);
  if (tid < R * TH / kWave) {
    s.above[tid] = above + a1 - a0;
    s.equal[tid] = equal + e1 - e0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int j = j0 + i * TH + tid;
    const bool is_above = j < early && (key[i] & f.mask) > f.prefix, is_equal = j < early && (key[i] & f.mask) == f.prefix;
    const uint64_t below = (1ull << lane) - 1;
    const int a = s.above[i * (TH / kWave) + wave] + __popcll(__ballot(is_above) & below);
    const int e = s.equal[i * (TH / kWave) + wave] + __popcll(__ballot(is_equal) & below);
    if (is_above || (is_equal && e < f.want)) kept[a + min(e, f.want)] = j;
  }
}

// The keys of a head's tokens j0 .., as far as the table goes: no load waits for the sequence's length.
template <int R, int TH>
__device__ __forceinline__ void load_keys(const CachePages& c, int b, int h, int j0, uint32_t (&key)[R]) {
  int page[R], slot[R];
  float w[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int j = j0 + i * TH + (int)threadIdx.x, at = div_by(j, c.by_page);
    slot[i] = j - at * c.page_size;
    page[i] = j < c.room ? c.table[b * c.table_stride + at] : -1;
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
    w[i] = (unsigned)page[i] < (unsigned)c.pages ? c.w[page[i] * c.w_page_stride + h * c.w_head_stride + slot[i]] : __builtin_nanf("");
#pragma unroll
  for (int i = 0; i < R; ++i) key[i] = weight_key(w[i]);
}

template <int R, int TH>
__device__ __forceinline__ void count_keys(const uint32_t (&key)[R], int j0, int early, int round, const Found& f, int* hist) {
  const int bits = round_bits<TH>(round), shift = round_shift<TH>(round);
  for (int i = threadIdx.x; i < 1 << bits; i += TH) hist[i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (j0 + i * TH + (int)threadIdx.x < early && (key[i] & f.mask) == f.prefix)
      atomicAdd(&hist[(key[i] >> shift) & ((1 << bits) - 1)], 1);
  __syncthreads();
}

// what needs no choice; false: `early` tokens to choose budget - recent of
template <int TH>
__device__ __forceinline__ bool no_choice(const CacheEvictParams& p, int n, int32_t* kept) {
  if (n <= p.budget) {
    for (int i = threadIdx.x; i < p.budget; i += TH) kept[i] = i < n ? i : -1;
    return true;
  }
  for (int i = threadIdx.x; i < p.recent; i += TH) kept[p.budget - p.recent + i] = n - p.recent + i;
  return p.budget == p.recent;
}

// Rows i of what a head keeps: key, value and weight of each, from tokens j (none: -1), by `lanes` threads of which this
// is `col`; per: vectors V of a row.  The loads of U rows are on their way together.
template <class V, int U>
__device__ __forceinline__ void copy_rows(const CacheEvictParams& p, int b, int h, const int (&i)[U], const int (&j)[U], int col,
                                          int lanes, int per) {
  const CachePages& c = p.c;
  int from[U], to[U], slot[U], slot_to[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = div_by(max(j[u], 0), c.by_page), at_to = div_by(i[u], c.by_page);
    from[u] = j[u] < 0 ? -1 : c.table[b * c.table_stride + at];
    to[u] = j[u] < 0 ? -1 : p.new_table[b * p.new_stride + at_to];
    slot[u] = j[u] - at * c.page_size;
    slot_to[u] = i[u] - at_to * c.page_size;
  }
  bool move[U];
  int64_t src[U], dst[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    move[u] = (unsigned)from[u] < (unsigned)c.pages && (unsigned)to[u] < (unsigned)c.pages &&
              (from[u] != to[u] || slot[u] != slot_to[u]);
    src[u] = (from[u] * c.page_stride + h * c.head_stride + slot[u] * c.slot_stride) * p.es;
    dst[u] = (to[u] * c.page_stride + h * c.head_stride + slot_to[u] * c.slot_stride) * p.es;
  }
  for (int x = col; x < per; x += lanes) {
    V k[U], v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (move[u]) {
        k[u] = ((const V*)((const char*)c.k + src[u]))[x];
        v[u] = ((const V*)((const char*)c.v + src[u]))[x];
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (move[u]) {
        ((V*)((char*)c.k + dst[u]))[x] = k[u];
        ((V*)((char*)c.v + dst[u]))[x] = v[u];
      }
  }
  if (col == 0) {
    float w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (move[u]) w[u] = c.w[from[u] * c.w_page_stride + h * c.w_head_stride + slot[u]];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (move[u]) c.w[to[u] * c.w_page_stride + h * c.w_head_stride + slot_to[u]] = w[u];
  }
}

constexpr int kOwnRows = 4;  // on their way together, of a thread whose workgroup chose them

// What a head keeps, by the workgroup that chose it
template <class V, int TH>
__device__ __forceinline__ void copy_own(const CacheEvictParams& p, int b, int h, const int* kept) {
  const int per = p.c.head_dim * p.es / (int)sizeof(V), lanes = min(per, kWave), here = TH / lanes;
  const int col = threadIdx.x % lanes, row = threadIdx.x / lanes;
  if (row >= here) return;
  int i[kOwnRows], j[kOwnRows];
#pragma unroll
  for (int u = 0; u < kOwnRows; ++u) {
    i[u] = row + u * here;
    j[u] = i[u] < p.budget ? kept[i[u]] : -1;
  }
  copy_rows<V, kOwnRows>(p, b, h, i, j, col, lanes, per);
}

// tables of at most R * TH tokens; OWN: the workgroup copies what it chose
template <int R, int TH, bool OWN>
__global__ __launch_bounds__(TH) void evict_select_kernel(CacheEvictParams p) {
  __shared__ int hist[kBins<TH>];
  __shared__ SelectShared<R, TH> s;
  __shared__ int own[OWN ? TH * kOwnRows : 1];
  const int b = blockIdx.x / p.c.kv_heads, h = blockIdx.x % p.c.kv_heads;
  uint32_t key[R];
  load_keys<R, TH>(p.c, b, h, 0, key);
  const int n = max(cache_count(p.c, b), 0);
  int32_t* const out = p.kept + (int64_t)blockIdx.x * p.budget;
  int32_t* const kept = OWN ? own : out;
  if (h == 0 && threadIdx.x == 0) p.left[b] = min(n, p.budget);
  if (!no_choice<TH>(p, n, kept)) {
    const int early = n - p.recent;
    Found f{0, 0, p.budget - p.recent, true};
    for (int round = 0; round < 3 && f.open; ++round) {
      count_keys<R, TH>(key, 0, early, round, f, hist);
      next_digit<false>(round, f, s, [&](int low, int* n, int*) {
        const int mine = (1 << round_bits<TH>(round)) / TH;
#pragma unroll
        for (int i = 0; i < kBins<TH> / TH; ++i)
          if (i < mine) n[i] = hist[low + mine - 1 - i];
      });
    }
    place(key, 0, early, f, 0, 0, kept, s);
  }
  if constexpr (OWN) {
    __syncthreads();
    if (p.vb == 16) copy_own<u32x4, TH>(p, b, h, own);
    else if (p.vb == 8) copy_own<u32x2, TH>(p, b, h, own);
    else if (p.vb == 4) copy_own<uint32_t, TH>(p, b, h, own);
    else copy_own<uint16_t, TH>(p, b, h, own);
    for (int i = threadIdx.x; i < p.budget; i += TH) out[i] = own[i];
  }
}

// Longer tables: kSlice tokens a workgroup, a launch for each round's counts and one that places what is kept.  Each
// launch finds the digit of the round before it, from the counts of all of the head's slices, and each workgroup
// keeps what it has found for its next launch.
// hist[head][slice]: counts of 16 bits of 4096, 1024, 1024 places, then prefix, mask, want, open, above, equal
constexpr int kSlots = kEvictSlots, kState = 2048 + 2 * 512;
static_assert(kSlots >= kState + 6 && kSlots % 2 == 0 && kSlice < 1 << 16, "places and state");
__device__ __forceinline__ int round_at(int round) { return round == 0 ? 0 : 2048 + 512 * (round - 1); }

// What the rounds before `round` have found; above, equal: keys of the slices before this one.
__device__ __forceinline__ Found found_before(const CacheEvictParams& p, int head, int slices, int slice, int round, int* above,
                                              int* equal, SelectShared<kR, kBig>& s) {
  Found f{0, 0, p.budget - p.recent, true};
  int a = 0, e = 0;
  int32_t* state = p.hist + ((int64_t)head * p.slices + slice) * kSlots + kState;
  if (round > 1) {
    f = Found{(uint32_t)state[0], (uint32_t)state[1], state[2], state[3] != 0};
    a = state[4];
    e = state[5];
  }
  if (round > 0 && f.open) {
    const int32_t* at = p.hist + (int64_t)head * p.slices * kSlots + round_at(round - 1);
    // four places of the first round's a thread, in one load, one of the others'
    static_assert(kBins<kBig> == 4 * kBig, "four places a thread");
    next_digit<true>(round - 1, f, s, [&](int low, int* n, int* before) {
      for (int i0 = 0; i0 < slices; i0 += 8)  // (eight slices' loads at once)
#pragma unroll
        for (int i = i0; i < i0 + 8; ++i) {
          const int32_t* from = at + (int64_t)min(i, slices - 1) * kSlots;
          u32x2 x = {0, 0};
          if (round == 1) x = *(const u32x2*)(from + low / 2);
          else x.y = (uint32_t)((const uint16_t*)from)[low] << 16;
          const int places[4] = {(int)(x.y >> 16), (int)(x.y & 0xffff), (int)(x.x >> 16), (int)(x.x & 0xffff)};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            n[q] += i < slices ? places[q] : 0;
            before[q] += i < slice ? places[q] : 0;
          }
        }
    });
    a += s.before_above;
    e = s.before_equal;
  }
  if (round < 3 && threadIdx.x == 0) {
    state[0] = (int32_t)f.prefix;
    state[1] = (int32_t)f.mask;
    state[2] = f.want;
    state[3] = f.open;
    state[4] = a;
    state[5] = e;
  }
  *above = a;
  *equal = e;
  return f;
}

// A head's slices in neighbouring places, which one XCD has: its L2 then holds the counts that they all read.
__device__ __forceinline__ int place_of_block() {
  const int grid = gridDim.x;
  return grid % 8 ? (int)blockIdx.x : (int)(blockIdx.x % 8 * (grid / 8) + blockIdx.x / 8);
}

__global__ __launch_bounds__(kBig) void evict_count_kernel(CacheEvictParams p, int round) {
  __shared__ int hist[kBins<kBig>];
  __shared__ SelectShared<kR, kBig> s;
  const int at = place_of_block(), head = at / p.slices, slice = at - head * p.slices;
  const int b = head / p.c.kv_heads, h = head - b * p.c.kv_heads, n = max(cache_count(p.c, b), 0);
  const int early = n - p.recent, j0 = slice * kSlice;
  if (n <= p.budget || p.budget == p.recent || j0 >= early) return;
  uint32_t key[kR];
  load_keys<kR, kBig>(p.c, b, h, j0, key);
  int above, equal;
  const Found f = found_before(p, head, (early + kSlice - 1) / kSlice, slice, round, &above, &equal, s);
  if (!f.open) return;
  count_keys<kR, kBig>(key, j0, early, round, f, hist);
  int32_t* to = p.hist + ((int64_t)head * p.slices + slice) * kSlots + round_at(round);
  for (int i = threadIdx.x; i < 1 << (round_bits<kBig>(round) - 1); i += kBig) to[i] = hist[2 * i] | hist[2 * i + 1] << 16;
}

__global__ __launch_bounds__(kBig) void evict_place_kernel(CacheEvictParams p) {
  __shared__ SelectShared<kR, kBig> s;
  const int at = place_of_block(), head = at / p.slices, slice = at - head * p.slices;
  const int b = head / p.c.kv_heads, h = head - b * p.c.kv_heads, n = max(cache_count(p.c, b), 0);
  int32_t* kept = p.kept + (int64_t)head * p.budget;
  if (slice == 0) {
    if (h == 0 && threadIdx.x == 0) p.left[b] = min(n, p.budget);
    if (no_choice<kBig>(p, n, kept)) return;
  }
  const int early = n - p.recent, j0 = slice * kSlice;
  if (n <= p.budget || p.budget == p.recent || j0 >= early) return;
  uint32_t key[kR];
  load_keys<kR, kBig>(p.c, b, h, j0, key);
  int above, equal;
  const Found f = found_before(p, head, (early + kSlice - 1) / kSlice, slice, 3, &above, &equal, s);
  place(key, j0, early, f, above, equal, kept, s);
}

// lanes: of a row (of its vectors V)
template <class V>
__global__ __launch_bounds__(256) void evict_copy_kernel(CacheEvictParams p, int lanes, int per, int64_t rows) {
  const int here = 256 / lanes, col = threadIdx.x % lanes;
  if ((int)threadIdx.x / lanes >= here) return;
  for (int64_t row = (int64_t)blockIdx.x * here + threadIdx.x / lanes; row < rows; row += (int64_t)gridDim.x * here) {
    const int bh = (int)(row / p.budget), i = (int)(row - (int64_t)bh * p.budget);
    const int b = bh / p.c.kv_heads, h = bh % p.c.kv_heads, j = p.kept[row];
    if (j >= 0) copy_rows<V, 1>(p, b, h, {i}, {j}, col, lanes, per);
  }
}

}  // namespace

hipError_t launch_cache_evict(const CacheEvictParams& p, hipStream_t st) {
  const int64_t heads = (int64_t)p.c.batch * p.c.kv_heads;
  const dim3 sel((unsigned)(heads * p.slices)), wg(kBig);
  const int per = p.c.head_dim * p.es / p.vb, lanes = per < 64 ? per : 64;
  // A workgroup copies what it chose where its threads take all of it at once, so that no second launch waits for the first
  // (us, one / two launches: 3 heads, 49 rows of 64 16-bit values 7.9 / 10.0; 16 x 12 heads, 128 rows 10.4 / 11.1; 40 x 16 heads
  // 15.0 / 17.4; 16 x 8 heads, 64 rows of 128 9.9 / 10.4.  In two turns: 128 rows of 128 14.0 / 12.0, 256 of 64 14.8 / 13.6).
  const bool own = p.c.room <= kR * kFew && p.budget <= kFew / lanes * kOwnRows;
  if (p.slices == 1) {
    if (own) evict_select_kernel<kR, kFew, true><<<sel, dim3(kFew), 0, st>>>(p);
    else if (p.c.room <= kR * kFew) evict_select_kernel<kR, kFew, false><<<sel, dim3(kFew), 0, st>>>(p);
    else if (p.c.room <= kSlice) evict_select_kernel<kR, kBig, false><<<sel, wg, 0, st>>>(p);
    else evict_select_kernel<2 * kR, kBig, false><<<sel, wg, 0, st>>>(p);
  } else {
    for (int round = 0; round < 3; ++round) evict_count_kernel<<<sel, wg, 0, st>>>(p, round);
    evict_place_kernel<<<sel, wg, 0, st>>>(p);
  }
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || own) return err;
  const int64_t rows = heads * p.budget, blocks = (rows + 256 / lanes - 1) / (256 / lanes);
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20));
  if (p.vb == 16) evict_copy_kernel<u32x4><<<grid, dim3(256), 0, st>>>(p, lanes, per, rows);
  else if (p.vb == 8) evict_copy_kernel<u32x2><<<grid, dim3(256), 0, st>>>(p, lanes, per, rows);
  else if (p.vb == 4) evict_copy_kernel<uint32_t><<<grid, dim3(256), 0, st>>>(p, lanes, per, rows);
  else evict_copy_kernel<uint16_t><<<grid, dim3(256), 0, st>>>(p, lanes, per, rows);
  return hipGetLastError();
}

}  // namespace attnres
