// Internal interface of the paged cache's kernels (attnres_cache_*.hip) and their
// C ABI (attnres_cache_capi.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace attnres {

// records the message that attnres_last_error() returns and gives back `code`
int api_fail(int code, const char* fmt, ...);

// n / d for 0 <= n < 2^31 and 1 <= d < 2^31 by a product: with 2^s < d <= 2^(s+1) and mul = ceil(2^(32+s) / d), mul * d
// exceeds 2^(32+s) by less than d <= 2^(s+1), so that n * mul / 2^(32+s) exceeds n / d by less than 1 / d.
struct FastDiv {
  uint32_t mul, shift;  // mul 0: d is 1
};
inline FastDiv fast_div(int32_t d) {
  if (d <= 1) return FastDiv{0, 0};
  uint32_t s = 0;
  while (((int64_t)2 << s) < d) ++s;
  return FastDiv{(uint32_t)((((uint64_t)1 << (32 + s)) + d - 1) / d), s};
}

struct CachePages {  // attnres_cache_desc
  void* k;
  void* v;
  int64_t page_stride, head_stride, slot_stride;
  float* w;
  int64_t w_page_stride, w_head_stride;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* cached;
  const int32_t* fresh;
  int32_t batch, kv_heads, head_dim, page_size, pages;
  int32_t room;  // tokens that a row of the table has pages for
  FastDiv by_page;  // page_size
  uint32_t page_bytes, slot_bytes;  // the strides, where a page lies within 32 bits
};

struct CacheAppendParams {
  CachePages c;
  const void* qkv;
  int64_t b_stride, t_stride;
  int32_t n_tok, tokens;  // batch * tokens; times the heads of a token below 2^31
  FastDiv by_tokens;
  int32_t q_heads, qk_norm;
  float eps;
  const void* sin;
  const void* cos;
  int64_t table_rows, table_stride;
  const int32_t* pos;
  void* q;
  void* k;  // or null
};

// vec: values of a load; lanes: loads of that width that cover a head
hipError_t launch_cache_append(int dtype, bool f32_table, const CacheAppendParams& p, int vec, int lanes, hipStream_t st);

constexpr int kAttUnit = 128;  // tokens of a unit of attention's work

struct CacheAttendParams {
  CachePages c;
  const void* q;
  int64_t q_b_stride, q_h_stride, q_t_stride;
  int32_t tokens, q_heads;
  int32_t group, rows, blocks;  // query heads of a key / value head; with the new tokens; blocks of them
  int32_t row_bits;             // 4 or 5: rows of a block, 2^row_bits
  int32_t wgs;                  // of a split cache
  int32_t weight_waves;         // that add the weights up in a launch of their own, four a workgroup
  int32_t own_weights;          // the workgroup of a whole segment does it
  FastDiv by_group, by_blocks, by_segs, by_wgs, by_weight_waves;  // segments: kv_heads * blocks
  int32_t direct;               // a workgroup takes a whole segment
  int32_t tile;                 // 64 / 128 / 256: the head width it covers
  int32_t vb;                   // bytes (16, 8, 4 or a value's) that every row starts and ends at a multiple of
  int32_t page16, whole, q_vec; // pages of whole 16 tokens; heads as wide as the tile; queries in rows of 16 bytes
  int32_t negate;               // the queries
  float scale;                  // of base-2 logarithms: the softmax's scale times log2(e), > 0
  float decay;
  void* out;
  float* part;     // [2 wgs][rows of a block][tile], pieces of rows
  float* part_ml;  // [2 wgs][rows of a block][2], their maxima and sums
  float* row_ml;   // [batch, q_heads][2], with weights: of rows that one workgroup had
  float* logits;   // [batch, q_heads, logit_stride], with weights
  int64_t logit_stride;
};

hipError_t launch_cache_attend_bf16(const CacheAttendParams& p, hipStream_t st);
hipError_t launch_cache_attend_f16(const CacheAttendParams& p, hipStream_t st);
hipError_t launch_cache_attend_f32(const CacheAttendParams& p, hipStream_t st);

constexpr int kEvictSlice = 8192;  // tokens whose keys a workgroup holds (twice as many where it has a whole head)
constexpr int kEvictSlots = 3080;  // counts and state of a workgroup, 4 bytes each

struct CacheEvictParams {
  CachePages c;
  const int32_t* new_table;
  int64_t new_stride;
  int32_t budget, recent;
  int32_t* kept;
  int32_t* left;
  int32_t es;   // bytes of a value
  int32_t slices;  // of a table
  int32_t* hist;   // [heads][slices][kEvictSlots], where there are several
  int32_t vb;      // bytes (16, 8, 4 or a value's) that every row starts and ends at a multiple of
};

hipError_t launch_cache_evict(const CacheEvictParams& p, hipStream_t st);

#ifdef __HIP__

__device__ __forceinline__ int div_by(int n, const FastDiv& d) {
  return d.mul ? (int)(__umulhi((uint32_t)n, d.mul) >> d.shift) : n;
}

// tokens in the cache before the call: 0 .. room, or -1 for a count that the table has no room for
__device__ __forceinline__ int cache_count(const CachePages& c, int b) {
  const int n = c.cached[b];
  return n >= 0 && n <= c.room ? n : -1;
}

// over the lanes up to and with this one, by moves inside rows of 16 lanes and broadcasts of a row's last
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // 1, 2, 4, 8 to the right
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // lane 15 into rows 1 and 3's, of 0 and 2
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31 into rows 2 and 3
  return x;
}

#endif

}  // namespace attnres
