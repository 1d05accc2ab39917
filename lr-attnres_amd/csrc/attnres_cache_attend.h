// Attention of the newest tokens over the paged cache.
//   p_j = softmax_j(scale <q, k_j>),   out = sum_j p_j v_j,   j < cached + t + 1
//
// Bound by memory: each key and value is read once for the (up to 16) query rows of its
// head -- the heads of its group times the new tokens -- so 2 rows flops a byte in 16 bits.  4 x 4 heads of
// 128 over 32768 to 131072 tokens, bf16: 782 MB in 135 us (5.8 TB/s; 6.2 without the ramp of the first tiles).  Rows
// above 16 read it again, from L2, at what a CU takes (48 bytes a ns), but where that is much two blocks of 16 share a
// workgroup's tiles: 128 rows of 16 x 2 heads of 64 over 4096 to 8192 tokens 53 -> 40 us, against 17 for 8 rows.  Four blocks
// were no faster: what is saved in loads is waited for in one wave's chain of products and exponentials.
//
// Products.  Query rows are columns of 16 x 16 matrix-core tiles: S^T = K Q^T with a tile's
// tokens as rows, then O^T = V^T P^T.  Lane l holds column l % 16 of both, so a row's maximum,
// sum and rescaling stay in its lanes, and the scores leave the first product in the very
// lanes in which the second takes its weights: nothing goes through LDS.  A lane loads 16 bytes of
// a key row as the product takes them, and of each of its tokens' value rows W consecutive
// values, turned in registers (one byte permute a word) into the columns that the product
// wants; output rows are d in the order (chunk, lane, value), put right when they are stored.
// The idle 16 - rows columns cost matrix-core time that a memory-bound kernel does not miss.
//
// Rounding.  Scores, weights, sums and outputs are fp32; a weight goes into the 16-bit
// product as the sum of two terms, rounded and the rest (one term alone would add an error
// as large as the result's own rounding); fp16 weights are scaled by 2^14 so that small ones
// keep their bits.
//
// Work.  A cache's units (kAttUnit tokens of one sequence's head and block of rows) are dealt
// evenly to a fixed number of workgroups from the lengths on the device, whatever they are:
// no length is known to the host, and a long sequence among short ones is shared by many.  A
// workgroup that has a head's whole length writes its rows; pieces go to the workspace as
// maximum, sum and output, joined by a second launch (3.5 to 5 us; 37 for 32768 rows).  Where the tables are so short
// that a workgroup can take a whole segment in less than that, each does, and there is one launch.
#pragma once

#include "attnres_cache.h"
#include "attnres_device.h"
#include "attnres_swiglu.h"

namespace attnres {

constexpr int kAttWaves = 4;

// The deal: `segs` segments (heads, blocks of rows) of each sequence, kAttUnit tokens a unit, unit x to
// workgroup deal_of(x).
struct Deal {
  int total, per, more;  // units; of a workgroup; the first `more` have one more
};

typedef const __attribute__((address_space(4))) int32_t att_const_i32;  // read by the scalar unit

// tokens that a sequence's queries see together; 0: it has none, -1: counts that cannot be
__device__ __forceinline__ int seen_of(const CacheAttendParams& p, int have, int fresh) {
  const int64_t n = (int64_t)have + fresh;
  if (have < 0 || fresh < 0 || n > p.c.room || (fresh > 0 && p.c.pages == 0)) return -1;
  return fresh > 0 ? (int)n : 0;
}
__device__ __forceinline__ int units_of(int n) { return (max(n, 0) + kAttUnit - 1) / kAttUnit; }

struct Seq {
  int have, n;
};
__device__ __forceinline__ Seq seq_of(const CacheAttendParams& p, int b) {  // b the same in all lanes
  const int have = ((att_const_i32*)(uintptr_t)p.c.cached)[b];
  const int fresh = p.c.fresh ? min(((att_const_i32*)(uintptr_t)p.c.fresh)[b], p.tokens) : p.tokens;
  return Seq{have, seen_of(p, have, fresh)};
}

// 64 sequences, one a lane: those from b0 on
struct Chunk {
  int b0, have, n, units, upto;  // upto: units of a segment of each sequence up to and with this one
  __device__ __forceinline__ void load(const CacheAttendParams& p, int b0_, int before) {
    const int b = b0_ + (int)(threadIdx.x & (kWave - 1));
    b0 = b0_;
    have = n = 0;
    if (b < p.c.batch) {
      have = p.c.cached[b];
      n = seen_of(p, have, p.c.fresh ? min(p.c.fresh[b], p.tokens) : p.tokens);
    }
    units = units_of(n);
    upto = wave_scan(units) + before;
  }
  __device__ __forceinline__ int last() const { return __builtin_amdgcn_readlane(upto, kWave - 1); }
};

// A cache's units among `wgs` workgroups.  Leaves the last 64 sequences in `c` (all of them, mostly).
__device__ __forceinline__ Deal deal(const CacheAttendParams& p, int segs, int wgs, const FastDiv& by_wgs, Chunk& c) {
  c.load(p, 0, 0);
  for (int b0 = kWave; b0 < p.c.batch; b0 += kWave) c.load(p, b0, c.last());
  Deal d;
  d.total = c.last() * segs;
  d.per = div_by(d.total, by_wgs);
  d.more = d.total - d.per * wgs;
  return d;
}
__device__ __forceinline__ int deal_start(const Deal& d, int w) { return w * d.per + min(w, d.more); }
__device__ __forceinline__ int deal_of(const Deal& d, int x) {
  const int big = d.more * (d.per + 1);
  return x < big ? x / (d.per + 1) : d.more + (x - big) / max(d.per, 1);
}

// The sequence that unit x is of, its first unit and how many a segment has.  Every x below the total is of one.
__device__ __forceinline__ void find_unit(const CacheAttendParams& p, int segs, int x, Chunk& c, int* b, Seq* q, int* start,
                                          int* units) {
  if (p.c.batch > kWave) {
    c.load(p, 0, 0);
    while (x >= c.last() * segs) c.load(p, c.b0 + kWave, c.last());
  }
  const int i = __popcll(__ballot(c.upto * segs <= x));
  *b = c.b0 + i;
  q->have = __builtin_amdgcn_readlane(c.have, i);
  q->n = __builtin_amdgcn_readlane(c.n, i);
  *units = __builtin_amdgcn_readlane(c.units, i);
  *start = (__builtin_amdgcn_readlane(c.upto, i) - *units) * segs;
}

#ifdef ATTNRES_CACHE_ATTEND_KERNELS

// A matrix product's result must not be read for 8 (16 bits) or 10 (fp32) issue slots.  The compiler counts them, but where
// a branch around some code lies between it has been seen to count the way through that code alone: the short way then
// reads too soon (a score tile whose zeroing branch came right before it was read two instructions after its product, and
// wrong).  Branches come from plain selects too, so this waits where one may come between (16 slots instead of 10: 24 x 40 / 5 heads of 32
// over up to 6506 tokens, fp16, with weights, 29.40 us instead of 29.25; none at all 28.95).
__device__ __forceinline__ void att_settle() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 9");
  __builtin_amdgcn_sched_barrier(0);
}

typedef _Float16 att_h4 __attribute__((ext_vector_type(4)));

// HD: head width's tile (64, 128, 256); VB: bytes that every row starts and ends at a multiple of, and that one load
// takes (16, or 8, 4, 2); PAGE16 (VB 16): pages of a multiple of 16 tokens, so that 16 tokens lie in one and the
// scalar unit finds it.  RB: blocks of 16 query rows that a workgroup has.
template <class DT, int HD, int VB, bool PAGE16, int RB>
struct Att {
  using S = typename DT::S;
  static constexpr int kSize = sizeof(S);
  static constexpr int kPer = 16 / kSize;                      // values of a key chunk
  static constexpr int kKs = HD * kSize / 64;                  // key chunks of a lane
  static constexpr bool k32 = kSize == 4;
  static constexpr bool VEC = VB == 16;
  static constexpr int kG = VB / kSize;                        // values of a load
  static constexpr int kSub = k32 || HD == 256 ? 1 : 2;        // 16-token subtiles of a tile (one: half the registers)
  static constexpr int kTok = 16 * kSub;
  static constexpr int kW = k32 ? 4 : HD == 64 ? 4 : 8;        // values of a value chunk
  static constexpr int kNi = HD / (16 * kW);
  static constexpr int kWords = kW * kSize / 4;
  static constexpr int kPitch = HD + 4;
  static constexpr float kShift = DT::kCode == 2 ? 14.f : 0.f;
  static constexpr float kCare = DT::kCode == 2 ? 0.f : 31.f;  // (fp16 values are far below fp32's largest)
  static constexpr int kStep = kAttWaves * kTok;               // tokens of a workgroup's round

  const CacheAttendParams& p;
  int lane, wave, c, g;          // column (query row of each block) and token group of the lane
  int b, h, n, have;
  int t_lo, t_hi;                // new tokens of the rows
  int kcol[kKs], vcol0;          // first value of each key chunk; of the first value chunk
  uint32_t kofs[kKs], vofs[4][kNi]; // PAGE16: bytes from a subtile's first row
  const S *kh, *vh;              // of the head, page 0
  att_const_i32* table;          // of the sequence
  u32x4 q[RB][kKs], k[kSub][kKs];
  uint32_t v[kSub][4][kNi][kWords];
  sw_f4 acc[RB][kNi][kW];
  float m[RB], l[RB];            // of the lane's rows: maximum of <q, k>, the lane's part of the sum
  float low;                     // the exponents' base is further up by it: kCare after a careful pass

  struct Rows {
    // PAGE16: of each subtile, bytes from the head's page 0 to its first token, and whether it has a page (one that has
    // none reads page 0)
    int64_t off[kSub];
    bool there[kSub];
    // else, of token `lane` of the tile: its page as the table has it (not looked at before the tile's loads: that
    // would wait for the table, and for all loads before it), and its slot
    int page, slot;
  };

  __device__ __forceinline__ Att(const CacheAttendParams& p_) : p(p_) {
    lane = threadIdx.x & (kWave - 1);
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    c = lane & 15;
    g = lane >> 4;
    const int Dh = p.c.head_dim;
    vcol0 = c * kW;
#pragma unroll
    for (int i = 0; i < kKs; ++i) kcol[i] = (i * 4 + g) * kPer;
    if constexpr (PAGE16) {  // lanes behind a row's end read inside it, and drop what they read
      const uint32_t slot = (uint32_t)p.c.slot_stride;
#pragma unroll
      for (int i = 0; i < kNi; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) vofs[t][i] = ((g * 4 + t) * slot + min(vcol0 + i * 16 * kW, Dh - kW)) * kSize;
#pragma unroll
      for (int i = 0; i < kKs; ++i) kofs[i] = (c * slot + min(kcol[i], Dh - kPer)) * kSize;
    }
  }

  // of the tile at t0 < limit: the sequence's length, or the table's room before that is known (a page that is not
  // there reads page 0, and the tile is not used)
  __device__ __forceinline__ Rows rows_of(int t0, int limit) const {
    Rows r;
    if constexpr (PAGE16) {
#pragma unroll
      for (int s = 0; s < kSub; ++s) {
        const uint32_t j = min((uint32_t)(t0 + 16 * s), (uint32_t)(limit - 1) & ~15u);
        const uint32_t at = __umulhi(j, p.c.by_page.mul) >> p.c.by_page.shift, slot = j - at * p.c.page_size;
        const uint32_t page = (uint32_t)table[at];
        r.there[s] = page < (uint32_t)p.c.pages;
        r.off[s] = (int64_t)((uint64_t)(r.there[s] ? page : 0) * p.c.page_bytes + slot * p.c.slot_bytes);
      }
    } else {
      const int j = min(t0 + (lane & (kTok - 1)), limit - 1), at = div_by(j, p.c.by_page);
      r.page = table[at];
      r.slot = j - at * p.c.page_size;
    }
    return r;
  }
  // values from the head's page 0 to token `lane` of the tile; of page 0 for one that has no page
  __device__ __forceinline__ int64_t token_off(const Rows& r) const {
    return (unsigned)r.page < (unsigned)p.c.pages ? r.page * p.c.page_stride + r.slot * p.c.slot_stride : 0;
  }

  // E values at `at`, whole words
  template <int E>
  static __device__ __forceinline__ void load_vec(const void* at, uint32_t* w) {
    if constexpr (E * kSize == 16) {
      const u32x4 x = *(const u32x4*)at;
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else if constexpr (E * kSize == 8) {
      const u32x2 x = *(const u32x2*)at;
      w[0] = x.x, w[1] = x.y;
    } else {
      w[0] = *(const uint32_t*)at;
    }
  }
  // values col .. col + E of a row, G a load; what is behind its end is read inside it (and not used)
  template <int E, int G>
  __device__ __forceinline__ void load_any(const S* row, int col, uint32_t* w) const {
    const int last = p.c.head_dim - G;
    if constexpr (G * kSize < 4) {
#pragma unroll
      for (int e = 0; e < E; e += 2)
        w[e / 2] = row[min(col + e, last)] | (uint32_t)row[min(col + e + 1, last)] << 16;
    } else {
      constexpr int kOne = G < E ? G : E;
#pragma unroll
      for (int e = 0; e < E; e += kOne) load_vec<kOne>(row + min(col + e, p.c.head_dim - kOne), w + e * kSize / 4);
    }
  }
  // the words of a chunk of 16 bytes from value col on, 0 behind the row's end
  __device__ __forceinline__ u32x4 inside(u32x4 w, int col) const {
    const int Dh = p.c.head_dim;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = col + i * 4 / kSize;
      if constexpr (k32) w[i] = at < Dh ? w[i] : 0;
      else w[i] = at + 1 < Dh ? w[i] : at < Dh ? w[i] & 0xffffu : 0;
    }
    return w;
  }

  // An offset as it is where it is used: one that is widened, added to or bounded outside the loop costs 64-bit
  // additions, or a register for each load.
  static __device__ __forceinline__ uint32_t here(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
  }

  __device__ __forceinline__ void load_k(const Rows& r) {
    const int64_t off = PAGE16 ? 0 : token_off(r);
#pragma unroll
    for (int s = 0; s < kSub; ++s) {
      if constexpr (PAGE16) {
        const char* row = (const char*)kh + r.off[s];
#pragma unroll
        for (int i = 0; i < kKs; ++i) k[s][i] = *(const u32x4*)(row + here(kofs[i]));
      } else {
        const S* row = kh + __shfl(off, 16 * s + c, kWave);
#pragma unroll
        for (int i = 0; i < kKs; ++i) {
          uint32_t w[4];
          load_any<kPer, kG>(row, (int)here(kcol[0]) + i * 4 * kPer, w);
          k[s][i] = u32x4{w[0], w[1], w[2], w[3]};
        }
      }
    }
  }

  __device__ __forceinline__ void load_v(const Rows& r) {
    const int64_t off = PAGE16 ? 0 : token_off(r);
#pragma unroll
    for (int s = 0; s < kSub; ++s)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if constexpr (PAGE16) {
          const char* row = (const char*)vh + r.off[s];
#pragma unroll
          for (int i = 0; i < kNi; ++i) load_vec<kW>(row + here(vofs[t][i]), v[s][t][i]);
        } else {
          const S* row = vh + __shfl(off, 16 * s + g * 4 + t, kWave);
#pragma unroll
          for (int i = 0; i < kNi; ++i) {
            load_any<kW, kG>(row, (int)here(vcol0) + i * 16 * kW, v[s][t][i]);
          }
        }
      }
  }

  // a tile's weights as the second product takes them: fp32, or in two terms
  struct Weights {
    u32x4 hi, lo;
    float e[kSub][4];
  };
  // two values in 16 bits; fp16 towards zero (one instruction): the second term takes what the first leaves
  static __device__ __forceinline__ uint32_t terms(float a, float b) {
    if constexpr (DT::kCode == 2) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
    else return pack2<DT>(a, b);
  }
  // SHOWN: a weight too small for the first term has its smallest value there, so that an infinite value times it is
  // infinite (fp16: 2^-38 of the largest weight, as much as the two terms may be off by anyway)
  template <bool SHOWN>
  static __device__ __forceinline__ Weights split(const float (&e)[kSub][4]) {
    Weights w;
#pragma unroll
    for (int s = 0; s < kSub; ++s)
#pragma unroll
      for (int t = 0; t < 4; t += 2) {
        w.e[s][t] = e[s][t], w.e[s][t + 1] = e[s][t + 1];
        if constexpr (!k32) {
          uint32_t x = terms(e[s][t], e[s][t + 1]);
          if constexpr (SHOWN) {
            x |= (x & 0xffffu) == 0 && e[s][t] > 0.f ? 1u : 0u;
            x |= x >> 16 == 0 && e[s][t + 1] > 0.f ? 0x10000u : 0u;
          }
          w.hi[s * 2 + t / 2] = x;
          w.lo[s * 2 + t / 2] = terms(e[s][t] - bits_to_float<DT>(x & 0xffffu), e[s][t + 1] - bits_to_float<DT>(x >> 16));
        }
      }
    return w;
  }
  // 16 tokens: a lane's four of each operand
  static __device__ __forceinline__ sw_f4 mfma16(u32x2 a, u32x2 b, sw_f4 to) {
    if constexpr (DT::kCode == 1)
      return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(sw_s4, a), __builtin_bit_cast(sw_s4, b), to, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(att_h4, a), __builtin_bit_cast(att_h4, b), to, 0, 0, 0);
  }
  // a pair of values, 0 for one that is not finite
  static __device__ __forceinline__ uint32_t finite(uint32_t w) {
    constexpr uint32_t kExp = DT::kCode == 1 ? 0x7f80u : 0x7c00u;
    return ((w & kExp) == kExp ? 0 : w & 0xffffu) | ((w >> 16 & kExp) == kExp ? 0 : w & 0xffff0000u);
  }
  // O^T += V^T P^T over a tile, value d of chunk i of the lanes' columns.  CARE: values of the lane's
  // tokens behind its `last` (16 s + t) count as 0, and an infinite value times the second term, which may have the
  // other sign, is left out.
  template <bool CARE>
  __device__ __forceinline__ sw_f4 weigh(const Weights& p, int i, int d, sw_f4 to, int last = 0) const {
    if constexpr (k32) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
        to = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(CARE && t > last ? 0 : v[0][t][i][d]), p.e[0][t], to, 0, 0, 0);
    } else {
      u32x4 a;
#pragma unroll
      for (int s = 0; s < kSub; ++s)
#pragma unroll
        for (int t = 0; t < 4; t += 2) {
          const uint32_t x = CARE && 16 * s + t > last ? 0 : v[s][t][i][d / 2];
          const uint32_t y = CARE && 16 * s + t + 1 > last ? 0 : v[s][t + 1][i][d / 2];
          a[s * 2 + t / 2] = d % 2 ? hi_pair(x, y) : lo_pair(x, y);
        }
      u32x4 a2 = a;
      if constexpr (CARE) {
#pragma unroll
        for (int x = 0; x < 2 * kSub; ++x) a2[x] = finite(a[x]);
      }
      if constexpr (kSub == 2) {
        sw_mfma<DT>(a, p.hi, to);
        sw_mfma<DT>(a2, p.lo, to);
      } else {
        to = mfma16({a.x, a.y}, {p.hi.x, p.hi.y}, to);
        to = mfma16({a2.x, a2.y}, {p.lo.x, p.lo.y}, to);
      }
    }
    return to;
  }

  // over the four lanes of a column
  template <class F>
  static __device__ __forceinline__ float across(float x, F f) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
  }

  // a maximum as the exponents' base; of no score at all: 0, so that -inf less it stays -inf
  __device__ __forceinline__ float base_of(float top) const { return top == -INFINITY ? 0.f : top * p.scale - kShift + low; }

  struct Row {       // one of the lane's
    float* logits;   // of token 0, or null
    int lim;         // tokens that it sees (one that is not there: whatever)
    int t;           // its new token
  };

  // The tile of tokens t0 .., whose keys and values are on their way.  AHEAD: all rows see all of it, and the next
  // tile's are loaded where its registers become free (in every turn of the loop: a load under a condition would make
  // each wait one for all loads).  CARE: a value that is not finite shows in the rows that see it and in no other, and
  // weights 2^31 times smaller keep sums of the largest values finite.
  template <bool AHEAD, bool CARE>
  __device__ __forceinline__ void tile(int t0, const Row (&row)[RB], Rows& now, Rows& next) {
    constexpr bool CUT = !AHEAD;
    Rows after;
    if constexpr (AHEAD) after = rows_of(min(t0 + 2 * kStep, (n - 1) & -kTok), n);
    if (!p.whole) {
#pragma unroll
      for (int s = 0; s < kSub; ++s)
#pragma unroll
        for (int i = 0; i < kKs; ++i) {
          if constexpr (!VEC) k[s][i] = inside(k[s][i], (int)here(kcol[0]) + i * 4 * kPer);
          else if (kcol[i] >= p.c.head_dim) k[s][i] = u32x4{0, 0, 0, 0};
        }
    }
    sw_f4 s4[RB][kSub];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int s = 0; s < kSub; ++s) {
        s4[r][s] = sw_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kKs; ++i) sw_mfma<DT>(k[s][i], q[r][i], s4[r][s]);
      }
    att_settle();
    // a page that is not there shows as NaN in the rows that see its tokens: all of them, or those that are not masked
    float scale[kSub];
#pragma unroll
    for (int s = 0; s < kSub; ++s) {
      scale[s] = PAGE16 && !CUT && !now.there[s] ? __builtin_nanf("") : p.scale;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const bool gone = PAGE16 ? CUT && !now.there[s] : (unsigned)__shfl(now.page, 16 * s + g * 4 + t, kWave) >= (unsigned)p.c.pages;
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          if (gone) s4[r][s][t] = __builtin_nanf("");
          if (CUT && t0 + 16 * s + g * 4 + t >= row[r].lim) s4[r][s][t] = -INFINITY;
        }
      }
    }
    if constexpr (AHEAD) load_k(next);
#pragma unroll
    for (int r = 0; r < RB; ++r)
      if (row[r].logits) {
#pragma unroll
        for (int s = 0; s < kSub; ++s) *(sw_f4*)(row[r].logits + t0 + 16 * s + g * 4) = s4[r][s] * scale[s];
      }
    float to[RB];
    bool higher = false;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      float top = s4[r][0][0];
#pragma unroll
      for (int s = 0; s < kSub; ++s)
#pragma unroll
        for (int t = 0; t < 4; ++t) top = fmaxf(top, s4[r][s][t]);
      top = across(top, [](float a, float b) { return fmaxf(a, b); });
      to[r] = fmaxf(m[r], top);
      higher |= to[r] != m[r];
    }
    if (__any(higher)) {
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const float was = m[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(base_of(m[r]) - base_of(to[r]));
        l[r] *= was;
#pragma unroll
        for (int i = 0; i < kNi; ++i)
#pragma unroll
          for (int d = 0; d < kW; ++d) acc[r][i][d] *= was;
        m[r] = to[r];
      }
    }
    if constexpr (CUT) {  // what lies behind the last token may be anything
#pragma unroll
      for (int s = 0; s < kSub; ++s)
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (t0 + 16 * s + g * 4 + t >= n) {
#pragma unroll
            for (int i = 0; i < kNi; ++i)
#pragma unroll
              for (int y = 0; y < kWords; ++y) v[s][t][i][y] = 0;
          }
    }
    const auto weights = [&](int r) {
      const float base = base_of(to[r]);
      float e[kSub][4];
#pragma unroll
      for (int s = 0; s < kSub; ++s)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          e[s][t] = __builtin_amdgcn_exp2f(__builtin_fmaf(s4[r][s][t], scale[s], -base));
          l[r] += e[s][t];
        }
      return split<CARE && DT::kCode == 2>(e);
    };
    if constexpr (!CARE) {
      Weights w[RB];
#pragma unroll
      for (int r = 0; r < RB; ++r) w[r] = weights(r);
#pragma unroll
      for (int i = 0; i < kNi; ++i)
#pragma unroll
        for (int d = 0; d < kW; ++d)
#pragma unroll
          for (int r = 0; r < RB; ++r) acc[r][i][d] = weigh<false>(w[r], i, d, acc[r][i][d]);
      if constexpr (AHEAD) {
        load_v(next);
        now = next;
        next = after;
      }
    } else {
      // (0 times such a value is NaN: each new token's rows take a product without the values behind it)
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const Weights w = weights(r);
        for (int tt = t_lo; tt <= t_hi; ++tt) {
#pragma unroll
          for (int i = 0; i < kNi; ++i)
#pragma unroll
            for (int d = 0; d < kW; ++d) {
              const sw_f4 with = weigh<true>(w, i, d, acc[r][i][d], have + tt - t0 - g * 4);
#pragma unroll
              for (int t = 0; t < 4; ++t) acc[r][i][d][t] = row[r].t == tt ? with[t] : acc[r][i][d][t];
            }
          att_settle();
        }
      }
    }
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int i = 0; i < kNi; ++i)
#pragma unroll
        for (int d = 0; d < kW; ++d) acc[r][i][d] = sw_f4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // tokens [first, end) of the head for rows [row0, row0 + rows), of those that there are (all of them, where a workgroup
  // takes a whole segment); this wave's: tiles wave, wave + 4, ...  stage: 16 rows of LDS that nobody uses.
  __device__ __forceinline__ void piece(int row0, int rows, int first, int end, Seq seq, void* stage) {
    table = (att_const_i32*)(uintptr_t)(p.c.table + b * p.c.table_stride);
    kh = (const S*)p.c.k + h * p.c.head_stride;
    vh = (const S*)p.c.v + h * p.c.head_stride;
    int t_row[RB], hq[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const int qr = row0 + 16 * r + c;
      t_row[r] = div_by(qr, p.by_group);
      hq[r] = h * p.group + qr - t_row[r] * p.group;
    }
    // (before the tiles' loads: a wait for what came last waits for all of them, in every turn of the loop)
    if (VEC && p.q_vec) {
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const S* src = (const S*)p.q + b * p.q_b_stride + hq[r] * p.q_h_stride + t_row[r] * p.q_t_stride;
#pragma unroll
        for (int i = 0; i < kKs; ++i) {
          q[r][i] = u32x4{0, 0, 0, 0};
          if (16 * r + c < rows && kcol[i] < p.c.head_dim) q[r][i] = *(const u32x4*)(src + kcol[i]);
        }
      }
    } else {  // (by single values, in few registers)
      S* const rows_q = (S*)stage;
#pragma unroll
      for (int r = 0; r < RB; ++r) {
#pragma unroll 1
        for (int i = threadIdx.x; i < 16 * HD; i += kAttWaves * kWave) {
          const int at = 16 * r + i / HD, col = i % HD, t = div_by(row0 + at, p.by_group);
          rows_q[i] = at < rows && col < p.c.head_dim
                          ? ((const S*)p.q)[b * p.q_b_stride + (h * p.group + row0 + at - t * p.group) * p.q_h_stride +
                                            t * p.q_t_stride + col]
                          : (S)0;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kKs; ++i) q[r][i] = *(const u32x4*)(rows_q + c * HD + kcol[i]);
        __syncthreads();
      }
    }
    // (the first tile's loads wait for the block table alone where the length is not known yet)
    const int t_first = first + wave * kTok, limit = p.direct ? p.c.room : seq.n;
    if (t_first >= limit) {
      clear();
      low = 0.f;
      n = seq.n;
      return;
    }
    Rows now = rows_of(t_first, limit), next;
    load_k(now);
    load_v(now);
    next = rows_of(min(t_first + kStep, (limit - 1) & -kTok), limit);
    if (p.negate) {
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int i = 0; i < kKs; ++i) q[r][i] ^= k32 ? 0x80000000u : 0x80008000u;
    }
    clear();
    low = 0.f;
    have = seq.have;
    n = seq.n;
    t_lo = div_by(row0, p.by_group);
    t_hi = div_by(row0 + rows - 1, p.by_group);
    end = min(end, min(have + t_hi + 1, n));  // (behind it no row sees any)
    const int all = have + t_lo + 1;          // tokens that every row sees
    if (t_first >= end) return;
    int t0 = t_first;
    Row row[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r)
      row[r] = Row{p.logits && 16 * r + c < rows ? p.logits + (b * (int64_t)p.q_heads + hq[r]) * p.logit_stride : nullptr,
                   min(have + t_row[r] + 1, n), t_row[r]};
    for (; t0 + kStep < end && t0 + kTok <= all; t0 += kStep) tile<true, false>(t0, row, now, next);
    // the last tile, and those that a row does not see all of: never many
    for (;;) {
      tile<false, false>(t0, row, now, next);
      t0 += kStep;
      if (t0 >= end) break;
      now = rows_of(t0, n);
      load_k(now);
      load_v(now);
    }
    att_settle();
    float none = 0.f;
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int i = 0; i < kNi; ++i)
#pragma unroll
        for (int d = 0; d < kW; ++d)
#pragma unroll
          for (int t = 0; t < 4; ++t) none = __builtin_fmaf(acc[r][i][d][t], 0.f, none);
    if (__any(none != 0.f)) {  // NaN: something was not finite
      clear();
      low = kCare;
      for (t0 = t_first; t0 < end; t0 += kStep) {
        now = rows_of(t0, n);
        load_k(now);
        load_v(now);
        tile<false, true>(t0, row, now, now);
      }
    }
#pragma unroll
    for (int r = 0; r < RB; ++r) l[r] = across(l[r], [](float a, float b) { return a + b; });
  }
};

// What a part of a row's tokens weighs against the row's maximum; a part that saw nothing (or scores of -inf
// alone) weighs nothing, whatever its values: 0 x NaN stays NaN.
__device__ __forceinline__ float att_share(float m, float top) {
  return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
}

// Columns col .. col + 3 of query row `row` of key / value head h: zeros where it saw nothing, NaN for counts that cannot be
template <class DT>
__device__ __forceinline__ void att_row_out(const CacheAttendParams& p, int b, int h, int row, int col, int n, sw_f4 o) {
  const int t = div_by(row, p.by_group), hq = h * p.group + row - t * p.group, Dh = p.c.head_dim;
  const bool seen = n > 0 && (!p.c.fresh || t < p.c.fresh[b]);
  typename DT::S* out = (typename DT::S*)p.out + ((b * (int64_t)p.tokens + t) * p.q_heads + hq) * Dh + col;
  float x[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = n < 0 ? __builtin_nanf("") : seen ? o[e] : 0.f;
  if (Dh % 4 == 0) {
    if (col < Dh) store_vec<DT, 4>(out, x);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < Dh) DT::store1(out + e, x[e]);
  }
}

// One token's weight: w_j <- decay w_j + got
struct OldWeight {
  float* at;  // null: no page
  float w;    // (decay 0 reads none)
};
__device__ __forceinline__ OldWeight old_weight(const CacheAttendParams& p, int b, int h, int j) {
  const int at = div_by(j, p.c.by_page), page = p.c.table[b * p.c.table_stride + at];
  if ((unsigned)page >= (unsigned)p.c.pages) return OldWeight{nullptr, 0.f};
  float* w = p.c.w + page * p.c.w_page_stride + h * p.c.w_head_stride + (j - at * p.c.page_size);
  return OldWeight{w, p.decay == 0.f ? 0.f : *w};
}
__device__ __forceinline__ void add_weight(const CacheAttendParams& p, const OldWeight& old, float got) {
  if (old.at) *old.at = p.decay == 0.f ? got : p.decay * old.w + got;
}

// By the workgroup that has all of the head's queries and tokens, from the scores that it has stored.
__device__ __forceinline__ void add_own_weights(const CacheAttendParams& p, int b, int h, int rows, int n, const float* lse) {
  const float* x = p.logits + (b * (int64_t)p.q_heads + h * p.group) * p.logit_stride;
  for (int j = threadIdx.x; j < n; j += kAttWaves * kWave) {
    const OldWeight old = old_weight(p, b, h, j);
    float sum = 0.f;
    for (int r = 0; r < rows; ++r) sum += __builtin_amdgcn_exp2f(x[r * p.logit_stride + j] - lse[r]);
    add_weight(p, old, sum);
  }
}

template <class DT, int HD, int VB, bool PAGE16, int RB>
__global__ __launch_bounds__(kAttWaves* kWave, HD == 256 || RB * HD > 128 ? 1 : 2) void cache_attend_kernel(CacheAttendParams p) {
  using A = Att<DT, HD, VB, PAGE16, RB>;
  using S = typename DT::S;
  constexpr int kRows = 16 * RB;
  __shared__ float so[kAttWaves][16][A::kPitch];  // a block of rows after the other
  __shared__ float sm[kAttWaves][kRows], sl[kAttWaves][kRows];
  __shared__ float lse[kRows];
  A a(p);
  const int Dh = p.c.head_dim, segs = p.c.kv_heads * p.blocks;
  // neighbouring workgroups run on different XCDs; those of one XCD take neighbouring units
  const int grid = gridDim.x;
  const int w = grid % 8 ? (int)blockIdx.x : (int)(blockIdx.x % 8 * (grid / 8) + blockIdx.x / 8);
  int x = 0, x1 = 1, b_start = 0, b_end = 0, units = 1;
  Chunk seqs;
  Seq seq;
  if (p.direct) {  // segment w
    a.b = div_by(w, p.by_segs);
    b_start = a.b * segs - w;
    b_end = 1;
    seq = seq_of(p, a.b);
  } else {
    const Deal d = deal(p, segs, p.wgs, p.by_wgs, seqs);
    x = deal_start(d, w);
    x1 = deal_start(d, w + 1);
  }
  while (x < x1) {
    if (x >= b_end) {
      find_unit(p, segs, x, seqs, &a.b, &seq, &b_start, &units);
      b_end = b_start + segs * units;
    }
    const int seg = (x - b_start) / units, u0 = x - b_start - seg * units, u1 = min(units, u0 + x1 - x);
    x += u1 - u0;
    a.h = div_by(seg, p.by_blocks);
    const int row0 = (seg - a.h * p.blocks) * kRows, rows = min(kRows, p.rows - row0);
    const bool whole = u0 == 0 && u1 == units;
    a.piece(row0, rows, u0 * kAttUnit, p.direct ? p.c.room : u1 * kAttUnit, seq, so);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      if (RB > 1 && rb * 16 >= rows) break;
      if (a.n > 0 && rb * 16 + a.c < rows) {
        if (a.g == 0) {
          sm[a.wave][rb * 16 + a.c] = a.m[rb] == -INFINITY ? a.m[rb] : a.base_of(a.m[rb]);
          sl[a.wave][rb * 16 + a.c] = a.l[rb];
        }
#pragma unroll
        for (int i = 0; i < A::kNi; ++i)
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < A::kW; e += 4)
              *(sw_f4*)&so[a.wave][a.c][(i * 16 + a.g * 4 + t) * A::kW + e] =
                  sw_f4{a.acc[rb][i][e][t], a.acc[rb][i][e + 1][t], a.acc[rb][i][e + 2][t], a.acc[rb][i][e + 3][t]};
      }
      __syncthreads();
      for (int at = threadIdx.x; at < min(16, rows - rb * 16) * (HD / 4); at += kAttWaves * kWave) {
        const int in = at / (HD / 4), r = rb * 16 + in, col = at % (HD / 4) * 4;
        float top = -INFINITY, l = 0.f;
        sw_f4 o = {0.f, 0.f, 0.f, 0.f};
        if (a.n > 0) {
#pragma unroll
          for (int i = 0; i < kAttWaves; ++i) top = fmaxf(top, sm[i][r]);
#pragma unroll
          for (int i = 0; i < kAttWaves; ++i) l += att_share(sm[i][r], top) * sl[i][r];
          // (shares of the whole sum first: sums of the largest values would not be finite)
          const float inv = l == 0.f && !whole ? 0.f : 1.f / l;  // (a piece that a row sees nothing of)
#pragma unroll
          for (int i = 0; i < kAttWaves; ++i) o += att_share(sm[i][r], top) * inv * *(const sw_f4*)&so[i][in][col];
        }
        if (whole) {
          att_row_out<DT>(p, a.b, a.h, row0 + r, col, a.n, o);
          if (p.own_weights) {
            if (col == 0) lse[r] = top + log2f(l);
          } else if (p.row_ml && col == 0) {
            float* ml = p.row_ml + (a.b * (int64_t)p.q_heads + a.h * p.group + row0 + r) * 2;
            ml[0] = top;
            ml[1] = l;
          }
        } else {
          const int64_t slot = 2 * w + (u0 == 0 ? 1 : 0);
          *(sw_f4*)(p.part + (slot * kRows + r) * HD + col) = o;
          if (col == 0) {
            p.part_ml[(slot * kRows + r) * 2] = top;
            p.part_ml[(slot * kRows + r) * 2 + 1] = l;
          }
        }
      }
      __syncthreads();
    }
    if (p.own_weights) add_own_weights(p, a.b, a.h, rows, a.n, lse);
  }
}

// The workgroups that have a segment of sequence b: w0 .. w1, none if it has no units.
struct Pieces {
  int w0, w1;
};
// first: the segment's first unit
__device__ __forceinline__ Pieces pieces_of(const CacheAttendParams& p, const Deal& d, int first, int units) {
  if (p.direct) return Pieces{0, 0};
  return Pieces{deal_of(d, first), deal_of(d, first + units - 1)};
}
__device__ __forceinline__ int64_t piece_row(const CacheAttendParams& p, const Pieces& s, int w, int row) {
  return ((int64_t)(2 * w + (w == s.w0 ? 1 : 0)) << p.row_bits) + (row & ((1 << p.row_bits) - 1));
}

// A head's pieces joined; zeros for rows that see nothing, NaN for counts that cannot be.  A workgroup's threads take
// four columns of a row each, and a share of its pieces.
template <class DT, int HD>
__device__ __forceinline__ void join_row(const CacheAttendParams& p, int at, const Deal& d, Chunk& seqs) {
  __shared__ float sm[256], sl[256];
  __shared__ sw_f4 so[256];
  const int row = at % p.rows, bh = at / p.rows, b = bh / p.c.kv_heads, h = bh - b * p.c.kv_heads;
  const int segs = p.c.kv_heads * p.blocks;
  if (b < seqs.b0 || b >= seqs.b0 + kWave) {
    seqs.load(p, 0, 0);
    while (b >= seqs.b0 + kWave) seqs.load(p, seqs.b0 + kWave, seqs.last());
  }
  const int n = __builtin_amdgcn_readlane(seqs.n, b - seqs.b0), units = units_of(n);
  Pieces s{0, -1};
  if (units)
    s = pieces_of(p, d, (__builtin_amdgcn_readlane(seqs.upto, b - seqs.b0) - units) * segs +
                            (h * p.blocks + (row >> p.row_bits)) * units, units);
  if (s.w0 == s.w1) return;  // one workgroup had all of it
  constexpr int kItems = HD / 4, kShares = 256 / kItems, kBatch = 4;
  const int item = threadIdx.x % kItems, share = threadIdx.x / kItems, col = item * 4;
  float top = -INFINITY, l = 0.f;
  sw_f4 o = {0.f, 0.f, 0.f, 0.f};
  for (int w = s.w0 + share; w <= s.w1; w += kShares * kBatch) {
    float m[kBatch], part[kBatch];
    sw_f4 x[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t r = piece_row(p, s, min(w + i * kShares, s.w1), row);
      m[i] = p.part_ml[r * 2];
      part[i] = p.part_ml[r * 2 + 1];
      x[i] = *(const sw_f4*)(p.part + r * HD + col);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (w + i * kShares > s.w1) break;
      const float to = fmaxf(top, m[i]), f = att_share(top, to) * l, g = att_share(m[i], to) * part[i];
      l = f + g;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      o = f * inv * o + g * inv * x[i];
      top = to;
    }
  }
  sm[threadIdx.x] = top;
  sl[threadIdx.x] = l;
  so[threadIdx.x] = o;
  __syncthreads();
  if (share) return;
  float all = top;
#pragma unroll
  for (int i = 1; i < kShares; ++i) all = fmaxf(all, sm[i * kItems + item]);
  float f[kShares], sum = 0.f;
#pragma unroll
  for (int i = 0; i < kShares; ++i) {
    f[i] = att_share(sm[i * kItems + item], all) * sl[i * kItems + item];
    sum += f[i];
  }
  const float inv = 1.f / sum;
  o = sw_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kShares; ++i) o += f[i] * inv * so[i * kItems + item];
  att_row_out<DT>(p, b, h, row, col, n, o);
}

// What each cached token received: with the scores x as attention left them (base-2 logarithms),
//   w_j <- decay w_j + sum over the head's queries of 2^(x_j - lse).
// 4 bytes a query and token are read, and the weights read and written: bound by the latency of its loads.  A wave takes
// a unit of tokens, two a lane, with no barrier; rows' lse come from their pieces again, beside the join, which would
// otherwise have to end first: a lane takes one piece of one row, as many rows at a time as lanes hold.
// (8 sequences of 4096 to 8191 tokens, 16 heads: 7 us; 9.6 with a workgroup a unit and a row's pieces over a wave.)
__device__ __forceinline__ void add_weights(const CacheAttendParams& p, int at) {
  constexpr int kEach = kAttUnit / kWave, kAhead = 4;  // tokens of a lane; rows whose scores are on their way together
  const int lane = threadIdx.x & (kWave - 1), segs = p.c.kv_heads, block = 1 << p.row_bits;
  Chunk seqs;
  Seq seq{0, 0};
  const Deal d = deal(p, segs, p.weight_waves, p.by_weight_waves, seqs);
  const int x1 = deal_start(d, at + 1);
  Deal of;  // attention's
  of.total = d.total * p.blocks;
  of.per = p.direct ? 0 : div_by(of.total, p.by_wgs);
  of.more = of.total - of.per * p.wgs;
  int b = 0, b_start = 0, b_end = 0, units = 1;
  for (int x = deal_start(d, at); x < x1; ++x) {
    if (x >= b_end) {
      find_unit(p, segs, x, seqs, &b, &seq, &b_start, &units);
      b_end = b_start + segs * units;
    }
    const int h = (x - b_start) / units, j0 = (x - b_start - h * units) * kAttUnit + lane;
    const float* const scores = p.logits + (b * (int64_t)p.q_heads + h * p.group) * p.logit_stride + j0;
    const float* const row_ml = p.row_ml + (b * (int64_t)p.q_heads + h * p.group) * 2;
    OldWeight old[kEach];
    float sum[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      sum[e] = 0.f;
      old[e] = j0 + e * kWave < seq.n ? old_weight(p, b, h, j0 + e * kWave) : OldWeight{nullptr, 0.f};
    }
    for (int r0 = 0; r0 < p.group; r0 += block) {  // rows whose pieces are the same workgroups'
      const int rows = min(block, p.group - r0);
      const Pieces s = pieces_of(p, of, b_start * p.blocks + (h * p.blocks + (r0 >> p.row_bits)) * units, units);
      // lanes of a row, 2^bits: as many as it has pieces, if all rows find room
      const int pieces = s.w1 - s.w0 + 1;
      const int bits = pieces <= 1 ? 0 : min(32 - __clz(pieces - 1), max(0, rows > 1 ? 6 - (32 - __clz(rows - 1)) : 6));
      for (int q0 = 0; q0 < rows; q0 += kWave >> bits) {
        const int some = min(kWave >> bits, rows - q0), q = q0 + (lane >> bits);
        float first[kAhead][kEach];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
#pragma unroll
          for (int e = 0; e < kEach; ++e)
            first[i][e] = i < some && j0 + e * kWave < seq.n ? scores[(r0 + q0 + i) * p.logit_stride + e * kWave] : -INFINITY;
        float top = -INFINITY, l = 0.f;
        if (q < rows) {
          if (pieces <= 1) {
            top = row_ml[(r0 + q) * 2];
            l = row_ml[(r0 + q) * 2 + 1];
          } else {
            for (int w = s.w0 + (lane & ((1 << bits) - 1)); w <= s.w1; w += kAhead << bits) {
              float m[kAhead], part[kAhead];
#pragma unroll
              for (int i = 0; i < kAhead; ++i) {
                const int64_t at = piece_row(p, s, min(w + (i << bits), s.w1), r0 + q);
                m[i] = p.part_ml[at * 2];
                part[i] = p.part_ml[at * 2 + 1];
              }
#pragma unroll
              for (int i = 0; i < kAhead; ++i) {
                if (w + (i << bits) > s.w1) break;
                const float to = fmaxf(top, m[i]);
                l = att_share(top, to) * l + att_share(m[i], to) * part[i];
                top = to;
              }
            }
          }
        }
        float all = top;
        for (int o = 1; o < 1 << bits; o <<= 1) all = fmaxf(all, __shfl_xor(all, o, kWave));
        l *= att_share(top, all);
        for (int o = 1; o < 1 << bits; o <<= 1) l += __shfl_xor(l, o, kWave);
        const float lse = all + log2f(l);
        for (int i0 = 0; i0 < some; i0 += kAhead) {
          float next[kAhead][kEach];
#pragma unroll
          for (int i = 0; i < kAhead; ++i)
#pragma unroll
            for (int e = 0; e < kEach; ++e)
              next[i][e] = i0 + kAhead + i < some && j0 + e * kWave < seq.n
                               ? scores[(r0 + q0 + i0 + kAhead + i) * p.logit_stride + e * kWave] : -INFINITY;
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            if (i0 + i >= some) break;
            const float base = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lse), (i0 + i) << bits));
#pragma unroll
            for (int e = 0; e < kEach; ++e) sum[e] += __builtin_amdgcn_exp2f(first[i][e] - base);
          }
#pragma unroll
          for (int i = 0; i < kAhead; ++i)
#pragma unroll
            for (int e = 0; e < kEach; ++e) first[i][e] = next[i][e];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) add_weight(p, old[e], sum[e]);
  }
}

// Of many rows most were one workgroup's and have nothing to join (512 new tokens of 4 x 16 heads
// over 2000 to 4096, 32768 rows: 169 us with a workgroup each, 158 with 2048 or 1024 in all).
constexpr int kAttJoins = 2048;  // workgroups at most

// joins: workgroups that join rows, one after the other and those of a segment in many; those behind them add weights up
template <class DT, int HD>
__global__ __launch_bounds__(256) void cache_join_kernel(CacheAttendParams p, int joins) {
  if ((int)blockIdx.x < joins) {
    Chunk seqs;
    const Deal d = deal(p, p.c.kv_heads * p.blocks, p.wgs, p.by_wgs, seqs);
    const int rows = p.c.batch * p.c.kv_heads * p.rows;
    for (int at = blockIdx.x;;) {
      join_row<DT, HD>(p, at, d, seqs);
      at += joins;
      if (at >= rows) break;
      __syncthreads();
    }
  } else {
    add_weights(p, (blockIdx.x - joins) * (256 / kWave) + threadIdx.x / kWave);
  }
}

template <class DT, int HD>
hipError_t run_attend(const CacheAttendParams& p, hipStream_t st) {
  const int64_t segs = (int64_t)p.c.batch * p.c.kv_heads * p.blocks;
  const dim3 grid((unsigned)(p.direct ? segs : p.wgs)), wg(kAttWaves * kWave);
  if (p.row_bits == 5) cache_attend_kernel<DT, HD, 16, true, 2><<<grid, wg, 0, st>>>(p);
  else if (p.vb == 16 && p.page16) cache_attend_kernel<DT, HD, 16, true, 1><<<grid, wg, 0, st>>>(p);
  else if (p.vb == 16) cache_attend_kernel<DT, HD, 16, false, 1><<<grid, wg, 0, st>>>(p);
  else if (p.vb == 8) cache_attend_kernel<DT, HD, 8, false, 1><<<grid, wg, 0, st>>>(p);
  else if (p.vb == 4) cache_attend_kernel<DT, HD, 4, false, 1><<<grid, wg, 0, st>>>(p);
  else if constexpr (DT::kCode != 0) cache_attend_kernel<DT, HD, 2, false, 1><<<grid, wg, 0, st>>>(p);
  const hipError_t err = hipGetLastError();
  const int rows = p.direct ? 0 : p.c.batch * p.c.kv_heads * p.rows, joins = rows < kAttJoins ? rows : kAttJoins;
  if (err != hipSuccess || joins + p.weight_waves == 0) return err;
  cache_join_kernel<DT, HD><<<dim3((unsigned)(joins + p.weight_waves / (256 / kWave))), dim3(256), 0, st>>>(p, joins);
  return hipGetLastError();
}

template <class DT>
hipError_t run_attend_type(const CacheAttendParams& p, hipStream_t st) {
  if (p.tile == 64) return run_attend<DT, 64>(p, st);
  if (p.tile == 128) return run_attend<DT, 128>(p, st);
  return run_attend<DT, 256>(p, st);
}

#endif

}  // namespace attnres
