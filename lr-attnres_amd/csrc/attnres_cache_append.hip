// Heads of new tokens into the paged cache: per-head rms-norm and rotary positions
// of a fused query / key / value projection (as attnres_qkv_rotary.hip, the same
// arithmetic), with each key and value written where the cache keeps it.
//   n = x / sqrt(<x, x> / Dh + eps)        y = R(p) n   (pairs (2i, 2i+1) turned)
//
// Bound by memory for prompts (each value read once and written once, rotated keys
// once more where the caller wants them for attention inside the prompt): 8 prompts of up to 2048 tokens, 24 + 24 heads
// of 64 in all, bf16, 166 MB in 36 us (4.6 TB/s).  Single tokens are bound by the latency of a launch and
// the chain count -> block table -> store, 3.5 us; the projection's loads do not wait for it.
//
// Layout.  As the projection's kernel: LANES lanes a head, vectors of VEC consecutive values (16
// bytes where rows allow) a lane, up to kGroups head groups a wave.  A row of a page is as long as a head, so
// stores are whole rows whatever the pages' order.
#include "attnres_cache.h"
#include "attnres_rotary.h"

namespace attnres {

namespace {

// Head groups of a wave, all loads of them in flight at once: 48 heads of 64 are one wave's (8 prompts of up to 2048: 40.7
// us in two waves of three groups, 38.1 in one of six).
constexpr int kGroups = 6;
constexpr int kFewWaves = 4096;  // half of what the CUs hold

struct Place {  // of one new token
  int64_t row;  // its elements in a page, head 0; -1: not written
  int64_t w;    // its weight's
  int64_t at;   // table row, -1: outside
  bool real;    // one of its sequence's
};

__device__ __forceinline__ Place place_of(const CacheAppendParams& p, int b, int t) {
  Place r{-1, 0, -1, !p.c.fresh || t < p.c.fresh[b]};
  const int have = p.c.cached[b];
  const int64_t j = (int64_t)have + t, at = (int64_t)(p.pos ? p.pos[b] : have) + t;
  if (at >= 0 && at < p.table_rows) r.at = at;
  if (r.real && have >= 0 && j < p.c.room) {
    const int i = div_by((int)j, p.c.by_page), slot = (int)j - i * p.c.page_size;
    const int page = p.c.table[b * p.c.table_stride + i];
    if ((unsigned)page < (unsigned)p.c.pages) {
      r.row = page * p.c.page_stride + slot * p.c.slot_stride;
      r.w = page * p.c.w_page_stride + slot;
    }
  }
  return r;
}

// A lane holds CHUNKS vectors of a head, LANES * VEC apart.
template <class DT, class TT, int VEC, int LANES, int CHUNKS>
__global__ __launch_bounds__(kRotWaves* kWave) void cache_append_kernel(CacheAppendParams p, int groups, int iters,
                                                                          FastDiv by_groups) {
  using S = typename DT::S;
  using TS = typename TT::S;
  constexpr int kHeads = kWave / LANES;  // heads of a group
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t wave_at = rot_wave();  // (a grid of two dimensions ends behind 2^31 waves)
  if (wave_at >= (int64_t)p.n_tok * groups) return;
  const int wid = (int)wave_at, tok = div_by(wid, by_groups);
  const int part = wid - tok * groups;
  const int b = div_by(tok, p.by_tokens), t = tok - b * p.tokens;
  const int n_rot = p.q_heads + p.c.kv_heads, n_all = n_rot + p.c.kv_heads;
  const int Dh = p.c.head_dim;
  const int col0 = (lane & (LANES - 1)) * VEC;
  const int head0 = part * (iters * kHeads) + lane / LANES;
  bool in[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) in[c] = col0 + c * LANES * VEC < Dh;

  const S* src = (const S*)p.qkv + b * p.b_stride + t * p.t_stride;
  const bool real = !p.c.fresh || t < p.c.fresh[b];  // (what is behind a sequence's tokens is not read)
  Raw<DT, VEC> x[kGroups][CHUNKS];
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int h = i < iters && real ? head0 + i * kHeads : n_all;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if (h < n_all && in[c]) load_raw<DT, VEC, true>(src + (int64_t)h * Dh + col0 + c * LANES * VEC, x[i][c]);
      else x[i][c] = {};
    }
  }
  const Place at = place_of(p, b, t);
  float sn[CHUNKS][VEC / 2], cs[CHUNKS][VEC / 2];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    if (at.at >= 0 && in[c]) {
      const int64_t o = at.at * p.table_stride + (col0 + c * LANES * VEC) / 2;
      load_vec<TT, VEC / 2>((const TS*)p.sin + o, sn[c]);
      load_vec<TT, VEC / 2>((const TS*)p.cos + o, cs[c]);
    } else {  // NaN outside the tables, so that the token shows it
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) sn[c][e] = cs[c][e] = __builtin_nanf("");
    }
  }
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    if (i >= iters) break;
    const int h = head0 + i * kHeads;
    float v[CHUNKS][VEC];
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      unpack<DT, VEC>(x[i][c], v[c]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) ss += v[c][e] * v[c][e];
    }
    const float inv = p.qk_norm ? 1.f / sqrtf(group_sum(ss, LANES) / (float)Dh + p.eps) : 1.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      float r[VEC];
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) {
        const float even = v[c][2 * e] * inv, odd = v[c][2 * e + 1] * inv;
        r[2 * e] = at.real ? cs[c][e] * even - sn[c][e] * odd : 0.f;
        r[2 * e + 1] = at.real ? sn[c][e] * even + cs[c][e] * odd : 0.f;
      }
      if (h >= n_all || !in[c]) continue;
      const int col = col0 + c * LANES * VEC;
      if (h < p.q_heads) {
        store_vec<DT, VEC>((S*)p.q + ((b * (int64_t)p.q_heads + h) * p.tokens + t) * Dh + col, r);
      } else if (h < n_rot) {
        const int hh = h - p.q_heads;
        if (p.k) store_vec<DT, VEC>((S*)p.k + ((b * (int64_t)p.c.kv_heads + hh) * p.tokens + t) * Dh + col, r);
        if (at.row >= 0) {
          store_vec<DT, VEC>((S*)p.c.k + at.row + hh * p.c.head_stride + col, r);
          if (p.c.w && col == 0) p.c.w[at.w + hh * p.c.w_head_stride] = 0.f;
        }
      } else if (at.row >= 0) {  // a value, bit for bit
        store_raw<DT, VEC>((S*)p.c.v + at.row + (h - n_rot) * p.c.head_stride + col, x[i][c]);
      }
    }
  }
}

// Any alignment: one wave per head, its pairs in turn, the sum and the pairs in two passes over the row.  Single
// values: 49 x 180 tokens of 66 heads of 86, fp16, 269 us, where pairs in the vector kernel take 66 (and 88 columns, in eights, 48).
template <class DT, class TT>
__global__ __launch_bounds__(kRotWaves* kWave) void cache_append_general(CacheAppendParams p) {
  using S = typename DT::S;
  using TS = typename TT::S;
  const int lane = threadIdx.x & (kWave - 1);
  const int n_rot = p.q_heads + p.c.kv_heads, n_all = n_rot + p.c.kv_heads;
  const int64_t wave_at = rot_wave();  // (a grid of two dimensions ends behind 2^31 waves)
  if (wave_at >= (int64_t)p.n_tok * n_all) return;
  const int wid = (int)wave_at, tok = wid / n_all;
  const int h = wid - tok * n_all;
  const int b = div_by(tok, p.by_tokens), t = tok - b * p.tokens;
  const int Dh = p.c.head_dim;
  const S* x = (const S*)p.qkv + b * p.b_stride + t * p.t_stride + (int64_t)h * Dh;
  const Place at = place_of(p, b, t);
  if (h >= n_rot) {
    if (at.row < 0) return;
    S* dst = (S*)p.c.v + at.row + (h - n_rot) * p.c.head_stride;
    for (int i = lane; i < Dh; i += kWave) dst[i] = x[i];
    return;
  }
  float inv = 1.f;
  if (p.qk_norm) {
    float ss = 0.f;
    for (int i = lane; i < Dh; i += kWave) {
      const float f = DT::load1(x + i);
      ss += f * f;
    }
    inv = 1.f / sqrtf(wave_sum(ss) / (float)Dh + p.eps);
  }
  const int hh = h - p.q_heads;
  S* const dense = hh < 0 ? (S*)p.q + ((b * (int64_t)p.q_heads + h) * p.tokens + t) * Dh
                   : p.k ? (S*)p.k + ((b * (int64_t)p.c.kv_heads + hh) * p.tokens + t) * Dh
                         : nullptr;
  S* const row = hh >= 0 && at.row >= 0 ? (S*)p.c.k + at.row + hh * p.c.head_stride : nullptr;
  for (int i = lane; i < Dh / 2; i += kWave) {
    const float s = at.at < 0 ? __builtin_nanf("") : TT::load1((const TS*)p.sin + at.at * p.table_stride + i);
    const float c = at.at < 0 ? __builtin_nanf("") : TT::load1((const TS*)p.cos + at.at * p.table_stride + i);
    const float even = DT::load1(x + 2 * i) * inv, odd = DT::load1(x + 2 * i + 1) * inv;
    const float lo = at.real ? c * even - s * odd : 0.f, hi = at.real ? s * even + c * odd : 0.f;
    if (dense) {
      DT::store1(dense + 2 * i, lo);
      DT::store1(dense + 2 * i + 1, hi);
    }
    if (row) {
      DT::store1(row + 2 * i, lo);
      DT::store1(row + 2 * i + 1, hi);
    }
  }
  if (row && p.c.w && lane == 0) p.c.w[at.w + hh * p.c.w_head_stride] = 0.f;
}

template <class DT, class TT, int VEC, int LANES, int CHUNKS = 1>
hipError_t run(const CacheAppendParams& p, hipStream_t st) {
  const int n_all = p.q_heads + 2 * p.c.kv_heads;
  const int all = (n_all + kWave / LANES - 1) / (kWave / LANES);
  // head groups shared evenly by as few waves as hold them; few tokens, whose launch is all latency, take a wave a
  // group (16 tokens of 36 heads of 64: 7.3 us a call, 8.2 with five groups in turn)
  const int most = (int64_t)p.n_tok * all <= kFewWaves ? 1 : kGroups;
  const int groups = (all + most - 1) / most, iters = (all + groups - 1) / groups;
  dim3 grid;
  if (!rot_grid((int64_t)p.n_tok * groups, &grid)) return hipErrorInvalidValue;
  cache_append_kernel<DT, TT, VEC, LANES, CHUNKS><<<grid, dim3(kRotWaves * kWave), 0, st>>>(p, groups, iters, fast_div(groups));
  return hipGetLastError();
}

template <class DT, class TT>
hipError_t pick(const CacheAppendParams& p, int vec, int lanes, hipStream_t st) {
  if constexpr (DT::kCode != 0) {
    if (vec == 8) {
      if (lanes == 4) return run<DT, TT, 8, 4>(p, st);
      if (lanes == 8) return run<DT, TT, 8, 8>(p, st);
      if (lanes == 16) return run<DT, TT, 8, 16>(p, st);
      if (lanes == 32) return run<DT, TT, 8, 32>(p, st);
    }
  }
  // Narrower vectors: 16 lanes a head, several vectors each, keep four heads' loads on their way in a group (us, 16 lanes / one
  // vector a lane: 9 x 209 tokens of 45 heads of 148, 16 bits, 19.1 / 24.3; of 32 heads of 128 in fp32 12.7 / 13.7; 49 x 180 of 66
  // heads of 86 66 / 95; but 9 x 400 of 24 heads of 252 25 / 23.  8 lanes were slower from 100 on; with eights, two vectors a
  // lane 45 / 43.5 for 8 x 2048 tokens of 24 heads of 128.)
  if (vec == 4) {
    if (lanes == 8) return run<DT, TT, 4, 8>(p, st);
    if (lanes == 16) return run<DT, TT, 4, 16>(p, st);
    if (lanes == 32) return run<DT, TT, 4, 16, 2>(p, st);
    if (lanes == 64) return run<DT, TT, 4, 16, 4>(p, st);
  }
  if (vec == 2) {
    if (lanes == 32) return run<DT, TT, 2, 16, 2>(p, st);
    if (lanes == 64) return run<DT, TT, 2, 16, 4>(p, st);
    if (lanes == 128) return run<DT, TT, 2, 16, 8>(p, st);
  }
  if (vec != 1) return hipErrorInvalidValue;
  dim3 grid;
  if (!rot_grid((int64_t)p.n_tok * (p.q_heads + 2 * p.c.kv_heads), &grid)) return hipErrorInvalidValue;
  cache_append_general<DT, TT><<<grid, dim3(kRotWaves * kWave), 0, st>>>(p);
  return hipGetLastError();
}

template <class DT>
hipError_t pick_table(bool f32_table, const CacheAppendParams& p, int vec, int lanes, hipStream_t st) {
  if constexpr (DT::kCode != 0) {
    if (!f32_table) return pick<DT, DT>(p, vec, lanes, st);
  }
  return pick<DT, F32>(p, vec, lanes, st);
}

}  // namespace

hipError_t launch_cache_append(int dtype, bool f32_table, const CacheAppendParams& p, int vec, int lanes, hipStream_t st) {
  if (dtype == F32::kCode) return pick_table<F32>(f32_table, p, vec, lanes, st);
  if (dtype == BF16::kCode) return pick_table<BF16>(f32_table, p, vec, lanes, st);
  return pick_table<F16>(f32_table, p, vec, lanes, st);
}

}  // namespace attnres
