// Heads of a fused query / key / value projection: per-head rms-norm and rotary
// positions in one pass, and its backward (MultiHeadAttention, model.py:430-569,
// with norm :28-31 and the rotation :291-313).
//   n = x / sqrt(<x, x> / Dh + eps)        y = R(p) n   (pairs (2i, 2i+1) turned)
//   g = R(p)^T dy                          dx = (g - n <g, n> / Dh) / rms
// The backward recomputes 1/rms from the projection's row, which it has to read
// anyway for n; nothing is saved but the forward's inputs.
//
// Bound by memory: the forward reads and writes (Hq + Hk) Dh values a token, the
// backward reads the raw queries and keys and the three upstream gradients and
// writes the whole projection's gradient (the values' part is a copy, so that no
// concatenation follows).  The values are not read in the forward at all.
//
// Layout.  A wave takes up to kIters groups of heads of one token: LANES lanes a
// head, VEC consecutive values (16 bytes) a lane, so a projection's row is read in
// whole lines, and a token's table row is loaded once for all of its heads.  A
// head's sum of squares is log2(LANES) DPP or shuffle steps.
//
// Measured (bf16, one MI355X, 16384 tokens): 12 heads of 64, forward 23 us and backward 47-49
// (4.4 and 4.1-4.3 TB/s of what each moves); 16 heads of 128, 53 and 98 us (5.1 and 5.5 TB/s; a
// non-temporal copy of 1 GiB reaches 6.5).  With head groups given to waves in whole fours, the last wave of a token
// short of work, the backward of 12 heads of 64 took 50.
#include "attnres_device.h"
#include "attnres_launch.h"
#include "attnres_rotary.h"
#include "attnres_sublayers.h"

namespace attnres {

namespace {

constexpr int kIters = 4;      // head groups of a wave, all loads of them in flight at once

// row of the tables for token (b, t); -1: outside
__device__ __forceinline__ int64_t rot_position(const QkvRotaryParams& p, int64_t b, int64_t t) {
  const int64_t at = p.pos ? p.pos[b * p.pos_b_stride + t * p.pos_t_stride] : p.start + t;
  return at >= 0 && at < p.table_rows ? at : -1;
}

// DT: values, TT: tables.  A lane holds CHUNKS vectors of a head, LANES * VEC apart.
template <class DT, class TT, int VEC, int LANES, int CHUNKS, bool BWD>
__global__ __launch_bounds__(kRotWaves* kWave) void qkv_rotary_kernel(QkvRotaryParams p, int groups, int iters) {
  using S = typename DT::S;
  using TS = typename TT::S;
  constexpr int kHeads = kWave / LANES;  // heads of a group
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t wid = rot_wave();
  const int64_t tok = wid / groups;
  if (tok >= p.n_tok) return;
  const int part = (int)(wid - tok * groups);
  const int64_t b = tok / p.tokens, t = tok - b * p.tokens;
  const int n_rot = p.q_heads + p.kv_heads, n_all = BWD ? n_rot + p.kv_heads : n_rot;
  const int Dh = p.head_dim;
  const int col = (lane & (LANES - 1)) * VEC;
  const int head0 = part * (iters * kHeads) + lane / LANES;
  bool in[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) in[c] = col + c * LANES * VEC < Dh;

  const S* src = (const S*)p.qkv + b * p.b_stride + t * p.t_stride;
  Raw<DT, VEC> x[kIters][CHUNKS], g[kIters][CHUNKS];
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    const int h = i < iters ? head0 + i * kHeads : n_all;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int at = col + c * LANES * VEC;
      if (h < n_rot && in[c]) load_raw<DT, VEC, true>(src + (int64_t)h * Dh + at, x[i][c]);
      else x[i][c] = {};
      if constexpr (BWD) {
        const int which = h < p.q_heads ? 0 : h < n_rot ? 1 : 2;
        const int hh = which == 0 ? h : which == 1 ? h - p.q_heads : h - n_rot;
        const S* gp = (const S*)(which == 0 ? p.grad[0] : which == 1 ? p.grad[1] : p.grad[2]);
        const int64_t bs = which == 0 ? p.grad_stride[0][0] : which == 1 ? p.grad_stride[1][0] : p.grad_stride[2][0];
        const int64_t hs = which == 0 ? p.grad_stride[0][1] : which == 1 ? p.grad_stride[1][1] : p.grad_stride[2][1];
        const int64_t ts = which == 0 ? p.grad_stride[0][2] : which == 1 ? p.grad_stride[1][2] : p.grad_stride[2][2];
        if (h < n_all && in[c] && gp) load_raw<DT, VEC, true>(gp + b * bs + hh * hs + t * ts + at, g[i][c]);
        else g[i][c] = {};
      }
    }
  }
  // a pair's sin and cos; NaN outside the table, so that the token shows it
  float sn[CHUNKS][VEC / 2], cs[CHUNKS][VEC / 2];
  const int64_t at = rot_position(p, b, t);
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int64_t o = at * p.table_stride + (col + c * LANES * VEC) / 2;
    if (at >= 0 && in[c]) {
      load_vec<TT, VEC / 2>((const TS*)p.sin + o, sn[c]);
      load_vec<TT, VEC / 2>((const TS*)p.cos + o, cs[c]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) sn[c][e] = cs[c][e] = __builtin_nanf("");
    }
  }
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
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
    float inv = 1.f;
    if (p.qk_norm) {
      ss = group_sum(ss, LANES);
      inv = 1.f / sqrtf(ss / (float)Dh + p.eps);
    }
    float r[CHUNKS][VEC];
    if constexpr (!BWD) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) {
          const float even = v[c][2 * e] * inv, odd = v[c][2 * e + 1] * inv;
          r[c][2 * e] = cs[c][e] * even - sn[c][e] * odd;
          r[c][2 * e + 1] = sn[c][e] * even + cs[c][e] * odd;
        }
      if (h >= n_rot) continue;
      const bool is_q = h < p.q_heads;
      const int hh = is_q ? h : h - p.q_heads, nh = is_q ? p.q_heads : p.kv_heads;
      S* dst = (S*)(is_q ? p.q : p.k) + ((b * nh + hh) * p.tokens + t) * Dh;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
        if (in[c]) store_vec<DT, VEC>(dst + col + c * LANES * VEC, r[c]);
    } else {
      float dot = 0.f;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        float gv[VEC];
        unpack<DT, VEC>(g[i][c], gv);
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) {
          r[c][2 * e] = cs[c][e] * gv[2 * e] + sn[c][e] * gv[2 * e + 1];
          r[c][2 * e + 1] = cs[c][e] * gv[2 * e + 1] - sn[c][e] * gv[2 * e];
          if (in[c]) dot += r[c][2 * e] * v[c][2 * e] + r[c][2 * e + 1] * v[c][2 * e + 1];
        }
      }
      if (p.qk_norm) {
        // x <g, x> / (Dh rms^3) = n <g, n> / (Dh rms)
        dot = group_sum(dot, LANES) * (inv * inv) / (float)Dh;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
          for (int e = 0; e < VEC; ++e) r[c][e] = inv * (r[c][e] - v[c][e] * dot);
      }
      if (h >= n_all) continue;
      S* dst = (S*)p.dqkv + (tok * n_all + h) * Dh;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        if (!in[c]) continue;
        if (h < n_rot) {
          store_vec<DT, VEC>(dst + col + c * LANES * VEC, r[c]);
        } else {  // the values' gradient, bit for bit
          store_raw<DT, VEC>(dst + col + c * LANES * VEC, g[i][c]);
        }
      }
    }
  }
}

// Any alignment and head width: one wave per head, its pairs in turn.  Two passes
// over the row (the sums, then the pairs), the second from the caches.  Bound by its
// accesses of single values: bf16, 16384 tokens, 4 heads of 512, 109 us forward and 241
// backward (2.8 and 2.4 TB/s), 8 heads of 258, 163 and 314 (1.8), where the vector kernels take
// 52 and 105 for 8 heads of 256.  Wider heads are not in use here, so they have no more.
template <class DT, class TT, bool BWD>
__global__ __launch_bounds__(kRotWaves* kWave) void qkv_rotary_general(QkvRotaryParams p) {
  using S = typename DT::S;
  using TS = typename TT::S;
  const int lane = threadIdx.x & (kWave - 1);
  const int n_rot = p.q_heads + p.kv_heads, n_all = BWD ? n_rot + p.kv_heads : n_rot;
  const int64_t wid = rot_wave();
  const int64_t tok = wid / n_all;
  if (tok >= p.n_tok) return;
  const int h = (int)(wid - tok * n_all);
  const int64_t b = tok / p.tokens, t = tok - b * p.tokens;
  const int Dh = p.head_dim, pairs = Dh / 2;
  const S* x = (const S*)p.qkv + b * p.b_stride + t * p.t_stride + (int64_t)h * Dh;
  const int which = h < p.q_heads ? 0 : h < n_rot ? 1 : 2;
  const int hh = which == 0 ? h : which == 1 ? h - p.q_heads : h - n_rot;
  const S* g = nullptr;
  if constexpr (BWD) {
    g = (const S*)(which == 0 ? p.grad[0] : which == 1 ? p.grad[1] : p.grad[2]);
    if (g)
      g += b * (which == 0 ? p.grad_stride[0][0] : which == 1 ? p.grad_stride[1][0] : p.grad_stride[2][0]) +
           hh * (which == 0 ? p.grad_stride[0][1] : which == 1 ? p.grad_stride[1][1] : p.grad_stride[2][1]) +
           t * (which == 0 ? p.grad_stride[0][2] : which == 1 ? p.grad_stride[1][2] : p.grad_stride[2][2]);
    if (which == 2) {
      S* dst = (S*)p.dqkv + (tok * n_all + h) * Dh;
      for (int i = lane; i < Dh; i += kWave) dst[i] = g ? g[i] : (S)0;
      return;
    }
  }
  const int64_t at = rot_position(p, b, t);
  const TS* sn = (const TS*)p.sin + (at < 0 ? 0 : at) * p.table_stride;
  const TS* cs = (const TS*)p.cos + (at < 0 ? 0 : at) * p.table_stride;
  const float nan = __builtin_nanf("");
  float ss = 0.f, dot = 0.f;
  for (int i = lane; i < pairs; i += kWave) {
    const float even = DT::load1(x + 2 * i), odd = DT::load1(x + 2 * i + 1);
    ss += even * even + odd * odd;
    if (BWD && g) {
      const float s = at < 0 ? nan : TT::load1(sn + i), c = at < 0 ? nan : TT::load1(cs + i);
      const float ge = DT::load1(g + 2 * i), go = DT::load1(g + 2 * i + 1);
      dot += (c * ge + s * go) * even + (c * go - s * ge) * odd;
    }
  }
  float inv = 1.f, k = 0.f;
  if (p.qk_norm) {
    inv = 1.f / sqrtf(wave_sum(ss) / (float)Dh + p.eps);
    if (BWD) k = wave_sum(dot) * (inv * inv) / (float)Dh;
  }
  S* dst = BWD ? (S*)p.dqkv + (tok * n_all + h) * Dh
               : (S*)(which == 0 ? p.q : p.k) + ((b * (which == 0 ? p.q_heads : p.kv_heads) + hh) * p.tokens + t) * Dh;
  for (int i = lane; i < pairs; i += kWave) {
    const float s = at < 0 ? nan : TT::load1(sn + i), c = at < 0 ? nan : TT::load1(cs + i);
    const float even = DT::load1(x + 2 * i), odd = DT::load1(x + 2 * i + 1);
    if constexpr (!BWD) {
      DT::store1(dst + 2 * i, c * (even * inv) - s * (odd * inv));
      DT::store1(dst + 2 * i + 1, s * (even * inv) + c * (odd * inv));
    } else {
      const float ge = g ? DT::load1(g + 2 * i) : 0.f, go = g ? DT::load1(g + 2 * i + 1) : 0.f;
      DT::store1(dst + 2 * i, inv * ((c * ge + s * go) - even * k));
      DT::store1(dst + 2 * i + 1, inv * ((c * go - s * ge) - odd * k));
    }
  }
}

template <class DT, class TT, bool BWD, int VEC, int LANES, int CHUNKS>
hipError_t run(const QkvRotaryParams& p, hipStream_t st) {
  const int n_all = p.q_heads + p.kv_heads * (BWD ? 2 : 1);
  // head groups shared evenly by as few waves as hold them (36 heads of 64: 3 + 2 groups, not 4 + 1)
  const int all = (n_all + kWave / LANES - 1) / (kWave / LANES);
  const int groups = (all + kIters - 1) / kIters, iters = (all + groups - 1) / groups;
  dim3 grid;
  if (!rot_grid(p.n_tok * groups, &grid)) return hipErrorInvalidValue;
  qkv_rotary_kernel<DT, TT, VEC, LANES, CHUNKS, BWD><<<grid, dim3(kRotWaves * kWave), 0, st>>>(p, groups, iters);
  return hipGetLastError();
}

template <class DT, class TT, bool BWD>
hipError_t run_general(const QkvRotaryParams& p, hipStream_t st) {
  dim3 grid;
  if (!rot_grid(p.n_tok * (p.q_heads + p.kv_heads * (BWD ? 2 : 1)), &grid)) return hipErrorInvalidValue;
  qkv_rotary_general<DT, TT, BWD><<<grid, dim3(kRotWaves * kWave), 0, st>>>(p);
  return hipGetLastError();
}

template <class DT, class TT, bool BWD>
hipError_t pick(const QkvRotaryParams& p, int vec, int lanes, int chunks, hipStream_t st) {
  if constexpr (DT::kCode != 0) {
    if (vec == 8) {
      if (lanes == 4) return run<DT, TT, BWD, 8, 4, 1>(p, st);
      if (lanes == 8) return run<DT, TT, BWD, 8, 8, 1>(p, st);
      if (lanes == 16) return run<DT, TT, BWD, 8, 16, 1>(p, st);
      if (lanes == 32) return run<DT, TT, BWD, 8, 32, 1>(p, st);
    }
  }
  if (vec == 4) {
    if (lanes == 8) return run<DT, TT, BWD, 4, 8, 1>(p, st);
    if (lanes == 16) return run<DT, TT, BWD, 4, 16, 1>(p, st);
    if (lanes == 32) return run<DT, TT, BWD, 4, 32, 1>(p, st);
    if (lanes == 64) return run<DT, TT, BWD, 4, 64, 1>(p, st);
  }
  if (vec == 2) {
    if (lanes == 32) return run<DT, TT, BWD, 2, 32, 1>(p, st);
    if (lanes == 64 && chunks == 1) return run<DT, TT, BWD, 2, 64, 1>(p, st);
    if (lanes == 64 && chunks == 2) return run<DT, TT, BWD, 2, 64, 2>(p, st);
  }
  if (vec == 1) return run_general<DT, TT, BWD>(p, st);
  return hipErrorInvalidValue;
}

template <class DT, bool BWD>
hipError_t pick_table(bool f32_table, const QkvRotaryParams& p, int vec, int lanes, int chunks, hipStream_t st) {
  if constexpr (DT::kCode != 0) {
    if (!f32_table) return pick<DT, DT, BWD>(p, vec, lanes, chunks, st);
  }
  return pick<DT, F32, BWD>(p, vec, lanes, chunks, st);
}

template <bool BWD>
hipError_t pick_type(int dtype, bool f32_table, const QkvRotaryParams& p, int vec, int lanes, int chunks,
                     hipStream_t st) {
  if (dtype == F32::kCode) return pick_table<F32, BWD>(f32_table, p, vec, lanes, chunks, st);
  if (dtype == BF16::kCode) return pick_table<BF16, BWD>(f32_table, p, vec, lanes, chunks, st);
  return pick_table<F16, BWD>(f32_table, p, vec, lanes, chunks, st);
}

}  // namespace

hipError_t launch_qkv_rotary(int dtype, bool f32_table, bool bwd, const QkvRotaryParams& p, int vec, int lanes,
                             int chunks, hipStream_t st) {
  return bwd ? pick_type<true>(dtype, f32_table, p, vec, lanes, chunks, st)
             : pick_type<false>(dtype, f32_table, p, vec, lanes, chunks, st);
}

}  // namespace attnres
