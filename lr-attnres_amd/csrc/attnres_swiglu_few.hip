// Gated feed-forward projections of a few tokens (generation): h = (x Wu^T) silu(x Wg^T)
// for up to 64 rows of x.  Bound by reading the weight once.
//
// Layout.  A workgroup forms 8 hidden columns: 8 up and 8 gate rows are the 16 rows of
// one MFMA tile (16 x 16, 64 bytes of k a step), the tokens its columns, 16 a tile.
// Its four waves split k into runs of whole 128-byte lines; weight and x go from
// memory straight to registers, several steps of loads in flight a wave, and the
// four sums meet in LDS, where u and z of an element come together.  So F / 8
// workgroups x 4 waves read the weight at once: with the tiles of the large product
// (64 hidden columns a workgroup) few of the CUs had anything to read.
//
// Measured (bf16, one MI355X): 1 token, dim 768, hidden 2048: 4.5 us (1.4 TB/s; of it a
// launch and one trip to memory; the tiled product: 5.8); dim 2048, hidden 4096: 7.5 us
// (4.5 TB/s; 14.8).  64 tokens, dim 1024, hidden 4096: 9.0 us (10.6): there every
// workgroup's copy of x from the L2 caches is most of what it reads.
#include "attnres_swiglu.h"

namespace attnres {

namespace {

constexpr int kCus = 256;

// TT: tiles of 16 tokens; HT: MFMA tiles of 16 weight rows, for 8 HT hidden columns
template <class DT, int TT, int HT>
__global__ __launch_bounds__(256) void swiglu_few_kernel(SwGemmParams p) {
  using S = typename DT::S;
  using E = SwElem<DT>;
  constexpr int U = 8;  // steps whose loads are in flight together
  constexpr int kHidden = 8 * HT, kPitch = 16 * HT + 4;
  __shared__ __align__(16) float sums[4][TT][16][kPitch];  // [wave][tile][token][row]: up rows, gate rows, padding
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int f0 = blockIdx.x * kHidden;
  const int r = lane & 15, c = lane >> 4;
  const S* w[HT];
#pragma unroll
  for (int h = 0; h < HT; ++h) {
    const int row = h * 16 + r, f = min(f0 + row % kHidden, p.F - 1);
    w[h] = (const S*)p.p + (int64_t)(row / kHidden * p.F + f) * p.p_stride + c * E::kPer;
  }
  const S* x[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) x[t] = (const S*)p.q + (int64_t)min(t * 16 + r, p.M - 1) * p.q_stride + c * E::kPer;

  const int steps = (p.K + E::kStep - 1) / E::kStep;
  const int per = (steps + 7) / 8 * 2;  // of a wave: whole pairs, 128 bytes of a row
  const int s0 = wave * per, s1 = min(s0 + per, steps);
  sw_f4 acc[TT][HT];
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int h = 0; h < HT; ++h) acc[t][h] = sw_f4{0.f, 0.f, 0.f, 0.f};
  for (int s = s0; s < s1; s += U) {
    u32x4 a[U][HT], b[U][TT];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int k = (s + i) * E::kStep;
      const bool in = s + i < s1 && k + c * E::kPer < p.K;  // (p.K is a whole number of chunks)
#pragma unroll
      for (int h = 0; h < HT; ++h) a[i][h] = in ? *(const u32x4*)(w[h] + k) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < TT; ++t) b[i][t] = in ? *(const u32x4*)(x[t] + k) : u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int h = 0; h < HT; ++h) sw_mfma<DT>(a[i][h], b[i][t], acc[t][h]);
  }
  // lane: token r of a tile, rows 4 c .. 4 c + 3
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int h = 0; h < HT; ++h) *(sw_f4*)&sums[wave][t][r][16 * h + 4 * c] = acc[t][h];
  __syncthreads();

  // a thread: four hidden columns of one token
  const int tok = threadIdx.x / (2 * HT), q = threadIdx.x % (2 * HT), n0 = f0 + 4 * q;
  if (tok >= TT * 16 || tok >= p.M || n0 >= p.F) return;
  sw_f4 u = {0.f, 0.f, 0.f, 0.f}, z = u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u += *(const sw_f4*)&sums[i][tok >> 4][tok & 15][4 * q];
    z += *(const sw_f4*)&sums[i][tok >> 4][tok & 15][kHidden + 4 * q];
  }
  float h[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (DT::kCode == 0) h[e] = u[e] * (z[e] / (1.f + expf(-z[e])));
    else h[e] = u[e] * (z[e] * __builtin_amdgcn_rcpf(1.f + __expf(-z[e])));
  }
  S* out = (S*)p.out + (int64_t)tok * p.out_stride + n0;
  if (p.out_vec) {
    store_vec<DT, 4>(out, h);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n0 + e < p.F) DT::store1(out + e, h[e]);
  }
  if (!p.saved) return;
  // (whole groups of four: the planes' rows are padded)
  using P = SwPlanes<DT>;
  const SwPlaneAddress to = sw_planes<DT>(p.saved, p.n_tok, p.Fp);
  const int64_t at = ((int64_t)(n0 / E::kStep) * p.n_tok + tok) * E::kStep + n0 % E::kStep;
  if constexpr (P::kLow == 0) {
    *(sw_f4*)((float*)to.u + at) = u;
    *(sw_f4*)((float*)to.z + at) = z;
  } else {
    uint32_t uw[4], zw[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uw[e] = sw_round_bits<P::kLow>(u[e]);
      zw[e] = sw_round_bits<P::kLow>(z[e]);
    }
    *(u32x2*)((uint16_t*)to.u + at) = u32x2{hi_pair(uw[0], uw[1]), hi_pair(uw[2], uw[3])};
    *(u32x2*)((uint16_t*)to.z + at) = u32x2{hi_pair(zw[0], zw[1]), hi_pair(zw[2], zw[3])};
    sw_store_low<P::kLow>(to.low, at, uw, zw);
  }
}

template <class DT, int HT>
hipError_t run_few(const SwGemmParams& p, hipStream_t st) {
  const dim3 grid((unsigned)((p.F + 8 * HT - 1) / (8 * HT))), block(256);
  if (p.M <= 16) swiglu_few_kernel<DT, 1, HT><<<grid, block, 0, st>>>(p);
  else if (p.M <= 32) swiglu_few_kernel<DT, 2, HT><<<grid, block, 0, st>>>(p);
  else if (p.M <= 48) swiglu_few_kernel<DT, 3, HT><<<grid, block, 0, st>>>(p);
  else if (p.M <= 64) swiglu_few_kernel<DT, 4, HT><<<grid, block, 0, st>>>(p);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}
template <class DT>
hipError_t pick_few(const SwGemmParams& p, hipStream_t st) {
  // Each workgroup reads all of x, so with many of them 16 hidden columns each: 40
  // tokens, dim 1024, hidden 4096, bf16 7.5 us against 9.4 (1 token: 5.2 both ways);
  // hidden 2048, dim 768: 5.6 against 4.9.
  return p.M > 8 && p.F > 8 * kCus ? run_few<DT, 2>(p, st) : run_few<DT, 1>(p, st);
}

}  // namespace

hipError_t launch_swiglu_few(int dtype, const SwGemmParams& p, hipStream_t st) {
  if (dtype == F32::kCode) return pick_few<F32>(p, st);
  return dtype == BF16::kCode ? pick_few<BF16>(p, st) : pick_few<F16>(p, st);
}

}  // namespace attnres
