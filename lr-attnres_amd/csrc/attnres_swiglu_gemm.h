// The product's kernels: one instantiation per type, form and tile, and the sum of
// split products.  Included by attnres_swiglu_{bf16,f16,f32}.hip.
#pragma once

#include "attnres_swiglu.h"

namespace attnres {

static __device__ uint4 sw_zeros;  // what k beyond its end is loaded from

// u silu(z); 16-bit results need no more than the hardware's exp2 and reciprocal
template <class DT>
__device__ __forceinline__ float sw_silu(float z) {
  if constexpr (DT::kCode == 0) return z / (1.f + expf(-z));
  else return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
}

// Tiles in an order that keeps what the 32 CUs of one XCD work on at a time within
// few rows and columns: workgroup b runs on XCD b % 8, so each XCD gets a run of
// consecutive tiles, and runs go down kGroup tile rows before the next column.
__device__ __forceinline__ void sw_tile(const SwGemmParams& p, int b, int n, int* split, int* tm, int* tn, int* tile) {
  constexpr int kXcd = 8, kGroup = 8;
  const int q = n / kXcd, r = n % kXcd, x = b % kXcd;
  const int at = x * q + min(x, r) + b / kXcd;
  const int tiles = p.tiles_m * p.tiles_n;
  // (the quotients are computed in vector registers; what follows from them is scalar)
  *split = __builtin_amdgcn_readfirstlane(at / tiles);
  const int t = at - *split * tiles;
  const int per = kGroup * p.tiles_n, g = __builtin_amdgcn_readfirstlane(t / per), first = g * kGroup;
  const int rows = min(p.tiles_m - first, kGroup);
  *tn = __builtin_amdgcn_readfirstlane((t - g * per) / rows);
  *tm = first + (t - g * per) - *tn * rows;
  *tile = t;
}

// A wave's 32 x COLS values (m = lane % 32; v[j][4 i + e]: n = 32 j + 8 i + 4 (lane / 32)
// + e) to rows of memory through the wave's own LDS, 16 bytes a lane.  `row` gives
// the address of row m of the wave's columns or null.
template <class DT, int COLS, class Row>
__device__ __forceinline__ void sw_store_rows(char* lds, int lane, const float (&v)[COLS / 32][16], int n0, int n_end,
                                              bool vec, Row row) {
  using S = typename DT::S;
  constexpr int kSize = sizeof(S), kPitch = COLS * kSize + 16, kChunks = COLS * kSize / 16, kPer = 16 / kSize;
  char* mine = lds + (lane & 31) * kPitch;
#pragma unroll
  for (int j = 0; j < COLS / 32; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      char* at = mine + (j * 32 + 8 * i + 4 * (lane >> 5)) * kSize;
      if constexpr (kSize == 2) *(u32x2*)at = u32x2{pack2<DT>(v[j][4 * i], v[j][4 * i + 1]), pack2<DT>(v[j][4 * i + 2], v[j][4 * i + 3])};
      else *(sw_f4*)at = sw_f4{v[j][4 * i], v[j][4 * i + 1], v[j][4 * i + 2], v[j][4 * i + 3]};
    }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < 32 * kChunks / kWave; ++i) {
    const int q = i * kWave + lane, m = q / kChunks, c = q % kChunks;
    const u32x4 x = *(const u32x4*)(lds + m * kPitch + c * 16);
    S* dst = (S*)row(m);
    const int n = n0 + c * kPer;
    if (!dst || n >= n_end) continue;
    if (vec && n + kPer <= n_end) {
      *(u32x4*)(dst + c * kPer) = x;
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        if (n + e >= n_end) break;
        if constexpr (kSize == 2) dst[c * kPer + e] = (S)(x[e / 2] >> (16 * (e & 1)));
        else dst[c * kPer + e] = __uint_as_float(x[e]);
      }
    }
  }
  __builtin_amdgcn_wave_barrier();
}

// What becomes of a wave's 32 rows m0.. x COLS columns of the product (fwd: COLS is
// u and z together).  v holds the sums.
template <class DT, int FORM, int COLS>
__device__ __forceinline__ void sw_finish(const SwGemmParams& p, char* lds, int lane, int m0, int n0,
                                          float (&v)[COLS / 32][16]) {
  using S = typename DT::S;
  if constexpr (FORM == kFwd) {
    constexpr int H = COLS / 64;  // 32-column groups of u
    if (p.saved) {
      const int n_end = (p.n_out + 7) / 8 * 8;  // (whole vectors: the rows are padded)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float x[H][16];
#pragma unroll
        for (int j = 0; j < H; ++j)
#pragma unroll
          for (int i = 0; i < 16; ++i) x[j][i] = v[half * H + j][i];
        sw_store_rows<DT, H * 32>(lds, lane, x, n0, n_end, true, [&](int m) -> void* {
          return m0 + m < p.M ? (S*)p.saved + ((int64_t)half * p.M + m0 + m) * p.saved_stride + n0 : nullptr;
        });
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    float h[H][16];
#pragma unroll
    for (int j = 0; j < H; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) h[j][i] = v[j][i] * sw_silu<DT>(v[H + j][i]);
    sw_store_rows<DT, H * 32>(lds, lane, h, n0, p.n_out, p.out_vec, [&](int m) -> void* {
      return m0 + m < p.M ? (S*)p.out + (int64_t)(m0 + m) * p.out_stride + n0 : nullptr;
    });
  } else {
    sw_store_rows<DT, COLS>(lds, lane, v, n0, p.n_out, p.out_vec, [&](int m) -> void* {
      int r = m0 + m;
      if constexpr (FORM == kDw) {  // rows of the padded halves
        const int half = r >= p.Fp, f = r - half * p.Fp;
        if (half * p.Fp + f >= 2 * p.Fp || f >= p.F) return nullptr;
        r = half * p.F + f;
      } else {
        if (r >= p.M) return nullptr;
      }
      return (S*)p.out + (int64_t)r * p.out_stride + n0;
    });
  }
}

template <class DT, int FORM, int BM, int BN, bool SPLIT>
__global__ __launch_bounds__(256, BM * BN >= 256 * 256 ? 1 : 2) void swiglu_gemm_kernel(SwGemmParams p) {
  using E = SwElem<DT>;
  using OpP = SwOperand<DT, BN, FORM != kFwd>;
  using OpQ = SwOperand<DT, BM, FORM == kDw>;
  constexpr int NP = BN / 64, NQ = BM / 64;  // 32 x 32 tiles of a wave
  constexpr int kStage = OpP::kBytes + OpQ::kBytes;
  constexpr int kLoads = OpP::kLoads + OpQ::kLoads;
  constexpr int kCols = FORM == kFwd ? BN / 2 : BN;  // output columns of a tile
  constexpr int es = E::kSize;
  __shared__ __align__(1024) char lds[kSwStages * kStage];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  int split, tm, tn, tile;
  sw_tile(p, blockIdx.x, gridDim.x, &split, &tm, &tn, &tile);
  const int m0 = tm * BM, n0 = tn * kCols;
  const int all_steps = (p.K + E::kStep - 1) / E::kStep;
  const int first = SPLIT ? split * p.steps : 0;
  const int nk = SPLIT ? min(p.steps, all_steps - first) : all_steps;

  OpP op;
  OpQ oq;
#pragma unroll
  for (int i = 0; i < OpP::kLoads; ++i) {
    int r, c;
    OpP::place(i, tid, &r, &c);
    if constexpr (FORM == kFwd) {  // up and gate rows of the same hidden columns, per wave column
      const int w = r / (BN / 2), rr = r % (BN / 2), half = rr / (BN / 4);
      const int f = min(n0 + w * (BN / 4) + rr % (BN / 4), p.F - 1);
      op.off[i] = (uint32_t)((int64_t)(half * p.F + f) * p.p_stride * es) + c * 16;
      op.kr[i] = c * E::kPer;
    } else {
      op.off[i] = (uint32_t)((int64_t)r * p.p_stride * es) + (min(n0 + c * E::kPer, p.N - E::kPer) - n0) * es;
      op.kr[i] = r;
    }
  }
#pragma unroll
  for (int i = 0; i < OpQ::kLoads; ++i) {
    int r, c;
    OpQ::place(i, tid, &r, &c);
    if constexpr (FORM != kDw) {
      oq.off[i] = (uint32_t)((int64_t)(min(m0 + r, p.M - 1) - m0) * p.q_stride * es) + c * 16;
      oq.kr[i] = c * E::kPer;
    } else {
      oq.off[i] = (uint32_t)((int64_t)r * p.q_stride * es) + (min(m0 + c * E::kPer, p.M - E::kPer) - m0) * es;
      oq.kr[i] = r;
    }
  }
  op.place_reads(wn * (BN / 2), lane, 0);
  oq.place_reads(wm * (BM / 2), lane, OpP::kBytes);
  const uint32_t lds0 = lds_address(lds) + wave * 1024;

  // loads of step s (counted within the split) into its stage
  auto load = [&](int s) {
    const int k0 = (first + s) * E::kStep;
    const char *bp, *bq;
    int left;  // k's of this step that exist
    if constexpr (FORM == kFwd) {
      bp = (const char*)p.p + (int64_t)k0 * es;
      bq = (const char*)p.q + ((int64_t)m0 * p.q_stride + k0) * es;
      left = p.K - k0;
    } else if constexpr (FORM == kDx) {
      const int half = k0 >= p.Fp, f = k0 - half * p.Fp;
      bp = (const char*)p.p + ((int64_t)(half * p.F + f) * p.p_stride + n0) * es;
      bq = (const char*)p.q + ((int64_t)m0 * p.q_stride + k0) * es;
      left = p.F - f;
    } else {
      bp = (const char*)p.p + ((int64_t)k0 * p.p_stride + n0) * es;
      bq = (const char*)p.q + ((int64_t)k0 * p.q_stride + m0) * es;
      left = p.K - k0;
    }
    const uint32_t to = lds0 + (s & (kSwStages - 1)) * kStage;
    if (left >= E::kStep) {
#pragma unroll
      for (int i = 0; i < OpP::kLoads; ++i) sw_dma(bp, op.off[i], to + i * 4096);
#pragma unroll
      for (int i = 0; i < OpQ::kLoads; ++i) sw_dma(bq, oq.off[i], to + OpP::kBytes + i * 4096);
    } else {
      const char* z = (const char*)&sw_zeros;
#pragma unroll
      for (int i = 0; i < OpP::kLoads; ++i) sw_dma64(op.kr[i] < left ? bp + op.off[i] : z, to + i * 4096);
#pragma unroll
      for (int i = 0; i < OpQ::kLoads; ++i)
        // (dx: the gradients' columns behind the end are there, and zero)
        sw_dma64(FORM == kDx || oq.kr[i] < left ? bq + oq.off[i] : z, to + OpP::kBytes + i * 4096);
    }
  };

  sw_f16 acc[NP][NQ];
#pragma unroll
  for (int a = 0; a < NP; ++a)
#pragma unroll
    for (int b = 0; b < NQ; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;

  u32x4 fp[2][NP], fq[2][NQ];
  auto read = [&](int buf, uint32_t stage, int kk) {
#pragma unroll
    for (int j = 0; j < NP; ++j) fp[buf][j] = op.read(lds, stage, kk, j);
#pragma unroll
    for (int j = 0; j < NQ; ++j) fq[buf][j] = oq.read(lds, stage, kk, j);
  };
  auto multiply = [&](int buf) {
#pragma unroll
    for (int a = 0; a < NP; ++a)
#pragma unroll
      for (int b = 0; b < NQ; ++b) sw_mfma<DT>(fp[buf][a], fq[buf][b], acc[a][b]);
  };

  // the loads of the next `ahead` steps may still be under way
  auto wait = [&](int ahead) {
    if (ahead >= 2) sw_wait_barrier<2 * kLoads>();
    else if (ahead == 1) sw_wait_barrier<kLoads>();
    else sw_wait_barrier<0>();
  };

#pragma unroll
  for (int s = 0; s < kSwStages - 1; ++s)
    if (s < nk) load(s);
  wait(nk - 1);
  read(0, 0, 0);
  for (int s = 0; s < nk; ++s) {
    const uint32_t stage = (s & (kSwStages - 1)) * kStage;
    read(1, stage, 1);
    if (s + kSwStages - 1 < nk) load(s + kSwStages - 1);
    multiply(0);
    __builtin_amdgcn_sched_barrier(0);
    wait(nk - 2 - s);
    if (s + 1 < nk) read(0, ((s + 1) & (kSwStages - 1)) * kStage, 0);
    multiply(1);
    __builtin_amdgcn_sched_barrier(0);
  }

  if constexpr (SPLIT) {
    float* to = p.partials + ((int64_t)split * p.tiles_m * p.tiles_n + tile) * (BM * BN) + wave * (BM * BN / 4) + lane * 4;
#pragma unroll
    for (int b = 0; b < NQ; ++b)
#pragma unroll
      for (int a = 0; a < NP; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(sw_f4*)(to + ((b * NP + a) * 4 + i) * 256) =
              sw_f4{acc[a][b][4 * i], acc[a][b][4 * i + 1], acc[a][b][4 * i + 2], acc[a][b][4 * i + 3]};
  } else {
    sw_wait_barrier<0>();  // the stages are free
    constexpr int kPitch = kCols / 2 * es + 16;
    char* mine = lds + wave * (32 * kPitch);
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      float v[NP][16];
#pragma unroll
      for (int a = 0; a < NP; ++a)
#pragma unroll
        for (int i = 0; i < 16; ++i) v[a][i] = acc[a][b][i];
      sw_finish<DT, FORM, NP * 32>(p, mine, lane, m0 + wm * (BM / 2) + 32 * b, n0 + wn * (kCols / 2), v);
      __builtin_amdgcn_sched_barrier(0);  // (the next rows' registers not before these are stored)
    }
  }
}

// The splits' sums, in their order, and what the unsplit kernel does with them: a
// wave per 32 rows of a wave's columns.
template <class DT, int FORM, int BM, int BN>
__global__ __launch_bounds__(256) void swiglu_reduce_kernel(SwGemmParams p) {
  constexpr int NP = BN / 64, NQ = BM / 64;
  constexpr int kCols = FORM == kFwd ? BN / 2 : BN;
  // columns of a wave: all of them where u and z belong together, else one group of 32
  constexpr int G = FORM == kFwd ? NP : 1;
  constexpr int kParts = NP / G;
  constexpr int kStaged = FORM == kFwd ? NP * 16 : 32;
  constexpr int kPitch = kStaged * (int)sizeof(typename DT::S) + 16;
  __shared__ __align__(16) char lds[4 * 32 * kPitch];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tiles = p.tiles_m * p.tiles_n;
  const int w = blockIdx.x * 4 + wave;
  const int part = w % kParts, b = w / kParts % NQ, tw = w / (kParts * NQ) % 4, tile = w / (kParts * NQ * 4);
  if (tile >= tiles) return;
  const int per = 8 * p.tiles_n, g = tile / per, rows = min(p.tiles_m - g * 8, 8);
  const int tm = g * 8 + (tile - g * per) % rows, tn = (tile - g * per) / rows;
  float v[G][16];
#pragma unroll
  for (int a = 0; a < G; ++a)
#pragma unroll
    for (int i = 0; i < 16; ++i) v[a][i] = 0.f;
  const float* from = p.partials + (int64_t)tile * (BM * BN) + tw * (BM * BN / 4) + (b * NP + part * G) * 1024 + lane * 4;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float* at = from + (int64_t)s * tiles * (BM * BN);
#pragma unroll
    for (int a = 0; a < G; ++a)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const sw_f4 x = *(const sw_f4*)(at + (a * 4 + i) * 256);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[a][4 * i + e] += x[e];
      }
  }
  const int wm = tw & 1, wn = tw >> 1;
  sw_finish<DT, FORM, G * 32>(p, lds + wave * 32 * kPitch, lane, tm * BM + wm * (BM / 2) + 32 * b,
                              tn * kCols + wn * (kCols / 2) + part * 32, v);
}

template <class DT, int FORM, int BM, int BN>
hipError_t sw_run(const SwGemmParams& p, hipStream_t st) {
  const int tiles = p.tiles_m * p.tiles_n;
  if (p.splits <= 1) {
    swiglu_gemm_kernel<DT, FORM, BM, BN, false><<<dim3(tiles), dim3(256), 0, st>>>(p);
    return hipGetLastError();
  }
  swiglu_gemm_kernel<DT, FORM, BM, BN, true><<<dim3(tiles * p.splits), dim3(256), 0, st>>>(p);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  const int waves = tiles * 4 * (BM / 64) * (FORM == kFwd ? 1 : BN / 64);
  swiglu_reduce_kernel<DT, FORM, BM, BN><<<dim3((waves + 3) / 4), dim3(256), 0, st>>>(p);
  return hipGetLastError();
}

template <class DT, int FORM>
hipError_t sw_tile_pick(int tile, const SwGemmParams& p, hipStream_t st) {
  if (tile == 0) return sw_run<DT, FORM, 256, 256>(p, st);
  if (tile == 1) return sw_run<DT, FORM, 128, 128>(p, st);
  return sw_run<DT, FORM, 64, 128>(p, st);
}

template <class DT>
hipError_t sw_form_pick(int form, int tile, const SwGemmParams& p, hipStream_t st) {
  if (form == kFwd) return sw_tile_pick<DT, kFwd>(tile, p, st);
  if (form == kDx) return sw_tile_pick<DT, kDx>(tile, p, st);
  return sw_tile_pick<DT, kDw>(tile, p, st);
}

}  // namespace attnres
