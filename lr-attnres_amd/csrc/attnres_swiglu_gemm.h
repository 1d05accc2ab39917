// The product's kernels: one instantiation per type, form and tile, and the sum of
// split products.  Included by attnres_swiglu_{bf16,f16,f32}.hip.
#pragma once

#include <type_traits>

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

// A wave's 32 x COLS values go to memory through its own LDS: lane l holds in v[j][4 i + e]
// row sw_row(l, i), column 32 j + sw_col(l, i) + e, and takes back 16 bytes of a row, so
// that memory sees whole 64-byte pieces.  Rows are 16 bytes longer than what they hold, so
// that those of a write start in different banks.  The reads of 16 bytes still meet in some:
// conflicts are 20% of the LDS cycles of the forward at dim 1024, hidden 4096 (rows of 144 and
// 80 bytes) and 57% of the split sums', which memory bounds, but 2% of dx's (rows of 272).
constexpr int sw_pitch(int row_bytes) { return row_bytes + 16; }
__device__ __forceinline__ int sw_row(int lane, int i) { return (lane & 15) + 16 * (i >> 1); }
__device__ __forceinline__ int sw_col(int lane, int i) { return 4 * (lane >> 4) + 16 * (i & 1); }

template <class DT, int G>
__device__ __forceinline__ void sw_put(char* lds, int lane, const float (&v)[G][16]) {
  constexpr int kSize = sizeof(typename DT::S);
#pragma unroll
  for (int j = 0; j < G; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* x = &v[j][4 * i];
      char* at = lds + sw_row(lane, i) * sw_pitch(G * 32 * kSize) + (j * 32 + sw_col(lane, i)) * kSize;
      if constexpr (kSize == 2) *(u32x2*)at = u32x2{pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3])};
      else *(sw_f4*)at = sw_f4{x[0], x[1], x[2], x[3]};
    }
}

// Rows of the output: chunk c of row m to row(m) + 16 c bytes, columns n0.. below n_end
template <int ROW_BYTES, int SIZE, class Row>
__device__ __forceinline__ void sw_take_rows(const char* lds, int lane, bool whole, int n0, int n_end, bool vec, Row row) {
  constexpr int kChunks = ROW_BYTES / 16, kPer = 16 / SIZE, kIters = 32 * kChunks / kWave;
  u32x4 x[kIters];
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    const int q = i * kWave + lane;
    x[i] = *(const u32x4*)(lds + q / kChunks * sw_pitch(ROW_BYTES) + q % kChunks * 16);
  }
  if (whole) {  // (the whole tile: no row or column is left out)
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      const int q = i * kWave + lane;
      *(u32x4*)(row(q / kChunks) + q % kChunks * 16) = x[i];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    const int q = i * kWave + lane, c = q % kChunks, n = n0 + c * kPer;
    char* dst = row(q / kChunks);
    if (!dst || n >= n_end) continue;
    if (vec && n + kPer <= n_end) {
      *(u32x4*)(dst + c * 16) = x[i];
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        if (n + e >= n_end) break;
        if constexpr (SIZE == 2) ((uint16_t*)dst)[c * kPer + e] = (uint16_t)(x[i][e / 2] >> (16 * (e & 1)));
        else ((uint32_t*)dst)[c * kPer + e] = x[i][e];
      }
    }
  }
}

// Rows of a plane in blocks (SwPlanes): G groups of 32 columns, BLOCK bytes of a row a block
template <int ROW_BYTES, int BLOCK>
__device__ __forceinline__ void sw_take_blocks(const char* lds, int lane, char* plane, int block0, int blocks, int64_t n,
                                               int m0, int M) {
  constexpr int kPer = BLOCK / 16, kBlocks = ROW_BYTES / BLOCK;  // chunks of a block's row, blocks
  constexpr int kRows = kWave / kPer, kIters = 32 / kRows;       // rows that a wave stores at a time
  const int r = lane / kPer, c = lane % kPer;
  const char* from = lds + r * sw_pitch(ROW_BYTES) + c * 16;
  u32x4 x[kBlocks][kIters];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int i = 0; i < kIters; ++i) x[b][i] = *(const u32x4*)(from + i * kRows * sw_pitch(ROW_BYTES) + b * BLOCK);
  char* to = plane + ((int64_t)block0 * n + m0 + r) * BLOCK + c * 16;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    if (block0 + b < blocks) {
      if (m0 + 32 <= M) {
#pragma unroll
        for (int i = 0; i < kIters; ++i) *(u32x4*)(to + i * kRows * BLOCK) = x[b][i];
      } else {
#pragma unroll
        for (int i = 0; i < kIters; ++i)
          if (m0 + r + i * kRows < M) *(u32x4*)(to + i * kRows * BLOCK) = x[b][i];
      }
    }
    to += n * BLOCK;
  }
}

// u and z of a wave's 32 rows to the planes that the backward reads
template <class DT, int H>
__device__ __forceinline__ void sw_save(const SwGemmParams& p, char* lds, int lane, int m0, int n0, const float (&v)[2 * H][16]) {
  using P = SwPlanes<DT>;
  constexpr int kSize = sizeof(typename DT::S), kRow = H * 32 * kSize;
  constexpr int kStep = SwElem<DT>::kStep;
  const SwPlaneAddress at = sw_planes<DT>(p.saved, p.n_tok, p.Fp);
  const int blocks = p.Fp / kStep, block0 = n0 / kStep;
  if constexpr (kSize == 4) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float x[H][16];
#pragma unroll
      for (int j = 0; j < H; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[j][i] = v[half * H + j][i];
      sw_put<DT, H>(lds, lane, x);
      __builtin_amdgcn_wave_barrier();
      sw_take_blocks<kRow, kSwStepBytes>(lds, lane, half ? at.z : at.u, block0, blocks, p.n_tok, m0, p.M);
      __builtin_amdgcn_wave_barrier();
    }
  } else {
    constexpr int L = P::kLow, kLowRow = H * 32 * L / 4;  // bytes of the low bits of a row's pairs
    char* zu = lds + 32 * sw_pitch(kRow);
    char* lo = zu + 32 * sw_pitch(kRow);
#pragma unroll
    for (int j = 0; j < H; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t u[4], z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u[e] = sw_round_bits<L>(v[j][4 * i + e]);
          z[e] = sw_round_bits<L>(v[H + j][4 * i + e]);
        }
        const int m = sw_row(lane, i), col = j * 32 + sw_col(lane, i);
        *(u32x2*)(lds + m * sw_pitch(kRow) + col * 2) = u32x2{hi_pair(u[0], u[1]), hi_pair(u[2], u[3])};
        *(u32x2*)(zu + m * sw_pitch(kRow) + col * 2) = u32x2{hi_pair(z[0], z[1]), hi_pair(z[2], z[3])};
        sw_store_low<L>(lo + m * sw_pitch(kLowRow), col, u, z);
      }
    __builtin_amdgcn_wave_barrier();
    sw_take_blocks<kRow, kSwStepBytes>(lds, lane, at.u, block0, blocks, p.n_tok, m0, p.M);
    sw_take_blocks<kRow, kSwStepBytes>(zu, lane, at.z, block0, blocks, p.n_tok, m0, p.M);
    sw_take_blocks<kLowRow, P::kLowBlock>(lo, lane, at.low, block0, blocks, p.n_tok, m0, p.M);
    __builtin_amdgcn_wave_barrier();
  }
}

// LDS bytes of a wave in sw_finish, COLS columns of the product
template <class DT, int FORM, int COLS>
constexpr int sw_finish_lds() {
  constexpr int kSize = sizeof(typename DT::S), H = FORM == kFwd ? COLS / 2 : COLS;
  int n = 32 * sw_pitch(H * kSize);
  if (FORM == kFwd && kSize == 2) n = 2 * n + 32 * sw_pitch(H * SwPlanes<DT>::kLow / 4);
  return n;
}

// What becomes of a wave's 32 rows m0.. x COLS columns of the product (fwd: COLS is
// u and z together).  v holds the sums.
template <class DT, int FORM, int COLS>
__device__ __forceinline__ void sw_finish(const SwGemmParams& p, char* lds, int lane, int m0, int n0,
                                          float (&v)[COLS / 32][16]) {
  constexpr int kSize = sizeof(typename DT::S);
  if constexpr (FORM == kFwd) {
    constexpr int H = COLS / 64;  // 32-column groups of u
    if (p.saved) sw_save<DT, H>(p, lds, lane, m0, n0, v);
    float h[H][16];
#pragma unroll
    for (int j = 0; j < H; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) h[j][i] = v[j][i] * sw_silu<DT>(v[H + j][i]);
    sw_put<DT, H>(lds, lane, h);
    __builtin_amdgcn_wave_barrier();
    const bool whole = m0 + 32 <= p.M && n0 + H * 32 <= p.n_out && p.out_vec;
    char* out = (char*)p.out + ((int64_t)m0 * p.out_stride + n0) * kSize;
    sw_take_rows<H * 32 * kSize, kSize>(lds, lane, whole, n0, p.n_out, p.out_vec, [&](int m) -> char* {
      return whole || m0 + m < p.M ? out + (int64_t)m * p.out_stride * kSize : nullptr;
    });
  } else {
    sw_put<DT, COLS / 32>(lds, lane, v);
    __builtin_amdgcn_wave_barrier();
    // dw: rows of the padded halves, these (perhaps) in both
    const int half = FORM == kDw && m0 >= p.Fp, skip = half * (p.Fp - p.F);
    const int end = FORM == kDw ? half * p.Fp + p.F : p.M;  // of the rows that begin here
    const bool whole = m0 + 32 <= end && n0 + COLS <= p.n_out && p.out_vec;
    char* out = (char*)p.out + ((int64_t)(m0 - skip) * p.out_stride + n0) * kSize;
    sw_take_rows<COLS * kSize, kSize>(lds, lane, whole, n0, p.n_out, p.out_vec, [&](int m) -> char* {
      char* row = out + (int64_t)m * p.out_stride * kSize;
      if (whole || m0 + m < end) return row;
      if (FORM == kDw && !half && m0 + m >= p.Fp && m0 + m < p.Fp + p.F) return row - (int64_t)(p.Fp - p.F) * p.out_stride * kSize;
      return nullptr;
    });
  }
  __builtin_amdgcn_wave_barrier();
}

template <class DT, int FORM, int BM, int BN, bool SPLIT>
__global__ __launch_bounds__(256, sw_per_cu(BM, BN) < 2 ? 1 : 2) void swiglu_gemm_kernel(SwGemmParams p) {
  using E = SwElem<DT>;
  constexpr int KS = FORM == kFwd ? 2 : 1;  // k steps of a stage
  constexpr int kStageK = E::kStep * KS;
  using OpP = SwOperand<DT, BN, FORM != kFwd, KS>;
  using OpQ = SwOperand<DT, BM, FORM == kDw, FORM == kFwd ? KS : 1>;
  constexpr int NP = BN / 32, NQ = BM / 32;  // 16 x 16 tiles of a wave
  constexpr int kStage = OpP::kBytes + OpQ::kBytes;
  constexpr int kStages = sw_steps(BM, BN) / KS, kAhead = kStages - 1;  // stages loaded ahead
  constexpr int kLoads = OpP::kLoads + OpQ::kLoads;
  constexpr int kCols = FORM == kFwd ? BN / 2 : BN;  // output columns of a tile
  constexpr int es = E::kSize;
  __shared__ __align__(1024) char lds[kStages * kStage];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  int split, tm, tn, tile;
  sw_tile(p, blockIdx.x, gridDim.x, &split, &tm, &tn, &tile);
  const int m0 = tm * BM, n0 = tn * kCols;
  const int all_steps = (p.K + kStageK - 1) / kStageK;  // (stages)
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
      // (dx: rows of a block are kSwStepBytes apart)
      oq.off[i] = (uint32_t)((min(m0 + r, p.M - 1) - m0) * (FORM == kDx ? kSwStepBytes : p.q_stride * es)) + c * 16;
      oq.kr[i] = c * E::kPer;
    } else {
      const int block = min(c / 4, (p.M - m0) / E::kStep - 1);
      oq.off[i] = (uint32_t)((block * p.n_tok + r) * kSwStepBytes) + c % 4 * 16;
      oq.kr[i] = r;
    }
  }
  op.place_reads(wn * (BN / 2), lane, 0);
  oq.place_reads(wm * (BM / 2), lane, OpP::kBytes);
  const uint32_t lds0 = lds_address(lds) + wave * 1024;

  // (kept in a register: read from memory in the loop, it would make every wait for
  // LDS a wait for everything)
  const char* zeros = (const char*)&sw_zeros;
  asm volatile("" : "+s"(zeros));

  // Loads of the next step into its stage, piece by piece so that the matrix cores
  // work between them.
  const int k0 = first * kStageK;
  const char* bp = (const char*)p.p + (FORM == kFwd ? (int64_t)k0 : (int64_t)k0 * p.p_stride + n0) * es;
  const char* bq = (const char*)p.q + (FORM == kFwd  ? ((int64_t)m0 * p.q_stride + k0) * es
                                       : FORM == kDx ? ((int64_t)(k0 / E::kStep) * p.n_tok + m0) * kSwStepBytes
                                                     : ((int64_t)(m0 / E::kStep) * p.n_tok + k0) * kSwStepBytes);
  const int64_t ahead_p = FORM == kFwd ? kSwStepBytes * KS : (int64_t)E::kStep * p.p_stride * es;
  const int64_t ahead_q = FORM == kFwd  ? kSwStepBytes * KS
                          : FORM == kDx ? p.n_tok * kSwStepBytes
                                        : (int64_t)E::kStep * kSwStepBytes;
  auto behind = [](uint32_t stage) { return stage == (kStages - 1) * kStage ? 0u : stage + kStage; };
  uint32_t to = 0;  // the step's stage, in bytes
  auto next_step = [&]() {
    bp += ahead_p;
    bq += ahead_q;
    to = behind(to);
  };
  auto load_piece = [&](int i) {  // of a whole step
    if (i < OpP::kLoads) sw_dma(bp, op.off[i % OpP::kLoads], lds0 + to + i * 4096);
    else sw_dma(bq, oq.off[(i - OpP::kLoads) % OpQ::kLoads], lds0 + to + OpP::kBytes + (i - OpP::kLoads) * 4096);
  };
  auto load = [&](int s) {  // step s of the split, k possibly ending in it
    const int left = p.K - (first + s) * kStageK;
    if (left >= kStageK) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) load_piece(i);
    } else {
#pragma unroll
      for (int i = 0; i < OpP::kLoads; ++i) sw_dma64(op.kr[i] < left ? bp + op.off[i] : zeros, lds0 + to + i * 4096);
#pragma unroll
      for (int i = 0; i < OpQ::kLoads; ++i)
        sw_dma64(oq.kr[i] < left ? bq + oq.off[i] : zeros, lds0 + to + OpP::kBytes + i * 4096);
    }
    next_step();
  };

  sw_f4 acc[NP][NQ];
#pragma unroll
  for (int a = 0; a < NP; ++a)
#pragma unroll
    for (int b = 0; b < NQ; ++b) acc[a][b] = sw_f4{0.f, 0.f, 0.f, 0.f};

  // A step's products in two halves, rows of P by rows of Q: fragments are read into the
  // registers of those that are used up, half a step and more before they are needed.
  //   half 0: rows 0.. H - 1 of P by all of Q, while the other rows of P are read (this
  //           step's)
  //   half 1: rows H.. by all of Q, column by column; behind each the next step's fragment
  //           of Q takes its place, and early on the next step's first rows of P
  // A later stage's loads are issued between the products of half 0, or (forward) of the
  // half 1 behind the barrier that frees the stage.
  constexpr int H = NP / 2, kHalf = H * NQ;
  using Yes = std::true_type;
  using No = std::false_type;
  u32x4 fp[NP], fq[NQ];
  auto half0 = [&](uint32_t stage, int ks, auto loads) {
    constexpr int kOps = H + (decltype(loads)::value ? kLoads : 0);
#pragma unroll
    for (int t = 0; t < kHalf; ++t) {
      sw_mfma<DT>(fp[t % H], fq[t / H], acc[t % H][t / H]);
#pragma unroll
      for (int i = 0; i < (kOps + kHalf - 1) / kHalf; ++i) {
        const int e = (t * kOps + kHalf - 1) / kHalf + i;  // op e goes behind product e kHalf / kOps
        if (e >= ((t + 1) * kOps + kHalf - 1) / kHalf) continue;
        if (e < H) fp[H + e % H] = op.read(lds, stage, ks, H + e % H);
        else load_piece(e - H);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto half1 = [&](uint32_t next, int ks, auto loads) {  // next, ks: the next step's stage and place in it
#pragma unroll
    for (int t = 0; t < kHalf; ++t) {
      sw_mfma<DT>(fp[H + t % H], fq[t / H], acc[H + t % H][t / H]);
      if (t < H) fp[t] = op.read(lds, next, ks, t);
      if (t % H == H - 1) fq[t / H] = oq.read(lds, next, ks, t / H);
      if constexpr (decltype(loads)::value) {
#pragma unroll
        for (int i = 0; i < (kLoads + kHalf - 1) / kHalf; ++i) {
          const int e = (t * kLoads + kHalf - 1) / kHalf + i;
          if (e < ((t + 1) * kLoads + kHalf - 1) / kHalf) load_piece(e);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // the loads of the next `ahead` stages may still be under way
  auto wait = [&](int ahead) {
    if (ahead >= 2 && kAhead > 2) sw_wait_barrier<(kAhead > 2 ? 2 : 0) * kLoads>();
    else if (ahead >= 1 && kAhead > 1) sw_wait_barrier<kLoads>();
    else sw_wait_barrier<0>();
  };

  constexpr int kBegin = KS == 2 ? kStages : kAhead;  // stages loaded before the first product
#pragma unroll
  for (int s = 0; s < kBegin; ++s)
    if (s < nk) load(s);
  if constexpr (KS == 2) {
    if (nk > 1) sw_wait_barrier<kLoads>();
    else sw_wait_barrier<0>();
  } else {
    wait(nk - 1);
  }
#pragma unroll
  for (int j = 0; j < H; ++j) fp[j] = op.read(lds, 0, 0, j);
#pragma unroll
  for (int j = 0; j < NQ; ++j) fq[j] = oq.read(lds, 0, 0, j);
  // (no instruction: between the two loops the largest tile's sums stand in the
  // accumulation registers, and so the compiler moves none of them around in either)
  auto pin = [&]() {
    if constexpr (NP * NQ == 64) {
#pragma unroll
      for (int a = 0; a < NP; ++a)
#pragma unroll
        for (int b = 0; b < NQ; ++b) asm volatile("" : "+a"(acc[a][b]));
    }
  };
  const int whole = (int)min((int64_t)nk, (int64_t)p.K / kStageK - first);  // stages in which k does not end
  int s = 0;
  uint32_t stage = 0;
  if constexpr (KS == 2) {
    for (; s + kStages < whole; ++s) {
      half0(stage, 0, No());
      half1(stage, 1, No());
      half0(stage, 1, No());
      stage = behind(stage);
      sw_wait_barrier<0>();  // the next stage has landed, this one is free
      half1(stage, 0, Yes());
      next_step();
    }
    pin();
    for (; s < nk; ++s) {
      half0(stage, 0, No());
      half1(stage, 1, No());
      half0(stage, 1, No());
      stage = behind(stage);
      sw_wait_barrier<0>();
      if (s + kStages < nk) load(s + kStages);
      half1(stage, 0, No());  // (behind the last step: fragments read, not used)
    }
  } else {
    for (; s + kAhead < whole; ++s) {
      half0(stage, 0, Yes());
      next_step();
      stage = behind(stage);
      sw_wait_barrier<(kAhead - 1) * kLoads>();
      half1(stage, 0, No());
    }
    pin();
    for (; s < nk; ++s) {
      if (s + kAhead < nk) load(s + kAhead);
      half0(stage, 0, No());
      stage = behind(stage);
      wait(nk - 2 - s);
      half1(stage, 0, No());  // (behind the last step: fragments read, not used)
    }
  }

  if constexpr (SPLIT) {
    float* to = p.partials + ((int64_t)split * p.tiles_m * p.tiles_n + tile) * (BM * BN) + wave * (BM * BN / 4) + lane * 4;
#pragma unroll
    for (int b = 0; b < NQ / 2; ++b)
#pragma unroll
      for (int a = 0; a < NP / 2; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) *(sw_f4*)(to + ((b * (NP / 2) + a) * 4 + i) * 256) = acc[2 * a + (i & 1)][2 * b + (i >> 1)];
  } else {
    sw_wait_barrier<0>();  // the stages are free
    constexpr int kMine = sw_finish_lds<DT, FORM, NP * 16>();
    static_assert(4 * kMine <= kStages * kStage, "LDS");
    char* mine = lds + wave * kMine;
#pragma unroll
    for (int b = 0; b < NQ / 2; ++b) {
      float v[NP / 2][16];
#pragma unroll
      for (int a = 0; a < NP / 2; ++a)
#pragma unroll
        for (int i = 0; i < 16; ++i) v[a][i] = acc[2 * a + (i >> 2 & 1)][2 * b + (i >> 3)][i & 3];
      sw_finish<DT, FORM, NP * 16>(p, mine, lane, m0 + wm * (BM / 2) + 32 * b, n0 + wn * (kCols / 2), v);
      __builtin_amdgcn_sched_barrier(0);  // (the next rows' registers not before these are stored)
    }
  }
}

// The splits' sums, in their order, and what the unsplit kernel does with them: a
// wave per 32 rows of a wave's columns.
template <class DT, int FORM, int BM, int BN>
__global__ __launch_bounds__(256) void swiglu_reduce_kernel(SwGemmParams p) {
  constexpr int NP = BN / 64, NQ = BM / 64;  // 32 x 32 values
  constexpr int kCols = FORM == kFwd ? BN / 2 : BN;
  // columns of a wave: all of them where u and z belong together, else one group of 32
  constexpr int G = FORM == kFwd ? NP : 1;
  constexpr int kParts = NP / G;
  constexpr int kMine = sw_finish_lds<DT, FORM, G * 32>();
  __shared__ __align__(16) char lds[4 * kMine];
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
  sw_finish<DT, FORM, G * 32>(p, lds + wave * kMine, lane, tm * BM + wm * (BM / 2) + 32 * b,
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
  if constexpr (sw_has_tile(FORM, DT::kCode, 0)) {
    if (tile == 0) return sw_run<DT, FORM, 256, 256>(p, st);
  }
  if constexpr (sw_has_tile(FORM, DT::kCode, 1)) {
    if (tile == 1) return sw_run<DT, FORM, 128, 256>(p, st);
  }
  if (tile < 2) return hipErrorInvalidValue;
  if (tile == 2) return sw_run<DT, FORM, 128, 128>(p, st);
  return sw_run<DT, FORM, 64, 128>(p, st);
}

template <class DT>
hipError_t sw_form_pick(int form, int tile, const SwGemmParams& p, hipStream_t st) {
  if (form == kFwd) return sw_tile_pick<DT, kFwd>(tile, p, st);
  if (form == kDx) return sw_tile_pick<DT, kDx>(tile, p, st);
  return sw_tile_pick<DT, kDw>(tile, p, st);
}

}  // namespace attnres
