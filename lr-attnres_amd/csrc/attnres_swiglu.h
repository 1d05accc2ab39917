// The matrix-core product of the gated feed-forward kernels (attnres_swiglu*.hip).
//
//   C[m, n] = sum_k Q[m, k] P[n, k]
// in three forms:
//   kFwd  P = W, Q = x (both with k contiguous), k over dim: a tile's P rows are half
//         up and half gate rows of the same hidden columns, so that a lane ends with
//         u and z of one element and forms u silu(z) in its registers
//   kDx   P = W^T, Q = [du dz], k over both halves of the hidden dimension
//   kDw   P = x^T, Q = [du dz]^T, k over tokens
//
// Tile.  Four waves, 2 x 2, each with a quarter of the BM x BN tile as 16 x 16 MFMA
// tiles.  P is the MFMA's row operand, so that a lane holds for one m (lane % 16)
// groups of 4 consecutive n.  k runs in steps of 64 bytes, one MFMA deep in 16 bits,
// through the stages of LDS, filled by loads that write LDS directly (16 bytes a
// lane; no registers) several steps ahead; a wave reads the fragments of the next
// step while the matrix cores work on this one, into the registers of used ones.  One
// barrier a stage: behind it the next stage has landed (each wave waited for its own
// loads) and nobody reads this one any more, so that the loads issued next go there.
//
// LDS layouts (a stage holds R rows of 64 bytes, or 32 / 16 rows of R values):
//   k contiguous: the 16-byte chunks of row r are swapped by f(r) = 3 (r / 8 % 2), of rows of
//     two steps by r / 2 % 8.  A read serves 16 lanes at once, lanes 0-3, 12-15 and 20-27
//     first: rows 0-3 and 12-15 with one chunk, rows 4-11 with the next; so they lie in
//     all banks (with r / 2 % 4 ^ r / 8 % 2 half of the cycles were conflicts)
//   k strided, 16-bit: 32-byte units of row k are swapped by s(k) = 2 (k % 4) ^ (k / 2 %
//     2) ^ (k / 8 % 2) for the transposing reads (4 rows x 32 bytes per 16 lanes, rows 8
//     apart in neighbouring 16s)
//   k strided, fp32: rows as they are; a fragment's values are read one by one
// The direct loads write LDS in lane order, so the swaps are made in the addresses
// that the lanes read from.
//
// Forward.  Both operands are rows of the caller's, and a step's 64 bytes of one are half a
// line: loaded step by step, the L2 caches serve twice the requests for the same bytes
// (33 million against 17 at 16384 tokens, dim 1024, hidden 4096) and become the limit.
// There a stage holds two steps; there are two of them, and one barrier a stage.
//
// Measured (bf16, one MI355X, 16384 tokens, dim 1024, hidden 4096; after a hundred
// passes): forward 273 us, with u and z kept 304-309 (1.01 and 0.89-0.9 PFLOP/s), dx
// 191-196 (1.4), dw 200-204 (1.35).  Matrix cores busy: 41%, 72% and 69% of the waves'
// life.  The clock falls to 1.55-1.8 GHz in these products, so power bounds dx and dw (in
// the first milliseconds of such a load all three take up to a third longer).  The forward
// is bound by what a tile does before and after its k steps (first loads 1.9 us, stores
// 3.6, 7.7 with u and z), in series with 26 us of products.  Two workgroups of 128 x 256 on a CU
// took 340 us without u and z where 256 x 256 took 290.  On 32 x 32 MFMAs dx took 212 and
// dw 218 where they then took 193 and 200.
//
// k beyond its end (dim not a whole number of steps, the last tokens, hidden columns
// that fill no step) is loaded from a block of zeros, so that both operands vanish
// there and no value behind the end is touched.
#pragma once

#include "attnres_device.h"
#include "attnres_sublayers.h"

namespace attnres {

enum SwForm { kFwd = 0, kDx = 1, kDw = 2 };

constexpr int kSwStepBytes = 64;  // of k, per row: 32 16-bit values, 16 fp32
constexpr int kSwTiles = 4;
constexpr int kSwTileM[kSwTiles] = {256, 128, 128, 64}, kSwTileN[kSwTiles] = {256, 256, 128, 128};
// which of them a product has: a forward's two stages of two steps do not fit three steps
// of LDS; in fp32, with a sixteenth of the matrix rate, smaller tiles are never slower
// than the largest one
constexpr bool sw_has_tile(int form, int dtype, int tile) {
  return tile > 1 || (tile == 1 ? form != kFwd : dtype != F32::kCode);
}
// k steps of LDS (forward: two stages of two steps), and the workgroups that a CU's 160 KB
// then hold
constexpr int sw_steps(int bm, int bn) { return bm + bn == 384 ? 3 : 4; }
constexpr int sw_per_cu(int bm, int bn) { return 160 * 1024 / (sw_steps(bm, bn) * (bm + bn) * kSwStepBytes); }

struct SwGemmParams {
  const void* p;            // fwd / dx: W; dw: x
  const void* q;            // fwd: x; dx / dw: [du dz], in blocks
  int64_t p_stride, q_stride;
  int32_t M, N;             // rows / columns of the product (fwd: N = hidden; else in whole chunks)
  int32_t n_out;            // columns of the output
  int32_t K;                // fwd: dim, dx: 2 Fp, dw: tokens
  int32_t F, Fp;            // hidden, and rounded up to a whole number of steps
  int32_t tiles_m, tiles_n;
  int32_t splits, steps;    // k steps of a split
  void* out;                // [M, N] (dw: rows of the padded halves are left out)
  int64_t out_stride;
  int32_t out_vec;          // whole 16-byte stores to out
  void* saved;              // fwd: u and z (SwPlanes), or null
  int64_t n_tok;
  float* partials;          // splits > 1: [splits, tiles, BM * BN] in the kernel's own order
};

hipError_t launch_swiglu_gemm(int dtype, int form, int tile, const SwGemmParams& p, hipStream_t st);
constexpr int kSwFew = 64;  // rows at most
hipError_t launch_swiglu_few(int dtype, const SwGemmParams& p, hipStream_t st);  // the forward

// [du dz] of the backward, in blocks, with zeros behind each half's F columns
struct SwGradParams {
  const void* dh;           // [n, F], rows of dh_stride
  const void* saved;        // u and z (SwPlanes)
  void* d;                  // [2 Fp / step blocks, n, step]
  int64_t n, dh_stride;
  int32_t F, Fp;
  int32_t vec;              // whole 16-byte loads of dh
};
hipError_t launch_swiglu_grad(int dtype, const SwGradParams& p, hipStream_t st);

// Copies of operands: blocks of `rows` rows of cols values to blocks of `to_rows` rows of
// to_stride (whole chunks), zeros behind the columns and the rows.  One or two at once.
struct SwPack {
  const void* from;
  void* to;
  int64_t rows, to_rows, from_stride;
  int32_t blocks;
};
struct SwPackParams {
  SwPack part[2];
  int32_t parts, cols, to_stride;
};
hipError_t launch_swiglu_pack(int dtype, const SwPackParams& p, hipStream_t st);
hipError_t launch_swiglu_clear(int dtype, void* to, int64_t values, hipStream_t st);

// ---------------------------------------------------------------------- device

template <class DT> struct SwElem {  // 16-byte fragments and their MFMA
  static constexpr int kSize = sizeof(typename DT::S);
  static constexpr int kPer = 16 / kSize;                // values in a chunk
  static constexpr int kStep = kSwStepBytes / kSize;     // k of a step
};

typedef float sw_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 sw_bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 sw_h8 __attribute__((ext_vector_type(8)));
typedef short sw_s4 __attribute__((ext_vector_type(4)));

// acc += P-fragment x Q-fragment, 16 x 16 values and 64 bytes of k: lane l holds 16 bytes
// of row l % 16, the l / 16-th of them.  fp32: four products of 4 k each, the same
// permutation of k on both sides.  Of the sums, lane l holds column l % 16 (of Q),
// rows 4 (l / 16) + 0..3 (of P).
template <class DT>
__device__ __forceinline__ void sw_mfma(const u32x4& a, const u32x4& b, sw_f4& c) {
  if constexpr (DT::kCode == 1) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(sw_bf8, a), __builtin_bit_cast(sw_bf8, b), c, 0, 0, 0);
  } else if constexpr (DT::kCode == 2) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(sw_h8, a), __builtin_bit_cast(sw_h8, b), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
  }
}

// What the forward keeps of u and z, and [du dz] of the backward, is the kernels' own
// and stands in blocks of one k step: [blocks, n, step] values.  A product's tile of
// [du dz] is then one run of memory (as rows of 2 Fp values it was 256 pieces of 64
// bytes, a page or more apart), and both sides of the activation's gradient are.
// u and z are kept to 16 + kLow bits of their fp32 value, in two planes: rounded to the
// dtype they would add two roundings to the one that [du dz] itself needs (an error of
// 1.7 times the result's own rounding in dx and dweight; so it is 1.4 times).
template <class DT> struct SwPlanes {
  static constexpr int kLow = DT::kCode == 1 ? 4 : DT::kCode == 2 ? 8 : 0;
  static constexpr int kLowBlock = SwElem<DT>::kStep * 2 * kLow / 8;  // bytes of a block's row of low bits
};
struct SwPlaneAddress {
  char *u, *z, *low;
};
template <class DT>
__host__ __device__ inline SwPlaneAddress sw_planes(const void* saved, int64_t n, int Fp) {
  const int64_t plane = n * Fp * SwElem<DT>::kSize;
  char* at = (char*)saved;
  return {at, at + plane, at + 2 * plane};
}

// fp32 bits to be cut to 16 + L of them, rounded to nearest.  (A NaN stays one: those of
// 16-bit operands, and the hardware's own, have no bits that the addition could carry.)
template <int L>
__device__ __forceinline__ uint32_t sw_round_bits(float x) {
  return __float_as_uint(x) + (1u << (15 - L));
}
// byte 1 of each of four words
__device__ __forceinline__ uint32_t sw_bytes1(const uint32_t (&w)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0501u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010c0cu);
  return a | b;
}
// and the low bits of four pairs (u, z) of a row, from column col on: u's below z's
template <int L>
__device__ __forceinline__ void sw_store_low(char* row, int64_t col, const uint32_t (&u)[4], const uint32_t (&z)[4]) {
  if constexpr (L == 4) {  // a byte a pair
    *(uint32_t*)(row + col) = (sw_bytes1(u) >> 4 & 0x0f0f0f0fu) | (sw_bytes1(z) & 0xf0f0f0f0u);
  } else {  // two bytes a pair
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_perm(z[e], u[e], 0x0c0c0501u);
    *(u32x2*)(row + col * 2) = u32x2{lo_pair(w[0], w[1]), lo_pair(w[2], w[3])};
  }
}

// 16 bytes a lane from global memory straight to LDS: lane l's to lds + 16 l.  No
// register is written, so nothing in flight can overwrite one; the waits are the
// kernel's own (sw_wait).
__device__ __forceinline__ void sw_dma(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void sw_dma64(const char* at, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(at), "s"(lds) : "memory", "m0");
}
// this wave's LDS reads are done and at most N of its loads are under way; then all waves meet
template <int N>
__device__ __forceinline__ void sw_wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}

// One operand of R rows (values along m or n) in LDS.  T: k strided in memory; KS: k steps
// of a stage (k contiguous: 2 make whole 128-byte lines of a row).
template <class DT, int R, bool T, int KS = 1>
struct SwOperand {
  using E = SwElem<DT>;
  static_assert(KS == 1 || !T, "steps of a stage");
  static constexpr int kBytes = R * kSwStepBytes * KS;    // of a stage
  static constexpr int kLoads = R / 64 * KS;              // direct loads of a thread per stage
  static constexpr int kRowChunks = R / E::kPer;          // strided: chunks of a row of R values
  static constexpr int kUnitMask = R / 16 - 1;            // strided 16-bit: 32-byte units of a row
  uint32_t off[kLoads];   // byte offsets of this thread's chunks from the step's base
  int kr[kLoads];         // and their k: chunk * kPer (contiguous) or row (strided)
  static constexpr int kReads = T ? R / 32 : KS;
  uint32_t rd[kReads];    // byte addresses of this lane's fragments: strided, one for each 16 rows of
                          // a wave; contiguous, for each step of a stage

  __device__ static int f_row(int r) {
    return KS == 2 ? (r >> 1) & 7 : ((r >> 3) & 1) * 3;
  }
  __device__ static int s_row(int k) { return ((2 * (k & 3)) ^ ((k >> 1) & 1) ^ ((k >> 3) & 1)) & kUnitMask; }

  // row / first k and chunk of load i of a thread
  __device__ __forceinline__ static void place(int i, int tid, int* row, int* chunk) {
    const int q = i * 256 + tid;
    if constexpr (!T) {
      *row = q / (4 * KS);
      *chunk = q % (4 * KS) ^ f_row(*row);
    } else {
      *row = q / kRowChunks;
      const int c = q % kRowChunks;
      if constexpr (E::kSize == 2) *chunk = (((c >> 1) ^ s_row(*row)) << 1) | (c & 1);
      else *chunk = c;
    }
  }

  // where this lane's fragments begin
  __device__ __forceinline__ void place_reads(int row0, int lane, uint32_t base) {
    if constexpr (!T) {
      const int r = row0 + (lane & 15);
#pragma unroll
      for (int k = 0; k < KS; ++k) rd[k] = base + r * (64 * KS) + ((4 * k + (lane >> 4)) ^ f_row(r)) * 16;
    } else if constexpr (E::kSize == 2) {
      const int i = lane & 15, k = (lane >> 4) * 8 + (i >> 2);
#pragma unroll
      for (int j = 0; j < kReads; ++j) rd[j] = base + k * (R * 2) + ((row0 / 16 + j) ^ s_row(k)) * 32 + (i & 3) * 8;
    } else {
#pragma unroll
      for (int j = 0; j < kReads; ++j) rd[j] = base + 4 * (lane >> 4) * (R * 4) + (row0 + 16 * j + (lane & 15)) * 4;
    }
  }

  // the fragment of the wave's j-th 16 rows, step ks of the stage at `stage`
  __device__ __forceinline__ u32x4 read(const char* lds, uint32_t stage, int ks, int j) const {
    if constexpr (!T) {
      return *(const u32x4*)(lds + stage + rd[ks] + j * (1024 * KS));
    } else if constexpr (E::kSize == 2) {
      typedef __attribute__((address_space(3))) sw_s4 lds_s4;
      const char* at = lds + stage + rd[j];
      const sw_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)at);
      const sw_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + 4 * (R * 2)));
      const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
      return u32x4{a.x, a.y, b.x, b.y};
    } else {
      const char* at = lds + stage + rd[j];
      u32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *(const uint32_t*)(at + e * (R * 4));
      return v;
    }
  }
};

}  // namespace attnres
