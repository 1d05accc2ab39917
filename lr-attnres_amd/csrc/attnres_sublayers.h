// Internal interface of the sublayer kernels (attnres_qkv_rotary.hip,
// attnres_swiglu*.hip) and their C ABI (attnres_sublayers_capi.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace attnres {

// records the message that attnres_last_error() returns and gives back `code`
int api_fail(int code, const char* fmt, ...);

struct QkvRotaryParams {
  const void* qkv;
  int64_t b_stride, t_stride;
  int64_t n_tok;              // batch * tokens
  int64_t tokens;
  int32_t q_heads, kv_heads, head_dim, qk_norm;
  float eps;
  const void* sin;
  const void* cos;
  int64_t table_rows, table_stride;
  const int64_t* pos;
  int64_t pos_b_stride, pos_t_stride, start;
  void* q;                    // forward
  void* k;
  const void* grad[3];        // backward: dq, dk, dv (null = zero)
  int64_t grad_stride[3][3];  // over batch, heads, tokens
  void* dqkv;
};

// vec: elements of a row per lane (8 / 4 / 2 with accesses of that width, 1 = the
// general kernel); lanes: lanes per head row; chunks: vectors per lane (1 or 2)
hipError_t launch_qkv_rotary(int dtype, bool f32_table, bool bwd, const QkvRotaryParams& p, int vec, int lanes,
                             int chunks, hipStream_t st);

}  // namespace attnres
