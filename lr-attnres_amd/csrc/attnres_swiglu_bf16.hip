// Gated feed-forward products, bf16 (attnres_swiglu_gemm.h)
#include "attnres_swiglu_gemm.h"
namespace attnres {
hipError_t launch_swiglu_gemm_bf16(int form, int tile, const SwGemmParams& p, hipStream_t st) {
  return sw_form_pick<BF16>(form, tile, p, st);
}
}  // namespace attnres
