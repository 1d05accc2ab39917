#define ATTNRES_CACHE_ATTEND_KERNELS
#include "attnres_cache_attend.h"

namespace attnres {
hipError_t launch_cache_attend_bf16(const CacheAttendParams& p, hipStream_t st) { return run_attend_type<BF16>(p, st); }
}  // namespace attnres
