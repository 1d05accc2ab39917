#define ATTNRES_CACHE_ATTEND_KERNELS
#include "attnres_cache_attend.h"

namespace attnres {
hipError_t launch_cache_attend_f16(const CacheAttendParams& p, hipStream_t st) { return run_attend_type<F16>(p, st); }
}  // namespace attnres
