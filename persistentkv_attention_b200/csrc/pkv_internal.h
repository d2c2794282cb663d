// pkv_internal.h -- what the translation units of the library share: error
// reporting into the thread-local message and the current device's state
// (both defined in pkv_api.cu).
#pragma once

#include <cuda.h>

#include "../../include/pkv_b200.h"

namespace pkv_internal {

// printf-style error reporting into the thread-local message of pkv_api.cu.
pkv_status fail_fmt(pkv_status st, const char* fmt, ...);
pkv_status ok();

// SM count and error word of the current device, which must be an sm_100 one.
pkv_status device_state(int* sm_count, unsigned** error_word);

// cuTensorMapEncodeTiled, reached at run time; null where it is unavailable.
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled();

}  // namespace pkv_internal
