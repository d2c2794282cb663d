// pkv_internal.h -- what the translation units of the library share: error
// reporting into the thread-local message and the current device's state
// (both defined in pkv_api.cu).
#pragma once

#include "../../include/pkv_b200.h"

namespace pkv_internal {

// printf-style error reporting into the thread-local message of pkv_api.cu.
pkv_status fail_fmt(pkv_status st, const char* fmt, ...);
pkv_status ok();

// SM count and error word of the current device, which must be an sm_100 one.
pkv_status device_state(int* sm_count, unsigned** error_word);

}  // namespace pkv_internal
