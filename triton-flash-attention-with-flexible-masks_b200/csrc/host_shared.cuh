// Host helpers that the two files with entry points share (defined in api.cu).
#pragma once
#include <cuda.h>

namespace fa {

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled, or null without a driver
EncodeFn encode_fn();
// Limit of one bounded wait inside the kernels, in SM clocks
long long wait_limit_clocks();
// SMs of the current device, or -1
int sm_count();

}  // namespace fa
