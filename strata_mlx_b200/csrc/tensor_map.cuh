// cuTensorMapEncodeTiled for the kernels that copy by TMA.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace sc {

// through the runtime's driver entry point (no link-time dependence on its version); NULL when there is none
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled();

}  // namespace sc
