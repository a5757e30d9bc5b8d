// Host access to the driver's tensor-map encoder.
#pragma once
#include <cuda.h>

namespace bdion {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn();  // resolved once; raises where the driver has none (gemm.cu)

}  // namespace bdion
