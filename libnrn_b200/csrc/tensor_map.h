// tensor_map.h -- the driver's encoder of TMA tensor maps, found through the
// runtime (no link against the driver library).
#pragma once
#include <cuda.h>

namespace nrn {

using TensorMapEncode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                     const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                     CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// Null where the driver has none.
TensorMapEncode tensor_map_encode();

}  // namespace nrn
