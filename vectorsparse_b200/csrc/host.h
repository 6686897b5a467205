// What the translation units of the library share on the host.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace vs {

// The current device's number of SMs and its status word (vs_device_status); binds the device's primary context to a thread that has none.
int current_device(int *sm_count, uint32_t **status);

// cuTensorMapEncodeTiled, fetched from the driver at first use; null where it cannot be had.
typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                  const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled();

}  // namespace vs
