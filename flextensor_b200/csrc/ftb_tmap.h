// Tensor maps of the TMA copies, shared by the launchers (defined in ftb_gemm.cu).
#pragma once
#include <cuda.h>
#include <stdint.h>

namespace ftb {

// rank-`rank` tiled map (128-byte swizzle unless told otherwise); strides in bytes for dims 1..rank-1.
int make_tmap(CUtensorMap* map, CUtensorMapDataType dt, int rank, const void* base, const uint64_t* dims,
              const uint64_t* strides_bytes, const uint32_t* box, const uint32_t* elem_strides,
              CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B);

}  // namespace ftb
