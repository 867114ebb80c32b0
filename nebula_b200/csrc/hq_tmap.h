// hq_tmap.h -- host-side creation of TMA tensor maps (cuTensorMapEncodeTiled),
// fetched through cudaGetDriverEntryPoint so the library needs no libcuda link.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace hq {

// 2-D row-major tensor [outer][inner] of `dt` elements, rows `row_bytes` apart
// (a multiple of 16), box [box_outer][box_inner]; out-of-range boxes read zeros.
cudaError_t make_tmap_2d(CUtensorMap* out, const void* base, CUtensorMapDataType dt, uint64_t inner,
                         uint64_t outer, uint64_t row_bytes, uint32_t box_inner, uint32_t box_outer,
                         CUtensorMapSwizzle swizzle);

// Tensor of 16-bit elements of `rank` (3 to 5) dimensions, innermost first; strides of
// dimensions 1 .. rank - 1 in bytes (multiples of 16).  128-byte swizzle: the box's
// innermost dimension is 64.
cudaError_t make_tmap_16bit(CUtensorMap* out, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                            const uint32_t* box);

}  // namespace hq
