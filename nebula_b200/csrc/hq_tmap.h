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

// 4-D tensor of 16-bit elements, innermost dimension first; strides of dimensions
// 1..3 in bytes (multiples of 16).  128-byte swizzle, boxes of 64 x rows x 1 x 1.
cudaError_t make_tmap_4d(CUtensorMap* out, const void* base, const uint64_t (&dims)[4], const uint64_t (&strides)[3],
                         uint32_t rows);

}  // namespace hq
