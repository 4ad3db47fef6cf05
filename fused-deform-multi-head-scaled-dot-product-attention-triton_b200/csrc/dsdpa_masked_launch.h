// Host side of the tensor-core kernels of masked attention: tensor maps and launches.
#pragma once

#include <cuda.h>

#include "dsdpa_host.h"
#include "dsdpa_masked.cuh"

namespace dsdpa {

// A tensor map of a [batch][head][row][D] tensor of 16-bit elements whose boxes are `rows` rows of 64 elements,
// swizzled by 128 bytes; what lies outside reads as zero.
cudaError_t tensor_map_16(CUtensorMap* map, int dtype, const void* base, int D, int rows, int L, int H, int B, const long long (&stride)[3]);

template <typename T> cudaError_t launch_masked_fwd_tc(const MaskedParams& p, cudaStream_t s);

}  // namespace dsdpa
