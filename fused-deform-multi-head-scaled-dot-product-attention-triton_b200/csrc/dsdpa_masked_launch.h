// Host side of masked attention's kernels: tensor maps and launches.
#pragma once

#include <cuda.h>

#include "dsdpa_host.h"
#include "dsdpa_masked.cuh"

namespace dsdpa {

// A tensor map of a [batch][head][row][D] tensor of 16-bit elements whose boxes are `rows` rows of 64 elements,
// swizzled by 128 bytes; what lies outside reads as zero.
cudaError_t tensor_map_16(CUtensorMap* map, int dtype, const void* base, int D, int rows, int L, int H, int B, const long long (&stride)[3]);

template <typename T> cudaError_t launch_masked_fwd_tc(const MaskedParams& p, cudaStream_t s);
// workspace: masked_bwd_space().bytes, p.delta pointing to its start; p.Lq > 0 and p.Lk > 0
template <typename T> cudaError_t launch_masked_bwd_tc(const MaskedParams& p, void* workspace, cudaStream_t s);

// fp32 arithmetic; p.Lq or p.Lk may be 0, p.delta is the backward's workspace
template <typename T> cudaError_t launch_masked_fwd_simt(const MaskedParams& p, cudaStream_t s);
template <typename T> cudaError_t launch_masked_bwd_simt(const MaskedParams& p, cudaStream_t s);

// Byte offsets in the backward's workspace: delta at 0, then what the tensor-core kernels pass on.
struct MaskedBwdSpace {
    size_t stats, ranges, tiles, amax, bytes;
    int n;          // tiles of 128 queries
};
inline MaskedBwdSpace masked_bwd_space(int B, int Hq, int Lq) {
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    MaskedBwdSpace w{};
    w.n = (Lq + 127) / 128;
    w.stats = up((size_t)B * Hq * Lq * 4);
    w.ranges = w.stats + up((size_t)B * Hq * w.n * 128 * 8);
    w.tiles = w.ranges + up((size_t)B * w.n * 128 * 8);
    w.amax = w.tiles + up((size_t)B * w.n * 16);
    w.bytes = w.amax + up((size_t)B * Hq * w.n * 4);
    return w;
}

}  // namespace dsdpa
