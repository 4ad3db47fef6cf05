// The few-row kernels over a cache of fp32.
#include "dsdpa_few_f32.cuh"
#include "dsdpa_host.h"
#include "dsdpa_share_launch.cuh"

namespace dsdpa {
namespace {

template <int HD, int NC>
cudaError_t tree(const CacheParams& p, const TreePlan& t, const TreeSplit& sp, cudaStream_t s) {
    tree_few_f32_kernel<HD, NC><<<t.blocks, kF32Warps * 32, 0, s>>>(p, sp);
    count_launches(1);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess ? e : launch_combine<float, F32Tile>(p, t, sp, s);
}
template <int HD, int NC>
cudaError_t weights(const CacheParams& p, const TreePlan& t, cudaStream_t s) {
    const TreeSplit sp{ 0, 1, 0, nullptr, nullptr, nullptr, 0 };
    weights_few_f32_kernel<HD, NC><<<t.weight_blocks, kF32Warps * 32, 0, s>>>(p, sp);
    count_launches(1);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_tree_few_f32(const CacheParams& p, const TreePlan& t, void* workspace, cudaStream_t s) {
    const TreeSplit sp = tree_split(t, workspace);
    const bool four = t.part_rows <= 4;
    if (p.D <= 32) return four ? tree<32, 1>(p, t, sp, s) : tree<32, 2>(p, t, sp, s);
    if (p.D <= 64) return four ? tree<64, 1>(p, t, sp, s) : tree<64, 2>(p, t, sp, s);
    return four ? tree<128, 1>(p, t, sp, s) : tree<128, 2>(p, t, sp, s);
}
cudaError_t launch_weights_few_f32(const CacheParams& p, const TreePlan& t, cudaStream_t s) {
    const bool four = t.part_rows <= 4;
    if (p.D <= 32) return four ? weights<32, 1>(p, t, s) : weights<32, 2>(p, t, s);
    if (p.D <= 64) return four ? weights<64, 1>(p, t, s) : weights<64, 2>(p, t, s);
    return four ? weights<128, 1>(p, t, s) : weights<128, 2>(p, t, s);
}

}  // namespace dsdpa
