// C ABI of the paged cache's operators: argument checks and launches.  Declarations are in include/dsdpa.h.
#include <math.h>

#include "dsdpa_cache_launch.h"
#include "dsdpa_evict.cuh"
#include "dsdpa_host.h"

namespace dsdpa {
namespace {

bool bad_v(const dsdpa_cache_problem* p) { return bad_stride(p->stride_v, p->dtype, p->pages, p->Hkv, p->page_size); }

int check(const dsdpa_cache_problem* p) {
    if (!p) return DSDPA_ERR_NULL_POINTER;
    if (p->dtype != DSDPA_F32 && p->dtype != DSDPA_BF16 && p->dtype != DSDPA_F16) return DSDPA_ERR_BAD_DTYPE;
    if (p->D < 8 || p->D > 256 || p->D % 8) return DSDPA_ERR_BAD_HEAD_DIM;
    if (p->B <= 0 || p->Hkv <= 0 || p->pages <= 0 || p->page_size <= 0 || p->table_width <= 0) return DSDPA_ERR_BAD_SHAPE;
    if ((long long)p->table_width * p->page_size > (1ll << 30) || (long long)p->B * p->Hkv >= (1ll << 20)) return DSDPA_ERR_BAD_SHAPE;
    if (p->flags) return DSDPA_ERR_BAD_FLAGS;
    return bad_stride(p->stride_k, p->dtype, p->pages, p->Hkv, p->page_size) ? DSDPA_ERR_MISALIGNED : DSDPA_OK;
}
int check_tokens(const dsdpa_cache_problem* p) {
    const int st = check(p);
    if (st != DSDPA_OK) return st;
    if (p->Hq <= 0 || p->Hq % p->Hkv || (long long)p->B * p->Hq >= (1ll << 24) || p->T <= 0) return DSDPA_ERR_BAD_SHAPE;
    if (p->T > kTreeMax) return DSDPA_ERR_TOO_LARGE;
    if (bad_score(p->sm_scale, p->softcap)) return DSDPA_ERR_BAD_SHAPE;
    return bad_stride(p->stride_q, p->dtype, p->B, p->Hq, p->T) ? DSDPA_ERR_MISALIGNED : DSDPA_OK;
}
bool odd4(const void* p) { return ((uintptr_t)p & 3) != 0; }
bool odd_tree(const dsdpa_cache_tree* t) {
    return t && (odd4(t->parents) || odd4(t->drafted) || odd4(t->positions) || odd4(t->start) || odd4(t->slopes));
}

CacheParams params(const dsdpa_cache_problem& p, const dsdpa_cache_tree* t, const void* q, const void* k, const void* v,
                   const int* table, const int* lens, int* err) {
    CacheParams c{};
    c.q = q; c.k = k; c.v = v; c.table = table; c.lens = lens;
    if (t) { c.parents = t->parents; c.drafted = t->drafted; c.positions = t->positions; c.start = t->start; c.slopes = t->slopes; }
    c.B = p.B; c.Hq = p.Hq; c.Hkv = p.Hkv; c.group = p.Hq / p.Hkv; c.T = p.T; c.D = p.D;
    c.pages = p.pages; c.page_size = p.page_size; c.width = p.table_width; c.slots = p.slots;
    c.sm_scale = p.sm_scale;
    c.cap = p.softcap > 0.0f ? p.softcap : 0.0f;
    for (int i = 0; i < 3; ++i) { c.sq[i] = p.stride_q[i]; c.sk[i] = p.stride_k[i]; c.sv[i] = p.stride_v[i]; }
    c.err = err;
    c.div = page_division(p.page_size);
    return c;
}

template <typename T>
cudaError_t tree_forward(const dsdpa_cache_problem& problem, const CacheParams& p, void* workspace, cudaStream_t s) {
    const TreePlan t = plan_tree(problem);
    if constexpr (DtypeOf<T>::value != DSDPA_F32)
        if (cache_on_tensor_cores(problem))
            return cache_few_rows(problem) ? launch_tree_few<T>(p, t, workspace, s) : launch_tree_tc<T>(p, t, workspace, s);
    if constexpr (DtypeOf<T>::value == DSDPA_F32)
        if (cache_few_f32(problem)) return launch_tree_few_f32(p, t, workspace, s);
    return launch_tree_simt<T>(p, t, workspace, s);
}
template <typename T>
cudaError_t weights_add(const dsdpa_cache_problem& problem, const CacheParams& p, cudaStream_t s) {
    const TreePlan t = plan_tree(problem);
    if constexpr (DtypeOf<T>::value != DSDPA_F32)
        if (cache_on_tensor_cores(problem)) return cache_few_rows(problem) ? launch_weights_few<T>(p, t, s) : launch_weights_tc<T>(p, t, s);
    if constexpr (DtypeOf<T>::value == DSDPA_F32)
        if (cache_few_f32(problem)) return launch_weights_few_f32(p, t, s);
    return launch_weights_simt<T>(p, t, s);
}

}  // namespace
}  // namespace dsdpa

using namespace dsdpa;

extern "C" {

size_t dsdpa_tree_workspace_bytes(const dsdpa_cache_problem* p) {
    return check_tokens(p) == DSDPA_OK ? plan_tree(*p).bytes : 0;
}

int dsdpa_tree_forward(const dsdpa_cache_problem* p, const dsdpa_cache_tree* tree, const void* q, const void* k_pages,
                       const void* v_pages, const int* page_table, const int* lens, void* out, float* lse,
                       void* workspace, size_t workspace_bytes, int device, void* stream) {
    const int st = check_tokens(p);
    if (st != DSDPA_OK) return st;
    if (!q || !k_pages || !v_pages || !page_table || !lens || !out || !lse) return DSDPA_ERR_NULL_POINTER;
    if (misaligned(q) || misaligned(k_pages) || misaligned(v_pages) || misaligned(out) || misaligned(workspace) ||
        odd4(page_table) || odd4(lens) || odd4(lse) || odd_tree(tree) || bad_v(p))
        return DSDPA_ERR_MISALIGNED;
    if (tree && tree->positions && p->slots < p->table_width * p->page_size) return DSDPA_ERR_BAD_SHAPE;
    const size_t need = dsdpa_tree_workspace_bytes(p);
    if (need > 0 && (!workspace || workspace_bytes < need)) return DSDPA_ERR_WORKSPACE;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return report_cuda_failure(guard.err);
    int* err = nullptr;
    cudaError_t e = device_error_word(device, &err);
    if (e != cudaSuccess) return report_cuda_failure(e);
    CacheParams c = params(*p, tree, q, k_pages, v_pages, page_table, lens, err);
    c.out = out;
    c.lse = lse;
    switch (p->dtype) {
        case DSDPA_F32: e = tree_forward<float>(*p, c, workspace, (cudaStream_t)stream); break;
        case DSDPA_BF16: e = tree_forward<__nv_bfloat16>(*p, c, workspace, (cudaStream_t)stream); break;
        default: e = tree_forward<__half>(*p, c, workspace, (cudaStream_t)stream); break;
    }
    return e == cudaSuccess ? DSDPA_OK : report_cuda_failure(e);
}

int dsdpa_cache_weights(const dsdpa_cache_problem* p, const dsdpa_cache_tree* tree, const void* q, const float* lse,
                        const void* k_pages, const int* page_table, const int* lens, const unsigned char* take,
                        float* weights, int device, void* stream) {
    const int st = check_tokens(p);
    if (st != DSDPA_OK) return st;
    if (!q || !lse || !k_pages || !page_table || !lens || !weights) return DSDPA_ERR_NULL_POINTER;
    if (misaligned(q) || misaligned(k_pages) || odd4(lse) || odd4(page_table) || odd4(lens) || odd4(weights) || odd_tree(tree))
        return DSDPA_ERR_MISALIGNED;
    if (p->slots < p->table_width * p->page_size) return DSDPA_ERR_BAD_SHAPE;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return report_cuda_failure(guard.err);
    int* err = nullptr;
    cudaError_t e = device_error_word(device, &err);
    if (e != cudaSuccess) return report_cuda_failure(e);
    CacheParams c = params(*p, tree, q, k_pages, nullptr, page_table, lens, err);
    c.lse = const_cast<float*>(lse);
    c.take = take;
    c.weights = weights;
    switch (p->dtype) {
        case DSDPA_F32: e = weights_add<float>(*p, c, (cudaStream_t)stream); break;
        case DSDPA_BF16: e = weights_add<__nv_bfloat16>(*p, c, (cudaStream_t)stream); break;
        default: e = weights_add<__half>(*p, c, (cudaStream_t)stream); break;
    }
    return e == cudaSuccess ? DSDPA_OK : report_cuda_failure(e);
}

int dsdpa_cache_evict(const dsdpa_cache_problem* p, void* k_pages, void* v_pages, const int* page_table, const int* lens,
                      const float* weights, const int* positions, int keep, int sinks, int recent,
                      const int* out_table, int out_width, int* kept, int* new_lens, float* new_weights,
                      int* new_positions, int device, void* stream) {
    const int st = check(p);
    if (st != DSDPA_OK) return st;
    if (!k_pages || !v_pages || !page_table || !lens || !weights || !out_table || !kept || !new_lens || !new_weights)
        return DSDPA_ERR_NULL_POINTER;
    if (new_weights == weights || (new_positions && new_positions == positions)) return DSDPA_ERR_BAD_SHAPE;
    if (misaligned(k_pages) || misaligned(v_pages) || odd4(page_table) || odd4(lens) || odd4(weights) || odd4(positions) ||
        odd4(out_table) || odd4(kept) || odd4(new_lens) || odd4(new_weights) || odd4(new_positions) || bad_v(p))
        return DSDPA_ERR_MISALIGNED;
    if (p->slots < p->table_width * p->page_size || keep <= 0 || sinks < 0 || recent < 0 || sinks > keep || recent > keep - sinks)
        return DSDPA_ERR_BAD_SHAPE;
    // the kept keys have to find room in out_table, and in a row of weights
    if (out_width <= 0 || (long long)out_width * p->page_size > (1ll << 30)) return DSDPA_ERR_BAD_SHAPE;
    const long long most = (long long)p->table_width * p->page_size < keep ? (long long)p->table_width * p->page_size : keep;
    if ((long long)out_width * p->page_size < most) return DSDPA_ERR_BAD_SHAPE;
    if (new_lens == lens) return DSDPA_ERR_BAD_SHAPE;      // the blocks of a sequence's other heads still read it
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return report_cuda_failure(guard.err);
    int* err = nullptr;
    cudaError_t e = device_error_word(device, &err);
    if (e != cudaSuccess) return report_cuda_failure(e);
    const int es = p->dtype == DSDPA_F32 ? 4 : 2;
    EvictParams v{};
    v.k = (char*)k_pages; v.v = (char*)v_pages;
    v.table = page_table; v.lens = lens; v.positions = positions; v.out_table = out_table; v.weights = weights;
    v.kept = kept; v.new_lens = new_lens; v.new_positions = new_positions; v.new_weights = new_weights;
    v.B = p->B; v.Hkv = p->Hkv; v.pages = p->pages; v.page_size = p->page_size; v.width = p->table_width;
    v.out_width = out_width; v.slots = p->slots; v.keep = keep; v.sinks = sinks; v.recent = recent;
    v.row_bytes = p->D * es;
    for (int i = 0; i < 3; ++i) { v.sk[i] = p->stride_k[i] * es; v.sv[i] = p->stride_v[i] * es; }
    v.err = err;
    cudaStream_t s = (cudaStream_t)stream;
    v.div = page_division(p->page_size);
    // up to 32768 ranks (128 KB) beside the histograms
    const int room = p->table_width * p->page_size;
    v.held = room < 32768 ? room : 32768;
    static SmemOnce once;
    if ((e = allow_smem(evict_select_kernel, 32768 * 4, once)) != cudaSuccess)
        return report_cuda_failure(e);
    evict_select_kernel<<<(unsigned)(p->B * p->Hkv), kSelectThreads, (size_t)v.held * 4, s>>>(v);
    if ((e = cudaGetLastError()) != cudaSuccess) return report_cuda_failure(e);
    // Whole rows where that gives every SM two blocks, narrower pieces (64 bytes at least, two sectors) where not:
    // 16 caches x 8 heads of 256-byte rows take 132 us whole (256 blocks), 100 us in halves, 109 us in quarters.
    int width = 1, slices = 1;
    while (width * 16 < v.row_bytes) width *= 2;
    while (width > 4 && (long long)p->B * p->Hkv * 2 * slices < kSMs * 2) width /= 2, slices = (v.row_bytes + width * 16 - 1) / (width * 16);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(p->B * p->Hkv * 2 * slices));
    cfg.blockDim = dim3(kMoveThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if ((e = cudaLaunchKernelEx(&cfg, evict_move_kernel, v, width, slices)) != cudaSuccess) return report_cuda_failure(e);
    count_launches(2);
    return DSDPA_OK;
}

}  // extern "C"
