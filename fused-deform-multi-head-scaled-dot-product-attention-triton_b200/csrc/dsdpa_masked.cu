// C ABI of masked attention: argument checks and launches.  Declarations are in include/dsdpa.h.
#include <cudaTypedefs.h>
#include <math.h>

#include <atomic>

#include "dsdpa_host.h"
#include "dsdpa_masked.cuh"
#include "dsdpa_masked_launch.h"

namespace dsdpa {

cudaError_t tensor_map_16(CUtensorMap* map, int dtype, const void* base, int D, int rows, int L, int H, int B, const long long (&stride)[3]) {
    // a driver call, reached through the runtime: the library links no driver library
    static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> known{ nullptr };
    PFN_cuTensorMapEncodeTiled_v12000 encode = known.load(std::memory_order_relaxed);
    if (!encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found);
        if (e != cudaSuccess) return e;
        if (!fn || found != cudaDriverEntryPointSuccess) return cudaErrorNotSupported;
        encode = (PFN_cuTensorMapEncodeTiled_v12000)fn;
        known.store(encode, std::memory_order_relaxed);
    }
    const cuuint64_t dims[4] = { (cuuint64_t)D, (cuuint64_t)L, (cuuint64_t)H, (cuuint64_t)B };
    const cuuint64_t strides[3] = { L > 1 ? (cuuint64_t)stride[2] * 2 : 16, H > 1 ? (cuuint64_t)stride[1] * 2 : 16,
                                    B > 1 ? (cuuint64_t)stride[0] * 2 : 16 };
    const cuuint32_t box[4] = { 64, (cuuint32_t)rows, 1, 1 }, step[4] = { 1, 1, 1, 1 };
    auto call = [&]() {
        return encode(map, dtype == DSDPA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base),
                      dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = call();
    if (r != CUDA_SUCCESS) {
        // a driver call wants the device's context bound to the thread, which the runtime does only when it has to: a
        // thread that an autograd engine has just started may come here first
        int device = 0;
        cudaError_t e;
        if ((e = cudaGetDevice(&device)) != cudaSuccess || (e = cudaSetDevice(device)) != cudaSuccess) return e;
        r = call();
    }
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

namespace {

int check(const dsdpa_masked_problem* p) {
    if (!p) return DSDPA_ERR_NULL_POINTER;
    if (p->dtype != DSDPA_F32 && p->dtype != DSDPA_BF16 && p->dtype != DSDPA_F16) return DSDPA_ERR_BAD_DTYPE;
    if (p->D < 8 || p->D > 256 || p->D % 8) return DSDPA_ERR_BAD_HEAD_DIM;
    if (p->B <= 0 || p->Hq <= 0 || p->Hkv <= 0 || p->Hq % p->Hkv || p->Lq < 0 || p->Lk < 0) return DSDPA_ERR_BAD_SHAPE;
    // positions are exact in fp32 and tile counts fit the grid
    if (p->Lq > (1 << 24) || p->Lk > (1 << 24) || (long long)p->B * p->Hq >= (1ll << 24)) return DSDPA_ERR_BAD_SHAPE;
    if (p->flags & ~DSDPA_MASKED_CAUSAL) return DSDPA_ERR_BAD_FLAGS;
    if (bad_score(p->sm_scale, p->softcap)) return DSDPA_ERR_BAD_SHAPE;
    return DSDPA_OK;
}

bool bad_q(const long long (&st)[3], const dsdpa_masked_problem* p) { return bad_stride(st, p->dtype, p->B, p->Hq, p->Lq); }
bool bad_k(const long long (&st)[3], const dsdpa_masked_problem* p) { return bad_stride(st, p->dtype, p->B, p->Hkv, p->Lk); }

MaskedParams params(const dsdpa_masked_problem& p, const void* q, const void* k, const void* v, const int* visible,
                    const float* slopes, int* err) {
    MaskedParams m{};
    m.q = q; m.k = k; m.v = v;
    m.visible = (const int2*)visible;
    m.slopes = slopes;
    m.B = p.B; m.Hq = p.Hq; m.Hkv = p.Hkv; m.group = p.Hq / p.Hkv; m.Lq = p.Lq; m.Lk = p.Lk; m.D = p.D;
    m.causal = (p.flags & DSDPA_MASKED_CAUSAL) != 0;
    m.sm_scale = p.sm_scale;
    m.cap = p.softcap > 0.0f ? p.softcap : 0.0f;
    m.s_visible = p.stride_visible / 2;
    m.err = err;
    for (int i = 0; i < 3; ++i) {
        m.sq[i] = p.stride_q[i]; m.sk[i] = p.stride_k[i]; m.sv[i] = p.stride_v[i];
        m.so[i] = p.stride_out[i]; m.sdo[i] = p.stride_dout[i];
        m.sdq[i] = p.stride_dq[i]; m.sdk[i] = p.stride_dk[i]; m.sdv[i] = p.stride_dv[i];
    }
    return m;
}

// The tensor-core kernels take 16-bit storage with up to 128 elements a row; fp32 arithmetic the rest.
template <typename T>
bool on_tensor_cores(const MaskedParams& p) {
    return DtypeOf<T>::value != DSDPA_F32 && p.D <= 128 && p.Lq > 0 && p.Lk > 0;
}

template <typename T>
cudaError_t forward(const MaskedParams& p, cudaStream_t s) {
    if constexpr (DtypeOf<T>::value != DSDPA_F32)
        if (on_tensor_cores<T>(p)) return launch_masked_fwd_tc<T>(p, s);
    return launch_masked_fwd_simt<T>(p, s);
}

template <typename T>
cudaError_t backward(const MaskedParams& p, void* workspace, cudaStream_t s) {
    if constexpr (DtypeOf<T>::value != DSDPA_F32)
        if (on_tensor_cores<T>(p)) return launch_masked_bwd_tc<T>(p, workspace, s);
    return launch_masked_bwd_simt<T>(p, s);
}

size_t backward_bytes(const dsdpa_masked_problem& p) {
    const MaskedBwdSpace w = masked_bwd_space(p.B, p.Hq, p.Lq);
    return p.dtype != DSDPA_F32 && p.D <= 128 ? w.bytes : w.stats;
}

}  // namespace
}  // namespace dsdpa

using namespace dsdpa;

extern "C" {

int dsdpa_masked_forward(const dsdpa_masked_problem* p, const void* q, const void* k, const void* v, const int* visible,
                         const float* slopes, void* out, float* lse, int device, void* stream) {
    int st = check(p);
    if (st != DSDPA_OK) return st;
    if (p->Lq == 0) return DSDPA_OK;
    if (!q || !out || !lse || (p->Lk > 0 && (!k || !v))) return DSDPA_ERR_NULL_POINTER;
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(out) || ((uintptr_t)visible & 7) ||
        ((uintptr_t)lse & 3) || ((uintptr_t)slopes & 3))
        return DSDPA_ERR_MISALIGNED;
    if (bad_q(p->stride_q, p) || bad_k(p->stride_k, p) || bad_k(p->stride_v, p) || bad_q(p->stride_out, p) || p->stride_visible % 2)
        return DSDPA_ERR_MISALIGNED;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return report_cuda_failure(guard.err);
    int* err = nullptr;
    cudaError_t e = device_error_word(device, &err);
    if (e != cudaSuccess) return report_cuda_failure(e);
    MaskedParams m = params(*p, q, k, v, visible, slopes, err);
    m.out = out;
    m.lse = lse;
    switch (p->dtype) {
        case DSDPA_F32: e = forward<float>(m, (cudaStream_t)stream); break;
        case DSDPA_BF16: e = forward<__nv_bfloat16>(m, (cudaStream_t)stream); break;
        default: e = forward<__half>(m, (cudaStream_t)stream); break;
    }
    return e == cudaSuccess ? DSDPA_OK : report_cuda_failure(e);
}

size_t dsdpa_masked_backward_workspace_bytes(const dsdpa_masked_problem* p) {
    return check(p) == DSDPA_OK ? backward_bytes(*p) : 0;
}

int dsdpa_masked_backward(const dsdpa_masked_problem* p, const void* q, const void* k, const void* v, const int* visible,
                          const float* slopes, const void* out, const float* lse, const void* dout, void* dq, void* dk,
                          void* dv, void* workspace, size_t workspace_bytes, int device, void* stream) {
    int st = check(p);
    if (st != DSDPA_OK) return st;
    if (p->Lq == 0 && p->Lk == 0) return DSDPA_OK;
    if ((p->Lq > 0 && (!q || !out || !lse || !dout || !dq)) || (p->Lk > 0 && (!k || !v || !dk || !dv)))
        return DSDPA_ERR_NULL_POINTER;
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(out) || misaligned(dout) || misaligned(dq) ||
        misaligned(dk) || misaligned(dv) || misaligned(workspace) || ((uintptr_t)visible & 7) || ((uintptr_t)lse & 3) ||
        ((uintptr_t)slopes & 3))
        return DSDPA_ERR_MISALIGNED;
    if (bad_q(p->stride_q, p) || bad_k(p->stride_k, p) || bad_k(p->stride_v, p) || bad_q(p->stride_out, p) || bad_q(p->stride_dout, p) ||
        bad_q(p->stride_dq, p) || bad_k(p->stride_dk, p) || bad_k(p->stride_dv, p) || p->stride_visible % 2)
        return DSDPA_ERR_MISALIGNED;
    const size_t need = dsdpa_masked_backward_workspace_bytes(p);
    if (need > 0 && (!workspace || workspace_bytes < need)) return DSDPA_ERR_WORKSPACE;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return report_cuda_failure(guard.err);
    int* err = nullptr;
    cudaError_t e = device_error_word(device, &err);
    if (e != cudaSuccess) return report_cuda_failure(e);
    MaskedParams m = params(*p, q, k, v, visible, slopes, err);
    m.out_in = out; m.lse = (float*)lse; m.dout = dout;
    m.dq = dq; m.dk = dk; m.dv = dv;
    m.delta = (float*)workspace;
    switch (p->dtype) {
        case DSDPA_F32: e = backward<float>(m, workspace, (cudaStream_t)stream); break;
        case DSDPA_BF16: e = backward<__nv_bfloat16>(m, workspace, (cudaStream_t)stream); break;
        default: e = backward<__half>(m, workspace, (cudaStream_t)stream); break;
    }
    return e == cudaSuccess ? DSDPA_OK : report_cuda_failure(e);
}

}  // extern "C"
