// tc_host.cpp — tensor maps for the TMA loads of the tensor-core kernels.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "tc.cuh"

namespace cailops {

namespace {
typedef CUresult (*encode_fn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                              const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

encode_fn encoder() {
    static std::atomic<encode_fn> f{nullptr};
    encode_fn e = f.load(std::memory_order_acquire);
    if (e) return e;
    void *p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
        cudaGetLastError();
        return nullptr;
    }
    e = reinterpret_cast<encode_fn>(p);
    f.store(e, std::memory_order_release);
    return e;
}
}  // namespace

bool tma_takes(const cail_ops_bthd &x, int B, int T, int H) {
    auto ok = [](int n, int64_t stride) { return n == 1 || (stride > 0 && (stride * 2) % 16 == 0 && stride * 2 < ((int64_t)1 << 40)); };
    return aligned(x.ptr, 16) && ok(B, x.sb) && ok(T, x.st) && ok(H, x.sh);
}

int tensor_map(CUtensorMap *m, const cail_ops_bthd &x, int type, int B, int T, int H, int D, int rows) {
    encode_fn e = encoder();
    if (!e) return fail(CAIL_OPS_ECUDA, "window attention: cuTensorMapEncodeTiled is not available");
    // the stride of a dimension of one is never used: any legal value
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)T, (cuuint64_t)H, (cuuint64_t)B};
    const cuuint64_t strides[3] = {T == 1 ? 16 : (cuuint64_t)x.st * 2, H == 1 ? 16 : (cuuint64_t)x.sh * 2, B == 1 ? 16 : (cuuint64_t)x.sb * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, steps[4] = {1, 1, 1, 1};
    auto encode = [&] {
        return e(m, type == CAIL_OPS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, x.ptr, dims, strides, box, steps,
                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = encode();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {
        // the first CUDA call of this thread (a thread of autograd's, a user's): setting the device makes its context current
        int device = 0;
        if (cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess) r = encode();
    }
    if (r != CUDA_SUCCESS) return fail(CAIL_OPS_ECUDA, "window attention: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return CAIL_OPS_OK;
}

}  // namespace cailops
