// ops_common.cuh — what the language-model kernels share: element types,
// 16-byte vectors, warp reductions, error text and launch accounting.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cail_ops.h"

namespace cailops {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// ------------------------------------------------------------------- host
int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
int launched(const char *what);  // after a launch: counts it, reports a launch error
int sm_count();                  // of the current device; a B200's where none answers (sizes may be asked for without one)
int earlier_error(const char *who);  // fails, once, when a kernel of an earlier call on the current device gave up a wait
int *device_error_flag();        // device address of the current device's error word (nullptr: none could be made)

inline bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline size_t type_size(int type) { return type == CAIL_OPS_F32 ? 4 : 2; }

// whether rows of a [B, T, H, D] array start on multiples of `bytes`
inline bool rows_aligned(const cail_ops_bthd &x, int B, int T, int H, size_t size, size_t bytes) {
    return aligned(x.ptr, bytes) && (B == 1 || (x.sb * (int64_t)size) % (int64_t)bytes == 0) &&
           (T == 1 || (x.st * (int64_t)size) % (int64_t)bytes == 0) &&
           (H == 1 || (x.sh * (int64_t)size) % (int64_t)bytes == 0);
}

#ifdef __CUDACC__
// Launches `groups` clusters of `blocks` blocks side by side in x (cfg gives the
// rest), of fewer where so many do not fit: a process, or a stream's context,
// may have been given a part of the SMs.  Kernels ask for the size they got.
template <typename... P, typename... A>
void launch_clusters(cudaLaunchConfig_t cfg, unsigned groups, int blocks, void (*kernel)(P...), const A &...args) {
    for (;; blocks /= 2) {
        cfg.gridDim.x = groups * (unsigned)blocks;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = (unsigned)blocks, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaErrorInvalidClusterSize || blocks == 1) return;
        cudaGetLastError();
    }
}

// ----------------------------------------------------------------- device
template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// N elements of T as one aligned load or store
template <typename T, int N> struct alignas(sizeof(T) * N) Vec { T v[N]; };

// two floats packed as T2 (first in the low half)
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void unpack2(uint32_t u, float &lo, float &hi, __nv_bfloat16) {
    lo = __uint_as_float(u << 16), hi = __uint_as_float(u & 0xffff0000u);
}
__device__ __forceinline__ void unpack2(uint32_t u, float &lo, float &hi, __half) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u));
    lo = f.x, hi = f.y;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// two floats side by side in one register pair: one instruction for both
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void apart(uint64_t x, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_two(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul_two(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
#endif

}  // namespace cailops
