// ops_host.cpp — error text, launch accounting and the per-device error word.
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdio.h>

#include <atomic>
#include <mutex>

#include "ops_common.cuh"

namespace cailops {

namespace {
thread_local char t_error[512] = "";
std::atomic<unsigned long long> g_launches{0};
constexpr int kMaxDevices = 64;
constexpr int kSms = 148;  // of a B200
std::atomic<int> g_sms[kMaxDevices];
std::mutex g_flag_mutex;
std::atomic<int *> g_flag_host[kMaxDevices];
std::atomic<int *> g_flag_dev[kMaxDevices];
}  // namespace

int fail(int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(t_error, sizeof t_error, fmt, ap);
    va_end(ap);
    return code;
}

int launched(const char *what) {
    g_launches.fetch_add(1, std::memory_order_relaxed);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(CAIL_OPS_ECUDA, "%s: %s", what, cudaGetErrorString(e));
    return CAIL_OPS_OK;
}

int sm_count() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        return kSms;
    }
    const bool kept = dev >= 0 && dev < kMaxDevices;
    if (kept) n = g_sms[dev].load(std::memory_order_relaxed);
    if (n > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) {
        cudaGetLastError();
        return kSms;
    }
    if (kept) g_sms[dev].store(n, std::memory_order_relaxed);
    return n;
}

int earlier_error(const char *who) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return CAIL_OPS_OK;
    volatile int *h = g_flag_host[dev].load(std::memory_order_acquire);
    if (!h || *h == 0) return CAIL_OPS_OK;
    *h = 0;
    return fail(CAIL_OPS_ECUDA, "%s: a kernel of an earlier call gave up waiting for its data; that call's results are wrong", who);
}

// One mapped host word per device: a kernel whose bounded wait ran out stores
// there, and the host reads it without touching the device.  Made on first
// use; the allocation is legal while another stream of this thread is being
// captured only in relaxed capture mode, hence the exchange around it.
int *device_error_flag() {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return nullptr;
    int *p = g_flag_dev[dev].load(std::memory_order_acquire);
    if (p) return p;
    std::lock_guard<std::mutex> lock(g_flag_mutex);
    p = g_flag_dev[dev].load(std::memory_order_acquire);
    if (p) return p;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
    void *h = nullptr, *d = nullptr;
    cudaError_t e = cudaHostAlloc(&h, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable);
    if (e == cudaSuccess) e = cudaHostGetDevicePointer(&d, h, 0);
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) {
        if (h) cudaFreeHost(h);
        cudaGetLastError();
        return nullptr;
    }
    *static_cast<volatile int *>(h) = 0;
    g_flag_host[dev].store(static_cast<int *>(h), std::memory_order_release);
    g_flag_dev[dev].store(static_cast<int *>(d), std::memory_order_release);
    return static_cast<int *>(d);
}

}  // namespace cailops

extern "C" const char *cail_ops_last_error(void) { return cailops::t_error; }

extern "C" unsigned long long cail_ops_launches(void) { return cailops::g_launches.load(); }

extern "C" int *cail_ops_device_error_word(int device) {
    if (device < 0 || device >= cailops::kMaxDevices) return nullptr;
    return cailops::g_flag_host[device].load();
}
