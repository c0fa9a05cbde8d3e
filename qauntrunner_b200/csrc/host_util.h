// host_util.h -- what the operator units (rows.cu, fp8.cu) share on the host:
// error texts, checks of types, pitches and pointers, the device check.
#pragma once
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <atomic>

#include "qrmoe.h"

extern "C" int qrm_set_error(int code, const char* msg);

namespace qrm {

inline int failf(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return qrm_set_error(code, buf);
}

// bytes of one value of an activation type, 0 when `type` is none
inline int type_bytes(int type) { return type == QRM_F32 ? 4 : type == QRM_F16 || type == QRM_BF16 ? 2 : 0; }

// the calling thread's current device, sm_100 or an error; asks the driver
// for the properties once per device
constexpr int kMaxDevices = 64;
inline int current_device(int* device, int* sms) {
    static std::atomic<int> count[kMaxDevices];   // SMs of a device that was looked at
    cudaError_t e = cudaGetDevice(device);
    if (e != cudaSuccess) return failf(QRM_E_CUDA, "no CUDA device: %s", cudaGetErrorString(e));
    if (*device < 0 || *device >= kMaxDevices) return failf(QRM_E_CUDA, "device %d is not supported", *device);
    int n = count[*device].load(std::memory_order_relaxed);
    if (!n) {
        int major = 0;
        if ((e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, *device)) != cudaSuccess ||
            (e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *device)) != cudaSuccess)
            return failf(QRM_E_CUDA, "device %d: %s", *device, cudaGetErrorString(e));
        if (major != 10) return failf(QRM_E_CUDA, "device %d is not sm_100", *device);
        count[*device].store(n, std::memory_order_relaxed);
    }
    *sms = n;
    return QRM_OK;
}

// Makes a device current and the caller's current again at the end: calls that
// have no handle run on the caller's, so a handle's may not change it.
class DeviceGuard {
public:
    DeviceGuard() = default;
    DeviceGuard(const DeviceGuard&) = delete;
    DeviceGuard& operator=(const DeviceGuard&) = delete;
    cudaError_t enter(int device) {
        int now;
        cudaError_t e = cudaGetDevice(&now);
        if (e != cudaSuccess || now == device) return e;
        if ((e = cudaSetDevice(device)) == cudaSuccess) caller_ = now;
        return e;
    }
    ~DeviceGuard() {
        if (caller_ >= 0) cudaSetDevice(caller_);
    }

private:
    int caller_ = -1;   // the device to go back to, if another one is current
};

// a pitch in elements: 0 stands for dense rows
inline bool pitch_ok(int64_t* ld, int64_t cols) {
    if (*ld == 0) *ld = cols;
    return *ld >= cols;
}

inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// A launch whose CTAs may start while the kernel before it in the stream still
// runs (programmatic dependent launch): every kernel of these units begins
// with pdl_start(), which lets the next one start likewise and then waits for
// the one before, in every CTA, so that waiting for a kernel means waiting for
// all that came before it.  Back to back, the launch is hidden behind the other
// kernel's end (combine of 2048 x 6 rows of 4096: 30.2 us in place of 32.5).
template <typename... P, typename... A>
cudaError_t launch_ahead(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream, A&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at = {};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

}  // namespace qrm
