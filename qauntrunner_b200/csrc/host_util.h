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

// a pitch in elements: 0 stands for dense rows
inline bool pitch_ok(int64_t* ld, int64_t cols) {
    if (*ld == 0) *ld = cols;
    return *ld >= cols;
}

inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

inline int launched(const char* what) {
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? QRM_OK : failf(QRM_E_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

}  // namespace qrm
