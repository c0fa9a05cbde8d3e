// A CUDA runtime of two devices for tests of the host code (no GPU): the
// functions that the units rows.cu and fp8.cu call, on host memory.  It keeps a
// log of what happened on which device.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime_api.h>
#include <stdlib.h>
#include <string.h>

#include <map>
#include <string>

namespace {
constexpr int kDevices = 2;
int current = 0, fail_malloc = 0;
std::string events, error;
std::map<const void*, int> owner;   // allocations, and pointers that a test gave to a device
void note(const char* what, int device) { events += std::string(what) + " " + std::to_string(device) + "\n"; }
CUresult encode(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                CUtensorMapFloatOOBfill) {
    return CUDA_SUCCESS;
}
}  // namespace

namespace qrm {
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() { return encode; }
}  // namespace qrm

extern "C" {
// what a test asks and sets
void fake_reset(int device) {
    current = device;
    fail_malloc = 0;
    events.clear();
}
int fake_current() { return current; }
const char* fake_events() { return events.c_str(); }
void fake_fail_malloc() { fail_malloc = 1; }
void fake_place(const void* p, int device) { owner[p] = device; }
int qrm_set_error(int code, const char* msg) {
    error = msg;
    return code;
}
const char* qrm_last_error() { return error.c_str(); }

// the runtime
void** __cudaRegisterFatBinary(void*) {
    static void* handle;
    return &handle;
}
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, void*, void*, void*, void*, int*) {}
void __cudaRegisterVar(void**, char*, char*, const char*, int, size_t, int, int) {}
unsigned __cudaPopCallConfiguration(void*, void*, size_t*, void*) { return 0; }
cudaError_t cudaGetDeviceCount(int* n) {
    *n = kDevices;
    return cudaSuccess;
}
cudaError_t cudaGetDevice(int* d) {
    *d = current;
    return cudaSuccess;
}
cudaError_t cudaSetDevice(int d) {
    if (d < 0 || d >= kDevices) return cudaErrorInvalidDevice;
    current = d;
    return cudaSuccess;
}
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr a, int) {
    *v = a == cudaDevAttrComputeCapabilityMajor ? 10 : 4;   // 4 SMs
    return cudaSuccess;
}
cudaError_t cudaDeviceSynchronize() {
    note("synchronise", current);
    return cudaSuccess;
}
cudaError_t cudaMalloc(void** p, size_t n) {
    if (fail_malloc) return cudaErrorMemoryAllocation;
    *p = aligned_alloc(256, (n + 255) / 256 * 256);
    owner[*p] = current;
    note("allocate", current);
    return cudaSuccess;
}
cudaError_t cudaFree(void* p) {
    if (p) note("free", current);
    owner.erase(p);
    free(p);
    return cudaSuccess;
}
cudaError_t cudaPointerGetAttributes(cudaPointerAttributes* a, const void* p) {
    memset(a, 0, sizeof *a);
    auto at = owner.find(p);
    a->type = at == owner.end() ? cudaMemoryTypeUnregistered : cudaMemoryTypeDevice;
    a->device = at == owner.end() ? -2 : at->second;
    return cudaSuccess;
}
cudaError_t cudaMemcpy(void* to, const void* from, size_t n, cudaMemcpyKind) {
    note("copy", current);
    memcpy(to, from, n);
    return cudaSuccess;
}
cudaError_t cudaMemcpy2D(void* to, size_t ld_to, const void* from, size_t ld_from, size_t width, size_t rows, cudaMemcpyKind) {
    note("copy", current);
    for (size_t i = 0; i < rows; i++) memcpy((char*)to + i * ld_to, (const char*)from + i * ld_from, width);
    return cudaSuccess;
}
cudaError_t cudaMemset(void* p, int v, size_t n) {
    memset(p, v, n);
    return cudaSuccess;
}
cudaError_t cudaMemcpyToSymbol(const void*, const void*, size_t, size_t, cudaMemcpyKind) {
    note("symbol", current);
    return cudaSuccess;
}
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) {
    note("attribute", current);
    return cudaSuccess;
}
cudaError_t cudaFuncGetAttributes(cudaFuncAttributes* a, const void*) {
    memset(a, 0, sizeof *a);
    a->numRegs = 168;
    return cudaSuccess;
}
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "fake"; }
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) {
    note("launch", current);
    return cudaSuccess;
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t*, const void*, void**) {
    note("launch", current);
    return cudaSuccess;
}
}
