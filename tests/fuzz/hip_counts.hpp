// A HIP runtime that only counts, for the library's host code: which code
// objects are loaded when, and what the last launch looked like.
#pragma once
#include <hip/hip_runtime_api.h>

#include <atomic>
#include <cstdio>
#include <cstring>
#include <map>
#include <mutex>
#include <set>
#include <string>
#include <thread>
#include <vector>

#include "vortx_hip.h"

#define IMAGE(n) const unsigned char n[16] = {}, n##_end[1] = {};
extern "C" {
extern const unsigned char vx_co_gemm[16], vx_co_gemm_end[1], vx_co_gemv_q[16], vx_co_gemv_q_end[1], vx_co_copy[16], vx_co_copy_end[1],
    vx_co_quantize[16], vx_co_quantize_end[1], vx_co_gemm_q[16], vx_co_gemm_q_end[1], vx_co_gemm_bf[16], vx_co_gemm_bf_end[1],
    vx_co_attn_d64[16], vx_co_attn_d64_end[1], vx_co_attn_d96[16], vx_co_attn_d96_end[1], vx_co_attn_d128[16], vx_co_attn_d128_end[1],
    vx_co_attn_d256[16], vx_co_attn_d256_end[1];
IMAGE(vx_co_gemm) IMAGE(vx_co_gemv_q) IMAGE(vx_co_copy) IMAGE(vx_co_quantize) IMAGE(vx_co_gemm_q) IMAGE(vx_co_gemm_bf)
IMAGE(vx_co_attn_d64) IMAGE(vx_co_attn_d96) IMAGE(vx_co_attn_d128) IMAGE(vx_co_attn_d256)
}

static std::mutex lock;
static std::map<const void*, int> loads;  // by image
static int live, launches, strict;        // modules; launches; captures that allow stream work only
static unsigned last_grid;
static std::set<hipFunction_t> launched;
static std::atomic<int> fail_after{-1};   // names that resolve before one does not
static std::map<std::string, hipFunction_t> names;
static thread_local int device;
static thread_local hipStreamCaptureMode capture = hipStreamCaptureModeGlobal;

extern "C" {
hipError_t hipGetDeviceCount(int* n) { *n = 2; return hipSuccess; }
hipError_t hipGetDevice(int* d) { *d = device; return hipSuccess; }
hipError_t hipSetDevice(int d) { device = d; return hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
    std::memset((void*)p, 0, sizeof *p);
    std::strcpy(p->gcnArchName, "gfx950");
    p->multiProcessorCount = 256;
    p->sharedMemPerBlock = 65536;
    return hipSuccess;
}
hipError_t hipModuleLoadData(hipModule_t* m, const void* image) {
    std::lock_guard<std::mutex> l(lock);
    if (strict && capture != hipStreamCaptureModeRelaxed) return hipErrorStreamCaptureUnsupported;
    ++loads[image];
    ++live;
    *m = (hipModule_t)const_cast<void*>(image);
    return hipSuccess;
}
hipError_t hipModuleUnload(hipModule_t) {
    std::lock_guard<std::mutex> l(lock);
    --live;
    return hipSuccess;
}
hipError_t hipModuleGetFunction(hipFunction_t* f, hipModule_t m, const char* name) {
    std::lock_guard<std::mutex> l(lock);
    // names of the attention are of the module of their head size, all others of any
    const char* d = std::strstr(name, "_d");
    const bool attention = std::strstr(name, "vx_attn") || std::strstr(name, "vx_kv_");
    const void* at = !attention || !d ? nullptr : !std::strncmp(d, "_d64", 4) ? vx_co_attn_d64 : !std::strncmp(d, "_d96", 4) ? vx_co_attn_d96
                     : !std::strncmp(d, "_d128", 5) ? vx_co_attn_d128 : vx_co_attn_d256;
    if (attention && at != (const void*)m) return hipErrorNotFound;
    if (attention && fail_after.load() >= 0 && fail_after.fetch_sub(1) == 0) return hipErrorNotFound;
    auto& e = names[name];
    if (!e) e = (hipFunction_t)(names.size() * 16);
    *f = e;
    return hipSuccess;
}
hipError_t hipModuleGetGlobal(hipDeviceptr_t* p, size_t* n, hipModule_t, const char*) {
    *p = (hipDeviceptr_t)0x1000;
    *n = VX_NOALLOC_SCRATCH_BYTES;
    return hipSuccess;
}
hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned grid, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned, hipStream_t, void**, void**) {
    std::lock_guard<std::mutex> l(lock);
    ++launches;
    last_grid = grid;
    launched.insert(f);
    return f ? hipSuccess : hipErrorInvalidHandle;
}
hipError_t hipThreadExchangeStreamCaptureMode(hipStreamCaptureMode* m) {
    std::swap(*m, capture);
    return hipSuccess;
}
const char* hipGetErrorString(hipError_t) { return "error"; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t*, unsigned) { return hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipHostFree(void*) { return hipSuccess; }
hipError_t hipHostMalloc(void**, size_t, unsigned) { return hipErrorOutOfMemory; }
hipError_t hipMemcpyAsync(void*, const void*, size_t, hipMemcpyKind, hipStream_t) { return hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t*, unsigned) { return hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t, unsigned) { return hipSuccess; }
}

static int failures;
#define CHECK(c) \
    if (!(c)) std::printf("line %d: %s\n", __LINE__, #c), ++failures
