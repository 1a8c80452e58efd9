// The library's host code on a HIP runtime that only counts: which code objects
// are loaded when, by how many threads, and what is left at the end.
#include <hip/hip_runtime_api.h>

#include <atomic>
#include <cstdio>
#include <cstring>
#include <map>
#include <mutex>
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
static std::atomic<int> fail_after{-1};   // names that resolve before one does not
static std::map<std::string, hipFunction_t> names;
static thread_local hipStreamCaptureMode capture = hipStreamCaptureModeGlobal;

extern "C" {
hipError_t hipGetDeviceCount(int* n) { *n = 1; return hipSuccess; }
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
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
hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned, hipStream_t, void**, void**) {
    std::lock_guard<std::mutex> l(lock);
    ++launches;
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

static int total() {
    int n = 0;
    for (auto& e : loads) n += e.second;
    return n;
}
static vx_kv_cache cache_of(uint32_t dim) {
    vx_kv_cache c = {(void*)0x10000, 1u << 30, 4, 16, 2, dim, VX_Q8_0, VX_Q8_0};
    return c;
}
static vx_layout rows_of(uint32_t dim, uint32_t heads) {
    vx_layout l = {};
    l.rank = 3;
    l.size[0] = 3, l.size[1] = heads, l.size[2] = dim;
    l.stride[0] = heads * dim, l.stride[1] = dim, l.stride[2] = 1;
    return l;
}
static int write(vx_ctx ctx, uint32_t dim) {
    const vx_kv_cache c = cache_of(dim);
    const vx_cview v = {(float*)0x100000, rows_of(dim, 2)};
    return vx_kv_write(ctx, nullptr, &c, &v, &v, (const int32_t*)0x2000);
}
static vx_attn_batch batch_of() {
    vx_attn_batch b = {};
    b.table = b.lens = b.starts = (const int32_t*)0x3000;
    b.seqs = 1, b.table_cols = b.table_stride = 4, b.max_queries = 3, b.max_len = 64;
    return b;
}
static int attend(vx_ctx ctx, uint32_t dim, void* ws, uint64_t bytes) {
    const vx_kv_cache c = cache_of(dim);
    const vx_cview q = {(float*)0x100000, rows_of(dim, 4)};
    const vx_mview o = {(float*)0x200000, rows_of(dim, 4)};
    const vx_attn_batch b = batch_of();
    return vx_attention(ctx, nullptr, &o, &q, &c, &b, nullptr, ws, bytes);
}

int main() {
    vx_ctx ctx = nullptr;
    CHECK(vx_init(0, &ctx) == VX_OK);
    CHECK(total() == 6 && live == 6);  // none of the attention's
    CHECK(write(ctx, 64) == VX_OK && total() == 7 && loads[vx_co_attn_d64] == 1 && launches == 1);
    CHECK(write(ctx, 64) == VX_OK && attend(ctx, 64, nullptr, 0) == VX_OK && total() == 7);
    const vx_kv_cache c = cache_of(128);
    const vx_attn_batch b = batch_of();
    uint64_t bytes = 0;
    CHECK(vx_attention_ws_size(ctx, &c, &b, nullptr, 3, 4, &bytes) == VX_OK && bytes && total() == 8);  // the plan loads
    CHECK(attend(ctx, 128, (void*)0x4000, bytes) == VX_OK && total() == 8 && launches == 5);              // (attention and its join)
    // a head size whose code is not there: an error, nothing launched, nothing left, and another try later
    const int before = live, launched = launches;
    fail_after = 7;
    CHECK(write(ctx, 96) == VX_ERR_NO_CODE_OBJECT && live == before && launches == launched);
    CHECK(std::strstr(vx_last_error_message(), "d96"));
    CHECK(write(ctx, 96) == VX_OK && live == before + 1);
    // the first use within a capture that allows stream work only
    strict = 1;
    CHECK(write(ctx, 256) == VX_OK && capture == hipStreamCaptureModeGlobal);
    strict = 0;
    CHECK(live == 10);
    CHECK(vx_destroy(ctx) == VX_OK && live == 0);
    // threads whose first use is the same
    CHECK(vx_init(0, &ctx) == VX_OK);
    loads.clear();
    launches = 0;
    std::vector<std::thread> threads;
    std::atomic<int> bad{0};
    for (int i = 0; i < 16; ++i)
        threads.emplace_back([&, i] {
            for (int j = 0; j < 50; ++j) bad += write(ctx, i % 2 ? 64 : 256) != VX_OK;
        });
    for (auto& t : threads) t.join();
    CHECK(!bad && total() == 2 && launches == 800);
    CHECK(vx_destroy(ctx) == VX_OK && live == 0);
    if (!failures) std::printf("fine\n");
    return failures != 0;
}
