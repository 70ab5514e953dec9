// A CUDA runtime of host memory and as many devices as a test wants, for what the library does on the host:
// which device is current at a call, what is waited for, and which attributes a launch finds. Nothing runs.
#include <cuda.h>
#include <cuda_runtime_api.h>

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>
#include <string>
#include <utility>

namespace {
std::mutex mu;
std::string events;
int devices = 2;
cudaError_t sync_result = cudaSuccess;
std::map<std::pair<const void*, int>, int> shared_limit;  // of a function on a device
thread_local int current = 0;
struct Config { dim3 grid, block; size_t shared; void* stream; };
thread_local Config pushed;

void note(const char* fmt, ...) {
    char line[128];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(line, sizeof line, fmt, ap);
    va_end(ap);
    std::lock_guard<std::mutex> lock(mu);
    events += line;
    events += '\n';
}

cudaError_t launch(const void* f, size_t shared) {
    int limit = 48 << 10;
    {
        std::lock_guard<std::mutex> lock(mu);
        auto it = shared_limit.find({f, current});
        if (it != shared_limit.end()) limit = it->second;
    }
    if (shared > static_cast<size_t>(limit)) {
        note("refused launch on %d", current);
        return cudaErrorInvalidValue;
    }
    note("launch on %d", current);
    return cudaSuccess;
}

CUresult encode_tiled(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                      const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
    return CUDA_SUCCESS;
}
CUresult encode_im2col(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const int*, const int*,
                       cuuint32_t, cuuint32_t, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                       CUtensorMapFloatOOBfill) {
    return CUDA_SUCCESS;
}
}  // namespace

extern "C" {
// ---- for the tests
__attribute__((visibility("default"))) void fake_set_device(int d) { current = d; }
__attribute__((visibility("default"))) int fake_device() { return current; }
__attribute__((visibility("default"))) void fake_sync_result(int e) { sync_result = static_cast<cudaError_t>(e); }
__attribute__((visibility("default"))) size_t fake_events(char* to, size_t room) {  // and forgets them
    std::lock_guard<std::mutex> lock(mu);
    const size_t n = events.size() < room - 1 ? events.size() : room - 1;
    memcpy(to, events.data(), n);
    to[n] = 0;
    events.clear();
    return n;
}

// ---- devices
cudaError_t cudaGetDeviceCount(int* n) { *n = devices; return cudaSuccess; }
cudaError_t cudaGetDevice(int* d) { *d = current; return cudaSuccess; }
cudaError_t cudaSetDevice(int d) {
    if (d < 0 || d >= devices) return cudaErrorInvalidDevice;
    current = d;
    return cudaSuccess;
}
#undef cudaGetDeviceProperties
cudaError_t cudaGetDeviceProperties_v2(cudaDeviceProp* p, int) {
    memset(p, 0, sizeof *p);
    p->major = 10;
    p->multiProcessorCount = 148;
    p->clockRate = 1965000;
    return cudaSuccess;
}
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr a, int) {
    *v = a == cudaDevAttrMultiProcessorCount ? 148 : 1965000;
    return cudaSuccess;
}
cudaError_t cudaDeviceSynchronize() { note("synchronize %d", current); return sync_result; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t e) { return e == cudaSuccess ? "no error" : "fake error"; }

// ---- memory
cudaError_t cudaMalloc(void** p, size_t n) { *p = aligned_alloc(256, (n + 255) / 256 * 256); return cudaSuccess; }
cudaError_t cudaFree(void* p) { free(p); return cudaSuccess; }
cudaError_t cudaMemcpy(void* d, const void* s, size_t n, cudaMemcpyKind) { memcpy(d, s, n); return cudaSuccess; }
cudaError_t cudaMemcpyAsync(void* d, const void* s, size_t n, cudaMemcpyKind, cudaStream_t) { memcpy(d, s, n); return cudaSuccess; }
cudaError_t cudaMemset(void* p, int v, size_t n) { memset(p, v, n); return cudaSuccess; }
cudaError_t cudaMemsetAsync(void* p, int v, size_t n, cudaStream_t) { memset(p, v, n); return cudaSuccess; }
cudaError_t cudaMemPoolCreate(cudaMemPool_t* p, const cudaMemPoolProps*) { *p = reinterpret_cast<cudaMemPool_t>(&devices); return cudaSuccess; }
cudaError_t cudaMemPoolDestroy(cudaMemPool_t) { return cudaSuccess; }
cudaError_t cudaMemPoolSetAttribute(cudaMemPool_t, cudaMemPoolAttr, void*) { return cudaSuccess; }
cudaError_t cudaMallocFromPoolAsync(void** p, size_t n, cudaMemPool_t, cudaStream_t) { note("workspace on %d", current); return cudaMalloc(p, n); }
cudaError_t cudaFreeAsync(void* p, cudaStream_t) { note("free on %d", current); free(p); return cudaSuccess; }
cudaError_t cudaGetSymbolAddress(void** p, const void*) { return cudaMalloc(p, 1 << 20); }

// ---- functions and launches
cudaError_t cudaFuncGetAttributes(cudaFuncAttributes* a, const void*) {
    memset(a, 0, sizeof *a);
    a->numRegs = 255;
    return cudaSuccess;
}
cudaError_t cudaFuncSetAttribute(const void* f, cudaFuncAttribute a, int v) {
    std::lock_guard<std::mutex> lock(mu);
    if (a == cudaFuncAttributeMaxDynamicSharedMemorySize) shared_limit[{f, current}] = v;
    return cudaSuccess;
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void**) { return launch(f, c->dynamicSmemBytes); }
cudaError_t cudaLaunchKernel(const void* f, dim3, dim3, void**, size_t shared, cudaStream_t) { return launch(f, shared); }
unsigned __cudaPushCallConfiguration(dim3 g, dim3 b, size_t shared, void* st) {
    pushed = Config{g, b, shared, st};
    return 0;
}
cudaError_t __cudaPopCallConfiguration(dim3* g, dim3* b, size_t* shared, void* st) {
    *g = pushed.grid;
    *b = pushed.block;
    *shared = pushed.shared;
    *static_cast<void**>(st) = pushed.stream;
    return cudaSuccess;
}
cudaError_t cudaGetDriverEntryPoint(const char* name, void** f, unsigned long long, cudaDriverEntryPointQueryResult* q) {
    *f = strstr(name, "Im2col") ? reinterpret_cast<void*>(&encode_im2col) : reinterpret_cast<void*>(&encode_tiled);
    *q = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
void** __cudaRegisterFatBinary(void*) { static void* handle; return &handle; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, void*, void*, void*, void*, int*) {}
void __cudaRegisterVar(void**, char*, char*, const char*, int, size_t, int, int) {}

// ---- not used by what is tested
cudaError_t cudaEventCreate(cudaEvent_t*) { return cudaErrorNotSupported; }
cudaError_t cudaEventDestroy(cudaEvent_t) { return cudaErrorNotSupported; }
cudaError_t cudaEventElapsedTime(float*, cudaEvent_t, cudaEvent_t) { return cudaErrorNotSupported; }
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t cudaGraphDestroy(cudaGraph_t) { return cudaErrorNotSupported; }
cudaError_t cudaGraphExecDestroy(cudaGraphExec_t) { return cudaErrorNotSupported; }
cudaError_t cudaGraphInstantiate(cudaGraphExec_t*, cudaGraph_t, unsigned long long) { return cudaErrorNotSupported; }
cudaError_t cudaGraphLaunch(cudaGraphExec_t, cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t cudaStreamBeginCapture(cudaStream_t, cudaStreamCaptureMode) { return cudaErrorNotSupported; }
cudaError_t cudaStreamEndCapture(cudaStream_t, cudaGraph_t*) { return cudaErrorNotSupported; }
}
