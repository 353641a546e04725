// A HIP runtime of two devices that runs nothing, for tests of the engine's host code on the CPU: loaded with global
// symbols ahead of libgqa.so, it takes that library's HIP calls, keeps the calls in a log and can be told to fail.
//
// A line of the log: the device that was current, the call, and what it was about.  An error stays for hipGetLastError
// until that is called, however many calls succeed in between, as the runtime's does.
#include <hip/hip_runtime_api.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>
#include <sys/mman.h>

#include <map>
#include <sstream>
#include <string>

namespace {
int g_device = 0;
hipError_t g_last = hipSuccess;
std::ostringstream g_log;
std::string g_taken;
size_t g_malloc_limit = ~(size_t)0;  // a larger allocation fails
int g_fail_launch = -1;              // launches until one fails (-1: none)
std::map<void*, size_t> g_sizes;
std::map<const void*, std::string> g_kernels;
uintptr_t g_handle = 0x1000;

struct Call {
    dim3 grid, block;
    size_t lds;
    hipStream_t stream;
} g_call;

hipError_t fail(hipError_t e) { return g_last = e; }

std::ostringstream& line(const char* call) {
    g_log << g_device << ' ' << call << ' ';
    return g_log;
}

hipError_t launch(const void* f, dim3 grid, dim3 block, hipStream_t s) {
    line("launch") << g_kernels[f] << ' ' << s << ' ' << grid.x << ' ' << grid.y << ' ' << grid.z << ' ' << block.x << '\n';
    if (g_fail_launch == 0) {
        g_fail_launch = -1;
        return fail(hipErrorLaunchFailure);
    }
    if (g_fail_launch > 0) --g_fail_launch;
    const uint64_t most = 0xFFFFFFFFull;  // work-items of a dimension
    if (grid.x < 1 || grid.y < 1 || grid.z < 1 || (uint64_t)grid.x * block.x > most || (uint64_t)grid.y * block.y > most ||
        grid.y > 65535 || grid.z > 65535 || (uint64_t)block.x * block.y * block.z > 1024)
        return fail(hipErrorInvalidConfiguration);
    return hipSuccess;
}
}  // namespace

extern "C" {

// ---- what the tests call ----
const char* stub_take_log() {
    g_taken = g_log.str();
    g_log.str("");
    return g_taken.c_str();
}
void stub_fail_malloc_above(size_t bytes) { g_malloc_limit = bytes; }
void stub_fail_launch(int after) { g_fail_launch = after; }
int stub_device() { return g_device; }

// ---- what the library calls ----
void** __hipRegisterFatBinary(const void*) {
    static void* handle;
    return &handle;
}
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, void*, void*, int*) {
    g_kernels[host] = name;
}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t s) {
    g_call = Call{grid, block, lds, s};
    return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* lds, hipStream_t* s) {
    *grid = g_call.grid;
    *block = g_call.block;
    *lds = g_call.lds;
    *s = g_call.stream;
    return hipSuccess;
}
hipError_t hipLaunchKernel(const void* f, dim3 grid, dim3 block, void**, size_t, hipStream_t s) { return launch(f, grid, block, s); }
hipError_t hipExtLaunchKernel(const void* f, dim3 grid, dim3 block, void**, size_t, hipStream_t s, hipEvent_t, hipEvent_t, int) {
    return launch(f, grid, block, s);
}
hipError_t hipGetLastError() {
    const hipError_t e = g_last;
    g_last = hipSuccess;
    return e;
}
const char* hipGetErrorString(hipError_t) { return "stub"; }
hipError_t hipGetDeviceCount(int* n) {
    *n = 2;
    return hipSuccess;
}
hipError_t hipGetDevice(int* d) {
    *d = g_device;
    return hipSuccess;
}
hipError_t hipSetDevice(int d) {
    if (d < 0 || d > 1) return fail(hipErrorInvalidDevice);
    g_device = d;
    return hipSuccess;
}
hipError_t hipGetDeviceProperties(hipDeviceProp_t* p, int) {  // (the header names it by its version)
    memset(p, 0, sizeof(*p));
    strcpy(p->gcnArchName, "gfx950");
    p->multiProcessorCount = 256;
    p->clockRate = 2400000;
    return hipSuccess;
}
hipError_t hipDeviceSynchronize() {
    line("hipDeviceSynchronize") << '\n';
    return hipSuccess;
}
hipError_t hipMalloc(void** p, size_t n) {
    line("hipMalloc") << n << '\n';
    *p = nullptr;
    if (n > g_malloc_limit) return fail(hipErrorOutOfMemory);
    if (n == 0) return hipSuccess;
    void* const at = mmap(nullptr, n, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
    if (at == MAP_FAILED) return fail(hipErrorOutOfMemory);
    g_sizes[at] = n;
    *p = at;
    return hipSuccess;
}
hipError_t hipFree(void* p) {
    if (p == nullptr) return hipSuccess;
    line("hipFree") << g_sizes[p] << '\n';
    munmap(p, g_sizes[p]);
    g_sizes.erase(p);
    return hipSuccess;
}
hipError_t hipHostMalloc(void** p, size_t n, unsigned) {
    *p = malloc(n);
    return *p != nullptr ? hipSuccess : fail(hipErrorOutOfMemory);
}
hipError_t hipHostFree(void* p) {
    free(p);
    return hipSuccess;
}
hipError_t hipMemcpyAsync(void*, const void*, size_t n, hipMemcpyKind, hipStream_t s) {
    line("hipMemcpyAsync") << n << ' ' << s << '\n';
    return hipSuccess;
}
hipError_t hipMemcpy2DAsync(void*, size_t, const void*, size_t, size_t w, size_t h, hipMemcpyKind, hipStream_t s) {
    line("hipMemcpyAsync") << w * h << ' ' << s << '\n';
    return hipSuccess;
}
hipError_t hipMemset(void*, int, size_t) { return hipSuccess; }
hipError_t hipMemsetAsync(void*, int, size_t, hipStream_t) { return hipSuccess; }
hipError_t hipGetSymbolAddress(void** p, const void* symbol) {
    *p = const_cast<void*>(symbol);
    return hipSuccess;
}
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) {
    *s = reinterpret_cast<hipStream_t>(g_handle += 16);
    return hipSuccess;
}
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* status) {
    *status = hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamWaitEvent(hipStream_t s, hipEvent_t e, unsigned) {
    line("hipStreamWaitEvent") << e << ' ' << s << '\n';
    return hipSuccess;
}
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) {
    *e = reinterpret_cast<hipEvent_t>(g_handle += 16);
    return hipSuccess;
}
hipError_t hipEventCreate(hipEvent_t* e) { return hipEventCreateWithFlags(e, 0); }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventQuery(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t e, hipStream_t s) {
    line("hipEventRecord") << e << ' ' << s << '\n';
    return hipSuccess;
}
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) {
    *ms = 0.f;
    return hipSuccess;
}

}  // extern "C"
