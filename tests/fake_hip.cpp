// The HIP calls that libbchip.so makes, without a device: memory from malloc, launches noted and
// not run, a switch that says whether the stream is captured. Loaded before the library, its
// symbols are the ones the library binds to, so the host side of its entry points (checks, plans,
// scratch) runs where no GPU is.
#include <hip/hip_runtime.h>

#include <cstdlib>
#include <cstring>
#include <map>
#include <string>
#include <vector>

namespace {
struct Block {
    void* at;
    size_t bytes, serial;
};
std::map<void*, size_t> live;  // addresses, which come back, and the serial numbers of their blocks
std::map<const void*, std::string> kernels;
std::vector<std::string> launches;
std::vector<Block> mallocs;
size_t serial = 0;
bool capturing = false;
hipError_t last = hipSuccess;  // of a call that failed, until hipGetLastError takes it
size_t budget = SIZE_MAX;  // what hipMalloc may still give
dim3 grid_, block_;
size_t shared_;
hipStream_t stream_;

hipError_t launch(const void* f, dim3 g) {
    launches.push_back(kernels[f] + " " + std::to_string(g.x) + " " + std::to_string(g.y) + " " + std::to_string(g.z));
    return hipSuccess;
}
}  // namespace

extern "C" {

void fake_capture(int on) { capturing = on; }
void fake_budget(size_t bytes) { budget = bytes; }
int fake_live(void* p, size_t serial) {
    const auto it = live.find(p);
    return it != live.end() && it->second == serial;
}
size_t fake_live_count() { return live.size(); }
size_t fake_mallocs() { return mallocs.size(); }  // since the last fake_clear, of hipMalloc
void* fake_malloc_at(size_t i, size_t* bytes, size_t* serial) { return *bytes = mallocs[i].bytes, *serial = mallocs[i].serial, mallocs[i].at; }
size_t fake_launches() { return launches.size(); }
const char* fake_launch(size_t i) { return launches[i].c_str(); }  // its kernel and grid
void fake_clear() { mallocs.clear(), launches.clear(); }

void** __hipRegisterFatBinary(const void*) {
    static void* handle;
    return &handle;
}
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* f, char*, const char* name, unsigned, void*, void*, void*, void*, int*) { kernels[f] = name; }
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t shared, hipStream_t s) {
    grid_ = g, block_ = b, shared_ = shared, stream_ = s;
    return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* shared, hipStream_t* s) {
    *g = grid_, *b = block_, *shared = shared_, *s = stream_;
    return hipSuccess;
}

hipError_t hipMalloc(void** p, size_t n) {
    if (capturing) return last = hipErrorStreamCaptureUnsupported;
    if (n > budget) return last = hipErrorOutOfMemory;
    *p = aligned_alloc(256, (n + 255) / 256 * 256);
    live[*p] = ++serial;
    mallocs.push_back({*p, n, serial});
    return hipSuccess;
}
hipError_t hipFree(void* p) {
    if (!p) return hipSuccess;
    if (!live.erase(p)) return hipErrorInvalidValue;
    free(p);
    return hipSuccess;
}
hipError_t hipHostMalloc(void** p, size_t n, unsigned) { return *p = calloc(1, n), hipSuccess; }
hipError_t hipHostFree(void* p) { return free(p), hipSuccess; }
hipError_t hipHostGetDevicePointer(void** d, void* h, unsigned) { return *d = h, hipSuccess; }
hipError_t hipGetSymbolAddress(void** p, const void*) {
    static void* scratch = aligned_alloc(256, (size_t)32 << 20);
    return *p = scratch, hipSuccess;
}
hipError_t hipMemset(void* p, int v, size_t n) { return memset(p, v, n), hipSuccess; }
hipError_t hipMemsetAsync(void* p, int v, size_t n, hipStream_t) { return memset(p, v, n), hipSuccess; }
hipError_t hipMemcpyAsync(void* d, const void* s, size_t n, hipMemcpyKind, hipStream_t) { return memcpy(d, s, n), hipSuccess; }
hipError_t hipMemGetInfo(size_t* f, size_t* t) { return *f = *t = (size_t)288 << 30, hipSuccess; }

hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDeviceCount(int* n) { return *n = 1, hipSuccess; }
hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) { return *v = 256, hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
    memset(p, 0, sizeof *p);
    strcpy(p->gcnArchName, "gfx950");
    p->multiProcessorCount = 256;
    return hipSuccess;
}
hipError_t hipGetLastError() {
    const hipError_t e = last;
    last = hipSuccess;
    return e;
}
const char* hipGetErrorString(hipError_t) { return "an error"; }

hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { return *s = (hipStream_t)&stream_, hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
    return *s = capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone, hipSuccess;
}
hipError_t hipEventCreate(hipEvent_t* e) { return *e = (hipEvent_t)&stream_, hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) { return *ms = 0, hipSuccess; }
hipError_t hipLaunchKernel(const void* f, dim3 g, dim3, void**, size_t, hipStream_t) { return launch(f, g); }
hipError_t hipExtLaunchKernel(const void* f, dim3 g, dim3, void**, size_t, hipStream_t, hipEvent_t, hipEvent_t, int) { return launch(f, g); }

}  // extern "C"
