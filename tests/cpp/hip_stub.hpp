// The HIP runtime as the library's host side sees it, without a GPU: device memory is host memory, launches
// are noted and not run.  A program that defines these functions and exports them (-rdynamic) is what
// libnabla_optim.so is bound to, ahead of libamdhip64.
#ifndef NBO_TEST_HIP_STUB_HPP
#define NBO_TEST_HIP_STUB_HPP
#include <hip/hip_runtime_api.h>

#include <cstdlib>
#include <cstring>
#include <map>
#include <string>
#include <vector>

namespace stub {
struct Launch {
    std::string name;
    uint32_t gx, gy, block, lds;
    std::vector<char> args;
};
inline std::vector<Launch> launches;
inline std::map<uintptr_t, size_t> blocks; // device memory: address, bytes
inline std::vector<const void *> modules;   // loaded, in order
inline int devices = 1, device = 0, fail_module = -1; // fail_module: which load (from 0) fails, this once
inline hipStreamCaptureMode capture_mode = hipStreamCaptureModeGlobal, load_mode = hipStreamCaptureModeGlobal;
// bytes of the argument block of a kernel whose arguments a test wants to look at
inline size_t (*args_bytes)(const std::string &name) = nullptr;

inline const std::map<uintptr_t, size_t>::value_type *block_of(const void *p)
{
    auto it = blocks.upper_bound((uintptr_t)p);
    if (it == blocks.begin()) return nullptr;
    --it;
    return (uintptr_t)p < it->first + it->second ? &*it : nullptr;
}
} // namespace stub

extern "C" {
void **__hipRegisterFatBinary(const void *) { static void *h; return &h; }
void __hipRegisterVar(void **, void *, char *, char *, int, size_t, int, int) {}
void __hipUnregisterFatBinary(void **) {}
hipError_t hipGetDeviceCount(int *n) { *n = stub::devices; return hipSuccess; }
hipError_t hipGetDevice(int *d) { *d = stub::device; return hipSuccess; }
hipError_t hipSetDevice(int d) { stub::device = d; return hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600 *p, int)
{
    std::memset((void *)p, 0, sizeof(*p));
    std::strcpy(p->gcnArchName, "gfx950");
    return hipSuccess;
}
const char *hipGetErrorString(hipError_t) { return "stub"; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipEventCreate(hipEvent_t *e) { *e = nullptr; return hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t *e, unsigned) { *e = nullptr; return hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float *ms, hipEvent_t, hipEvent_t) { *ms = 1.0f; return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipGetSymbolAddress(void **p, const void *) { static char image[1 << 16]; *p = image; return hipSuccess; }
hipError_t hipMalloc(void **p, size_t n)
{
    // address space alone, up to sizes that no test touches
    *p = n < ((size_t)64 << 20) ? std::malloc(n) : (void *)((uintptr_t)0x10000000000 + ((uintptr_t)stub::blocks.size() << 40));
    stub::blocks[(uintptr_t)*p] = n;
    return hipSuccess;
}
hipError_t hipFree(void *p)
{
    auto it = stub::blocks.find((uintptr_t)p);
    if (it == stub::blocks.end()) return hipErrorInvalidValue;
    if (it->second < ((size_t)64 << 20)) std::free(p);
    stub::blocks.erase(it);
    return hipSuccess;
}
hipError_t hipHostMalloc(void **p, size_t n, unsigned) { *p = std::malloc(n); return hipSuccess; }
hipError_t hipMemGetInfo(size_t *f, size_t *t) { *f = *t = (size_t)1 << 30; return hipSuccess; }
hipError_t hipMemcpyAsync(void *d, const void *s, size_t n, hipMemcpyKind, hipStream_t) { std::memcpy(d, s, n); return hipSuccess; }
hipError_t hipPointerGetAttributes(hipPointerAttribute_t *a, const void *p)
{
    std::memset((void *)a, 0, sizeof(*a));
    a->type = stub::block_of(p) ? hipMemoryTypeDevice : hipMemoryTypeUnregistered;
    return hipSuccess;
}
hipError_t hipMemGetAddressRange(hipDeviceptr_t *base, size_t *size, hipDeviceptr_t p)
{
    const auto *b = stub::block_of(p);
    if (!b) return hipErrorNotFound;
    *base = (hipDeviceptr_t)b->first;
    *size = b->second;
    return hipSuccess;
}
hipError_t hipThreadExchangeStreamCaptureMode(hipStreamCaptureMode *m) { std::swap(*m, stub::capture_mode); return hipSuccess; }
hipError_t hipModuleLoadData(hipModule_t *m, const void *image)
{
    if (stub::fail_module == (int)stub::modules.size()) {
        stub::fail_module = -1;
        return hipErrorNoBinaryForGpu;
    }
    stub::load_mode = stub::capture_mode;
    stub::modules.push_back(image);
    *m = (hipModule_t)(uintptr_t)stub::modules.size();
    return hipSuccess;
}
hipError_t hipModuleUnload(hipModule_t) { return hipSuccess; }
hipError_t hipModuleGetFunction(hipFunction_t *f, hipModule_t, const char *name)
{
    static std::map<std::string, int> names;
    *f = (hipFunction_t)&*names.insert({name, 0}).first;
    return hipSuccess;
}
hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned gx, unsigned gy, unsigned, unsigned bx, unsigned, unsigned,
                                 unsigned lds, hipStream_t, void **args, void **)
{
    stub::Launch l{((std::pair<const std::string, int> *)f)->first, gx, gy, bx, lds, {}};
    if (const size_t n = stub::args_bytes ? stub::args_bytes(l.name) : 0) l.args.assign((char *)args[0], (char *)args[0] + n);
    stub::launches.push_back(l);
    return hipSuccess;
}
}
#endif
