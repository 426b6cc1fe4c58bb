// The parts of the HIP runtime that the page cache's host code uses, on the CPU: device memory is the host's, filled
// with a pattern; a launch runs its threads one after the other (for kernels without barriers); allocations and
// launches can be made to fail.
#pragma once

#include <sys/mman.h>

#include <cstddef>
#include <cstdint>
#include <cstring>
#include <map>

#define __global__
#define __device__
#define __host__
#define __shared__ static
#define __forceinline__ inline
#define __launch_bounds__(...)

struct dim3 {
    unsigned x, y, z;
    dim3(unsigned a = 1, unsigned b = 1, unsigned c = 1) : x(a), y(b), z(c) {}
};
struct uint2 {
    unsigned x, y;
};
struct int4 {
    int x, y, z, w;
};
inline dim3 blockIdx, threadIdx, blockDim, gridDim;

typedef enum { hipSuccess = 0, hipErrorOutOfMemory = 2, hipErrorInvalidConfiguration = 9 } hipError_t;
typedef struct ihipStream_t *hipStream_t;
typedef int *hipEvent_t;
enum { hipMemcpyHostToDevice = 1, hipEventDisableTiming = 2, hipHostMallocDefault = 0 };

namespace stub {
inline int mallocs_left = -1, host_mallocs_left = -1, launches_left = -1, memcpys_left = -1;  // until one fails; -1: none does
inline int device = 0;
inline hipError_t last = hipSuccess;
inline bool capture = false;
inline std::map<void *, size_t> live;
inline bool fails(int *left) {
    if (*left < 0) return false;
    if (*left == 0) return true;
    --*left;
    return false;
}
inline hipError_t allocate(void **p, size_t n) {
    *p = mmap(nullptr, n, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
    if (*p == MAP_FAILED) return last = hipErrorOutOfMemory;
    if (n < ((size_t)64 << 20)) std::memset(*p, 0xa5, n);  // (larger ones: zeros that take no memory)
    live[*p] = n;
    return hipSuccess;
}
inline hipError_t release(void *p) {
    auto it = live.find(p);
    if (it == live.end()) return hipSuccess;
    munmap(p, it->second);
    live.erase(it);
    return hipSuccess;
}
template <class K, class... A>
void launch(K k, dim3 grid, dim3 block, A... args) {
    if (fails(&launches_left) || (uint64_t)grid.x * block.x >> 32 || grid.y > 65535 || grid.z > 65535) {
        last = hipErrorInvalidConfiguration;
        return;
    }
    gridDim = grid;
    blockDim = block;
    for (blockIdx.z = 0; blockIdx.z < grid.z; blockIdx.z++)
        for (blockIdx.y = 0; blockIdx.y < grid.y; blockIdx.y++)
            for (blockIdx.x = 0; blockIdx.x < grid.x; blockIdx.x++)
                for (threadIdx.x = 0; threadIdx.x < block.x; threadIdx.x++) k(args...);
}
}  // namespace stub

#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) stub::launch(kernel, grid, block, __VA_ARGS__)

template <class T>
hipError_t hipMalloc(T **p, size_t n) {
    if (stub::fails(&stub::mallocs_left)) return stub::last = hipErrorOutOfMemory;
    return stub::allocate((void **)p, n);
}
inline hipError_t hipHostMalloc(void **p, size_t n, unsigned) {
    if (stub::fails(&stub::host_mallocs_left)) return stub::last = hipErrorOutOfMemory;
    return stub::allocate(p, n);
}
inline hipError_t hipFree(void *p) { return stub::release(p); }
inline hipError_t hipHostFree(void *p) { return stub::release(p); }
inline hipError_t hipGetDevice(int *d) {
    *d = stub::device;
    return hipSuccess;
}
inline hipError_t hipGetLastError() {
    const hipError_t e = stub::last;
    stub::last = hipSuccess;
    return e;
}
inline const char *hipGetErrorString(hipError_t) { return "HIP error"; }
inline hipError_t hipMemsetAsync(void *p, int v, size_t n, hipStream_t) {
    if (n < ((size_t)64 << 20)) std::memset(p, v, n);
    return hipSuccess;
}
inline hipError_t hipMemcpyAsync(void *to, const void *from, size_t n, int, hipStream_t) {
    if (stub::fails(&stub::memcpys_left)) return hipErrorInvalidConfiguration;
    std::memcpy(to, from, n);
    return hipSuccess;
}
inline hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
inline hipError_t hipEventCreateWithFlags(hipEvent_t *e, unsigned) {
    *e = new int;
    return hipSuccess;
}
inline hipError_t hipEventDestroy(hipEvent_t e) {
    delete e;
    return hipSuccess;
}
inline hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
inline hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
