// What the checkpoint tables (mpc_amd/csrc/prg.hip) use of the HIP runtime, on the CPU: device memory is host memory, a copy
// is carried out when its stream is synchronised (so its source has to be there until then), kernels are not run.  Every copy
// is written down, with the memory that it was given as its source.
#pragma once
#include <stddef.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>
#include <mutex>
#include <vector>

enum hipError_t { hipSuccess = 0, hipErrorOutOfMemory = 2 };
enum hipMemcpyKind { hipMemcpyHostToDevice = 1 };
enum { hipStreamNonBlocking = 1, hipHostMallocDefault = 0 };
typedef struct stub_event *hipEvent_t;

struct StubCopy {
    void *dst;
    const void *src;
    size_t bytes;
};
struct stub_stream {
    std::vector<StubCopy> queued;
};
typedef stub_stream *hipStream_t;
struct Stub {
    std::mutex mu;
    std::vector<std::pair<const char *, size_t>> pinned; // what hipHostMalloc gave out
    size_t copies = 0, copied = 0, from_pageable = 0;
};
inline Stub &stub() {
    static Stub *s = new Stub();
    return *s;
}
inline const char *hipGetErrorString(hipError_t) { return "error"; }
inline hipError_t hipGetLastError() { return hipSuccess; }
inline hipError_t hipSetDevice(int) { return hipSuccess; }
inline hipError_t hipMalloc(void **p, size_t n) { return (*p = malloc(n)) ? hipSuccess : hipErrorOutOfMemory; }
inline hipError_t hipFree(void *p) {
    free(p);
    return hipSuccess;
}
inline hipError_t hipHostMalloc(void **p, size_t n, unsigned) {
    std::lock_guard<std::mutex> g(stub().mu);
    if (!(*p = malloc(n))) return hipErrorOutOfMemory;
    stub().pinned.emplace_back((const char *)*p, n);
    return hipSuccess;
}
inline hipError_t hipStreamCreateWithFlags(hipStream_t *s, unsigned) {
    *s = new stub_stream();
    return hipSuccess;
}
inline hipError_t hipMemcpyAsync(void *dst, const void *src, size_t n, hipMemcpyKind, hipStream_t s) {
    std::lock_guard<std::mutex> g(stub().mu);
    bool pinned = false;
    for (auto &r : stub().pinned) pinned |= (const char *)src >= r.first && (const char *)src + n <= r.first + r.second;
    stub().copies++;
    stub().copied += n;
    if (!pinned) stub().from_pageable += n;
    s->queued.push_back(StubCopy{dst, src, n});
    return hipSuccess;
}
inline hipError_t hipStreamSynchronize(hipStream_t s) {
    std::vector<StubCopy> todo;
    {
        std::lock_guard<std::mutex> g(stub().mu);
        if (s) todo.swap(s->queued);
    }
    for (auto &c : todo) memcpy(c.dst, c.src, c.bytes);
    return hipSuccess;
}
inline hipError_t hipEventCreate(hipEvent_t *) { return hipErrorOutOfMemory; }
inline hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }

// enough of the kernel language for the kernels of the file to be parsed
#define __global__
#define __device__
#define __host__
#define __shared__ static
#define __launch_bounds__(...)
#define __builtin_amdgcn_fence(...)
#define __builtin_amdgcn_wave_barrier()
struct dim3 {
    uint32_t x, y = 1, z = 1;
    dim3(uint32_t a) : x(a) {}
};
static const dim3 threadIdx(0), blockIdx(0), blockDim(1), gridDim(1);
struct uint4 {
    uint32_t x, y, z, w;
};
inline uint4 make_uint4(uint32_t x, uint32_t y, uint32_t z, uint32_t w) { return {x, y, z, w}; }
inline uint32_t __umul24(uint32_t a, uint32_t b) { return (a & 0xFFFFFFu) * (b & 0xFFFFFFu); }
#define hipLaunchKernelGGL(...) ((void)0)
