// The kernel-provider handle and the host helpers its entry points share (provider.cu, routed.cu,
// matmul_i8.cu).
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <string>

#include <cuda_runtime.h>

#include "../../include/stlq_b200.h"

namespace stlq_b200 {
int SetError(int code, const char* msg);

inline int Ck(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return 0;
    cudaGetLastError();
    return SetError(e == cudaErrorMemoryAllocation ? STLQ_B200_ENOMEM : STLQ_B200_ECUDA,
                    (std::string(what) + ": " + cudaGetErrorString(e)).c_str());
}

inline int Bad(const char* msg) { return SetError(STLQ_B200_EINVAL, msg); }
inline bool Aligned(const void* p, int64_t to) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(to) == 0; }

// Runs an entry point's body: nothing is thrown across the C boundary.
template <typename F>
int Guard(F&& f) {
    try {
        return f();
    } catch (...) {
        return STLQ_B200_ENOMEM;  // the only thing that throws here is a message's memory
    }
}

struct Scratch {
    void* p = nullptr;
    size_t bytes = 0;
    int Ensure(size_t need) {
        if (need <= bytes) return 0;
        if (p) cudaFree(p);
        p = nullptr;
        bytes = 0;
        if (int rc = Ck(cudaMalloc(&p, need), "cudaMalloc (kernel-provider scratch)")) return rc;
        bytes = need;
        return 0;
    }
    void Release() {
        if (p) cudaFree(p);
        p = nullptr;
        bytes = 0;
    }
};

class DeviceScope {
public:
    explicit DeviceScope(int device) {
        if (cudaGetDevice(&prev_) != cudaSuccess) prev_ = -1;
        ok_ = prev_ == device || cudaSetDevice(device) == cudaSuccess;
        restore_ = prev_ >= 0 && prev_ != device;
    }
    ~DeviceScope() {
        if (restore_) cudaSetDevice(prev_);
    }
    bool ok() const { return ok_; }

private:
    int prev_ = -1;
    bool ok_ = false, restore_ = false;
};

#ifdef __CUDACC__
// Programmatic dependent launch: a kernel launched with LaunchAfter may start while the one before it
// in the stream ends.  Each such kernel calls WaitForEarlier before it touches global memory; that
// returns when everything launched earlier in the stream has finished and is visible (each of these
// kernels waits for the one before it), so the results are those of launches one after the other.
// The kernel's life overlaps that of the launch that writes its inputs, so nothing in it may claim that
// memory is read-only or its own while it runs: no __ldg and no __restrict__, whose loads the compiler may
// fetch past the caches' order and move ahead of the wait.  Ordinary loads stay behind it.
// LetLaterStart allows the next one to come up, which it does once every block has called it or left.
__device__ __forceinline__ void WaitForEarlier() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void LetLaterStart() { asm volatile("griddepcontrol.launch_dependents;"); }

template <typename... P, typename... A>
cudaError_t LaunchAfter(void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream, A&&... args) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(block);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, P(args)...);
}
#endif

}  // namespace stlq_b200

struct stlq_b200_kernels {
    int device = 0;
    int num_sms = 148;
    stlq_b200::Scratch At, Bt;  // op(A) rows / op(B) columns made contiguous when the operand layout needs it
    stlq_b200::Scratch err;     // kernels OR DeviceError bits into its first word; stlq_b200_kernels_sync takes them into its second
};
