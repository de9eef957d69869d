// dynamic_smem.cuh -- the dynamic shared memory that a kernel may ask for, raised once per device instead of at every launch (which takes
// as long as a small kernel).
#pragma once
#include <atomic>
#include <mutex>

#include <cuda_runtime.h>

namespace pa {

template <auto Kernel>
static cudaError_t allow_dynamic_smem(size_t bytes) {
    static std::atomic<size_t> most[64];
    static std::mutex lock;
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && most[dev].load(std::memory_order_acquire) >= bytes)) return e;
    std::lock_guard<std::mutex> held(lock);         // never lowered: another thread may be about to launch
    if (dev < 64 && most[dev].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
    const cudaError_t set = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (set == cudaSuccess && dev < 64) most[dev].store(bytes, std::memory_order_release);
    return set;
}

}  // namespace pa
