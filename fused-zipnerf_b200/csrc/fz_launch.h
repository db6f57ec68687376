// fz_launch.h -- host-side launch helpers shared by the 8-bit operators: what a launch asks of a device, asked once; the
// alignment of what it is given.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace zf {

// every pointer lies on a multiple of T's size (null does too): another address would fault on the device
template <typename T, typename... P>
bool aligned_as(const P*... pointers) {
    return ((reinterpret_cast<uintptr_t>(pointers) % sizeof(T) == 0) && ...);
}

constexpr int kMaxDevices = 64;

// the current device's multiprocessors
inline cudaError_t current_multiprocessors(int* count) {
    static std::atomic<int> known[kMaxDevices];
    int device = 0;
    cudaError_t error = cudaGetDevice(&device);
    if (error != cudaSuccess) return error;
    if (device < kMaxDevices && (*count = known[device].load(std::memory_order_relaxed)) != 0) return cudaSuccess;
    error = cudaDeviceGetAttribute(count, cudaDevAttrMultiProcessorCount, device);
    if (error == cudaSuccess && device < kMaxDevices) known[device].store(*count, std::memory_order_relaxed);
    return error;
}

// allows the kernel `bytes` of dynamic shared memory on the current device
template <auto kKernel>
cudaError_t allow_shared_memory(const int bytes) {
    static std::atomic<bool> done[kMaxDevices];
    int device = 0;
    cudaError_t error = cudaGetDevice(&device);
    if (error != cudaSuccess) return error;
    if (device < kMaxDevices && done[device].load(std::memory_order_relaxed)) return cudaSuccess;
    error = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (error == cudaSuccess && device < kMaxDevices) done[device].store(true, std::memory_order_relaxed);
    return error;
}

}  // namespace zf
