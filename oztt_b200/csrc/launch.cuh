// SPDX-License-Identifier: Apache-2.0
// What the asynchronous calls share: the device of a call, and launches that overlap.
#pragma once
#include <atomic>

#include "runtime.cuh"

namespace oztt {

// While it lives, this thread may make calls that are no part of a stream's capture (they wait for no stream and add
// nothing to one) although one is going on: what a process does once must not fail a capture that happens to be first.
struct OutsideCapture {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    OutsideCapture() { OZTT_CUDA(cudaThreadExchangeStreamCaptureMode(&mode)); }
    ~OutsideCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
    OutsideCapture(const OutsideCapture&) = delete;
};

// The word that a bounded wait of a layer product writes when it gives up: host memory, a word for each device. These
// calls do not wait for their kernels, so the device's next call, or the optimiser's that would use what they computed,
// looks at it and throws (linear.cu).
int* error_word(int device);
void check_earlier_calls(int device);

// Makes `device` current for one call.
struct DeviceScope {
    int before = 0;
    bool changed = false;
    explicit DeviceScope(int device) {
        if (device < 0) throw Error(OZTT_EINVAL, "device_id must be nonnegative");
        OZTT_CUDA(cudaGetDevice(&before));
        if (before != device) {
            OZTT_CUDA(cudaSetDevice(device));
            changed = true;
        }
        static std::atomic<uint64_t> opened{0};
        if (device < 64 && (opened.load() >> device & 1)) return;
        try {
            OutsideCapture outside;
            open_device(device);
        } catch (...) {
            cudaSetDevice(before);
            throw;
        }
        if (device < 64) opened.fetch_or(1ull << device);
    }
    ~DeviceScope() {
        if (changed) cudaSetDevice(before);
    }
};

constexpr int KNOWN_DEVICES = 64;  // of which what was asked once is kept

// The current device, and the SMs of a device.
inline int current_device() {
    int device = 0;
    OZTT_CUDA(cudaGetDevice(&device));
    return device;
}
inline uint32_t multiprocessors(int device) {
    static std::atomic<int> known[KNOWN_DEVICES];
    int n = device < KNOWN_DEVICES ? known[device].load() : 0;
    if (!n) {
        OZTT_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device));
        if (device < KNOWN_DEVICES) known[device].store(n);
    }
    return (uint32_t)n;
}

// Lets the next kernel of the stream start while this one ends, and waits for the one before, which must be over
// before anything in memory is read or written (both do nothing where the launch did not ask for the overlap). The
// kernel before may still be writing what this one reads, so no input of such a kernel is `const __restrict__`.
// early: false to let the next kernel start only when this one has ended.
__device__ __forceinline__ void overlap_launches(bool early = true) {
    if (early) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Launches a kernel so that it may start while the kernel before it on the stream ends (overlap_launches), its
// blocks in clusters of `cluster` (as the kernel says where that is {0}).
template <class... Params, class... Args>
inline void launch_overlapped(void (*kernel)(Params...), dim3 grid, uint32_t threads, uint32_t smem, dim3 cluster,
                   cudaStream_t st, Args&&... args) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster.x;
    attr[1].val.clusterDim.y = cluster.y;
    attr[1].val.clusterDim.z = cluster.z;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = cluster.x ? 2 : 1;
    OZTT_CUDA(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
}

// Allows a kernel its dynamic shared memory, and clusters of up to 16, once on each device.
template <class Kernel>
inline void allow_smem(Kernel* kernel, uint32_t bytes, std::atomic<uint64_t>& allowed, bool large_clusters = false) {
    const int device = current_device();
    if (device < 64 && (allowed.load() >> device & 1)) return;
    OZTT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    if (large_clusters) OZTT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (device < 64) allowed.fetch_or(1ull << device);
}

}  // namespace oztt
