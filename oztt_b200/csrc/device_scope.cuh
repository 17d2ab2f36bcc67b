// SPDX-License-Identifier: Apache-2.0
// The device of one asynchronous call.
#pragma once
#include <atomic>

#include "runtime.cuh"

namespace oztt {

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
        if (device < 64 && !(opened.load() >> device & 1)) {
            open_device(device);
            opened.fetch_or(1ull << device);
        }
    }
    ~DeviceScope() {
        if (changed) cudaSetDevice(before);
    }
};

}  // namespace oztt
