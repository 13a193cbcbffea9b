// Host helpers shared by the block-scaled quantiser and the matrix products.
#pragma once

#include "blockscale.h"
#include "common.h"

namespace aeisu {

// Makes `dev` current for the scope.  Set even where it already is: that is what gives a thread that
// has not used the GPU yet (one of autograd's) the device's context, which tensor maps need.
struct OnDevice {
    int prev = -1;
    explicit OnDevice(int dev) {
        AEISU_CUDA(cudaGetDevice(&prev));
        AEISU_CUDA(cudaSetDevice(dev));
        if (prev == dev) prev = -1;
    }
    ~OnDevice() {
        if (prev >= 0) cudaSetDevice(prev);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
};

inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
inline bool is_code(int t) { return t == kE4M3 || t == kE5M2; }

}  // namespace aeisu
