// What the C entry points that work on the caller's device memory and stream share (scores.cu, gated.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>
#include <string>

#include "../../include/vmcuda.h"
#include "conv_dispatch.hpp"

namespace vm {

// engine.cu: the message of vm_last_error, and the status of the exception in flight (called inside a handler)
vm_status fail(vm_status s, const std::string& msg);
vm_status status_of_exception();

// The caller's device is current again when the call returns.
class OnDevice {
public:
    explicit OnDevice(int device) {
        VM_CUDA(cudaGetDevice(&before_));
        if (device >= 0 && device != before_) VM_CUDA(cudaSetDevice(device));
        changed_ = device >= 0 && device != before_;
    }
    ~OnDevice() {
        if (changed_) cudaSetDevice(before_);
    }
    OnDevice(const OnDevice&)            = delete;
    OnDevice& operator=(const OnDevice&) = delete;

private:
    int before_   = 0;
    bool changed_ = false;
};

inline size_t element_size(int32_t type) {
    return type == VM_F32 ? 4 : 2;
}
inline bool known_type(int32_t type) {
    return type == VM_F32 || type == VM_F16 || type == VM_BF16;
}
inline bool aligned(const void* p, size_t to) {
    return reinterpret_cast<uintptr_t>(p) % to == 0;
}

// whether all of these begin on their 32-bit elements (NULL: absent)
inline bool words_aligned(std::initializer_list<const void*> pointers) {
    for (const void* p : pointers)
        if (!aligned(p, 4)) return false;
    return true;
}

// f(a value of the element type) for one of the three types
template <typename F>
void with_type(int32_t type, F f) {
    if (type == VM_F32) f(float{});
    else if (type == VM_F16) f(__half{});
    else f(__nv_bfloat16{});
}

}  // namespace vm
