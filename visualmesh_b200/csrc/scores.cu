// vm_scores and vm_scores_backward: checks and launches of the kernels in scores.cuh.
#include "device_call.hpp"
#include "scores.cuh"

namespace {

using namespace vm;
using namespace vm::answers;

vm_status check_rows(const void* x, int32_t type, int64_t rows, int32_t classes, int64_t row_stride, uint32_t flags, const void* labels) {
    if (!known_type(type)) return fail(VM_ERR_INVALID_ARGUMENT, "unknown element type");
    if ((flags & ~static_cast<uint32_t>(VM_PROBABILITIES | VM_LABELS_64)) != 0) return fail(VM_ERR_INVALID_ARGUMENT, "unknown flags");
    if (rows < 0 || rows > INT32_MAX || classes < 1) return fail(VM_ERR_INVALID_ARGUMENT, "rows must be 0..2^31-1 and classes at least 1");
    if (row_stride < 0 || (row_stride > 0 && row_stride > (INT64_MAX >> 4) / (rows > 0 ? rows : 1))) return fail(VM_ERR_INVALID_ARGUMENT, "row stride out of range");
    if (rows > 0 && x == nullptr) return fail(VM_ERR_INVALID_ARGUMENT, "null x");
    if (!aligned(x, element_size(type)) || !aligned(labels, (flags & VM_LABELS_64) != 0 ? 8 : 4)) return fail(VM_ERR_INVALID_ARGUMENT, "x or labels are not aligned to their elements");
    return VM_OK;
}

}  // namespace

extern "C" {

vm_status vm_scores(int device, const void* x, int32_t type, int64_t rows, int32_t classes, int64_t row_stride, uint32_t flags, const void* labels, int32_t top,
                    float* log_prob, float* entropy, float* log_sum, float* top_log_prob, int32_t* top_index, void* stream) {
    try {
        const vm_status s = check_rows(x, type, rows, classes, row_stride, flags, labels);
        if (s != VM_OK) return s;
        if (top < 0 || top > VM_MAX_TOP || top > classes) return fail(VM_ERR_INVALID_ARGUMENT, "top must be 0..min(classes, VM_MAX_TOP)");
        if (rows == 0) return VM_OK;
        if (top > 0 && (top_log_prob == nullptr || top_index == nullptr)) return fail(VM_ERR_INVALID_ARGUMENT, "top without its outputs");
        if (log_prob != nullptr && labels == nullptr) return fail(VM_ERR_INVALID_ARGUMENT, "log_prob without labels");
        const OnDevice on(device);
        const ScoresArgs a{x, rows, classes, row_stride, labels, (flags & VM_LABELS_64) != 0, top, log_prob, entropy, log_sum, top_log_prob, top_index};
        const auto q       = static_cast<cudaStream_t>(stream);
        const int64_t grid = (rows + 7) / 8;
        with_type(type, [&](auto kind) {
            using T = decltype(kind);
            if ((flags & VM_PROBABILITIES) != 0) launch_kernel(k_scores<T, true>, dim3(grid), 256, 0, q, false, a);
            else launch_kernel(k_scores<T, false>, dim3(grid), 256, 0, q, false, a);
        });
    }
    catch (...) {
        return status_of_exception();
    }
    return VM_OK;
}

vm_status vm_scores_backward(int device, const void* x, int32_t type, int64_t rows, int32_t classes, int64_t row_stride, uint32_t flags, const void* labels,
                             const float* entropy, const float* log_sum, const float* d_log_prob, const float* d_entropy, const float* d_log_sum, void* dx,
                             int64_t dx_row_stride, void* stream) {
    try {
        const vm_status s = check_rows(x, type, rows, classes, row_stride, flags, labels);
        if (s != VM_OK) return s;
        if (dx_row_stride < classes || dx_row_stride > (INT64_MAX >> 4) / (rows > 0 ? rows : 1)) return fail(VM_ERR_INVALID_ARGUMENT, "the rows of dx overlap");
        if (rows == 0) return VM_OK;
        if (dx == nullptr || log_sum == nullptr) return fail(VM_ERR_INVALID_ARGUMENT, "null dx or log_sum");
        if (!aligned(dx, element_size(type))) return fail(VM_ERR_INVALID_ARGUMENT, "dx is not aligned to its elements");
        if (d_log_prob != nullptr && labels == nullptr) return fail(VM_ERR_INVALID_ARGUMENT, "d_log_prob without labels");
        if (d_entropy != nullptr && entropy == nullptr) return fail(VM_ERR_INVALID_ARGUMENT, "d_entropy without entropy");
        const OnDevice on(device);
        const ScoresGradArgs a{x, rows, classes, row_stride, labels, (flags & VM_LABELS_64) != 0, entropy, log_sum, d_log_prob, d_entropy, d_log_sum, dx, dx_row_stride};
        const auto q       = static_cast<cudaStream_t>(stream);
        const int64_t grid = (rows + 7) / 8;
        with_type(type, [&](auto kind) {
            using T = decltype(kind);
            if ((flags & VM_PROBABILITIES) != 0) launch_kernel(k_scores_grad<T, true>, dim3(grid), 256, 0, q, false, a);
            else launch_kernel(k_scores_grad<T, false>, dim3(grid), 256, 0, q, false, a);
        });
    }
    catch (...) {
        return status_of_exception();
    }
    return VM_OK;
}

}  // extern "C"
