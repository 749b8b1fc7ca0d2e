// vm_scores and vm_scores_backward: checks and launches of the kernels in scores.cuh.
#include <algorithm>
#include <type_traits>

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

constexpr int SMS = 148;  // of a B200; which launch is taken depends on it, no result
// Classes that a thread holds in its registers. 1,000,000 rows of 8 floats, with the two best / their gradient: 19 / 19 us, by two lanes a row
// 35 / 23; of 3 floats 11 / 11 and 36 / 16.
constexpr int MOST_OF_THREAD = 8;
// Classes that lanes of a warp share with the best of them, without, and for gradients; beyond that a warp at least streams through its row.
// 100,000 rows of 256 floats with five best 91 us and 117; 60,000 of 512 bf16 without 33 and 44, of 1024 69 and 50; the gradient of 1024 64 and 194.
constexpr int MOST_OF_LANES_TOP = 256, MOST_OF_LANES = 512, MOST_OF_LANES_GRADIENT = 1024;

// f(classes), as a constant
template <typename F>
void with_classes(int classes, F f) {
    using std::integral_constant;
    switch (classes) {
        case 1: return f(integral_constant<int, 1>{});
        case 2: return f(integral_constant<int, 2>{});
        case 3: return f(integral_constant<int, 3>{});
        case 4: return f(integral_constant<int, 4>{});
        case 5: return f(integral_constant<int, 5>{});
        case 6: return f(integral_constant<int, 6>{});
        case 7: return f(integral_constant<int, 7>{});
        default: return f(integral_constant<int, 8>{});
    }
}
// f(lanes of a row, values of a lane), as constants, for up to MOST classes
template <int MOST, typename F>
void with_lanes(int classes, F f) {
    using std::integral_constant;
    if (classes <= 16) f(integral_constant<int, 2>{}, integral_constant<int, 8>{});
    else if (classes <= 32) f(integral_constant<int, 4>{}, integral_constant<int, 8>{});
    else if (classes <= 64) f(integral_constant<int, 8>{}, integral_constant<int, 8>{});
    else if (classes <= 128) f(integral_constant<int, 16>{}, integral_constant<int, 8>{});
    else if (MOST <= 256 || classes <= 256) f(integral_constant<int, 32>{}, integral_constant<int, 8>{});
    else if constexpr (MOST > 256) {
        if (MOST <= 512 || classes <= 512) f(integral_constant<int, 32>{}, integral_constant<int, 16>{});
        else if constexpr (MOST > 512) f(integral_constant<int, 32>{}, integral_constant<int, 32>{});
    }
}
template <typename F>
void with_values(int32_t type, uint32_t flags, F f) {
    with_type(type, [&](auto kind) {
        if ((flags & VM_PROBABILITIES) != 0) f(kind, std::true_type{});
        else f(kind, std::false_type{});
    });
}

dim3 grid_of(int64_t blocks) {
    if (blocks > INT32_MAX) throw std::string("too many rows for one call");
    return dim3(static_cast<unsigned>(blocks));
}
bool starts_on_16(const void* p, int64_t stride, int32_t type) {
    return aligned(p, 16) && stride * static_cast<int64_t>(element_size(type)) % 16 == 0;
}
// Whether lanes of a row take pieces of 16 bytes where its rows begin on them: all of a warp, two, or four that a row fills; else single elements,
// which are spread better. 1,000,000 rows, scores / gradient by elements and by pieces, us: 16 floats 36 / 48 and 19 / 28, 12 19 / 36 and
// 19 / 24, 32 40 / 70 and 35 / 50, 48 55 / 82 and 60 / 87, 96 97 / 151 and 111 / 166; bf16 16 21 / 40 and 19 / 21, 24 29 / 44 and 33 / 48, 32
// 39 / 53 and 29 / 45.
bool in_pieces(int lanes, int classes) {
    return lanes == 2 || lanes == WARP || (lanes == 4 && classes == 32);
}
// whether loads of 8 or 16 bytes fit every row of a few classes
bool starts_on_row(const void* x, int64_t stride, int classes, int32_t type) {
    const int64_t size = static_cast<int64_t>(element_size(type)), to = classes * size == 8 ? 8 : 16;
    return aligned(x, to) && stride * size % to == 0;
}

// Blocks of a cluster for one row, where rows are so few that SMs would have none, each with at least two pieces of 16 bytes a thread: the
// cluster's barrier and the joining cost 2 to 4 us. 4 x 131072 bf16 with five best: one block 18.9 us, 2 14.8, 4 10.9, 8 10.7; 32 x 65536
// 13.0, 2 10.9; but 64 x 32768 9.9, 2 10.7 and 290 x 60000 15.3, 2 18.3.
int blocks_of_row(int64_t rows, int64_t classes, int32_t type) {
    int n = 1;
    while (n < MOST_BLOCKS && rows * n * 2 <= SMS * 2 / 3 && classes * static_cast<int64_t>(element_size(type)) / 16 / (n * 2) >= 2 * STREAM_BLOCK) n *= 2;
    return n;
}

// Rows from which on a block of half the threads takes one, and pieces of 16 bytes up to which a warp alone does: what follows a row's last
// piece keeps fewer threads waiting. bf16 with five best by 32, 128 and 256 threads, us: 300 x 2048 8.9, 7.4, 8.9; 1024 x 9000 17.0, 13.1,
// 16.9; 1024 x 60000 91, 37.5, 39.7; 8000 x 2048 25, 40, 68; 4000 x 8192 25, 29, 40; 4000 x 12000 37.5, 35.3, 49.7; 600 x 3000 10.0, 8.9, 11.1.
constexpr int64_t HALF_BLOCKS_FROM = 2 * SMS, WARPS_FROM = 8 * SMS, WARP_UP_TO = 1024;

template <typename Kernel>
void launch_cluster(Kernel kernel, dim3 grid, int blocks, cudaStream_t q, const ScoresArgs& a) {
    cudaLaunchAttribute attribute{};
    attribute.id               = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = blocks;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    cudaLaunchConfig_t config{};
    config.gridDim  = grid;
    config.blockDim = dim3(STREAM_BLOCK);
    config.stream   = q;
    config.attrs    = &attribute;
    config.numAttrs = 1;
    VM_CUDA(cudaLaunchKernelEx(&config, kernel, a, blocks));
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
        if (!words_aligned({log_prob, entropy, log_sum, top_log_prob, top_index})) return fail(VM_ERR_INVALID_ARGUMENT, "an output is not aligned to its elements");
        if (log_prob != nullptr && labels == nullptr) return fail(VM_ERR_INVALID_ARGUMENT, "log_prob without labels");
        const OnDevice on(device);
        const ScoresArgs a{x, rows, classes, row_stride, labels, (flags & VM_LABELS_64) != 0, top, log_prob, entropy, log_sum, top_log_prob, top_index};
        const auto q       = static_cast<cudaStream_t>(stream);
        with_values(type, flags, [&](auto kind, auto probabilities) {
            using T = decltype(kind);
            constexpr bool P = decltype(probabilities)::value;
            if (classes <= MOST_OF_THREAD) {
                const bool pairs = top == 2 && aligned(top_log_prob, 8) && aligned(top_index, 8);
                with_classes(classes, [&](auto c) {
                    launch_kernel(k_scores_own_row<T, P, decltype(c)::value>, grid_of((rows + ROW_BLOCK - 1) / ROW_BLOCK), ROW_BLOCK, 0, q, false, a,
                                  starts_on_row(x, row_stride, classes, type), pairs);
                });
                return;
            }
            const auto launch_rows = [&](auto best, auto lanes, auto values) {
                constexpr int G = decltype(lanes)::value, E = decltype(values)::value;
                // as many rows for the same lanes as leave every SM two warps a scheduler
                const int64_t each  = std::clamp<int64_t>(rows * G / (WARP * 8 * SMS), 1, G);
                const int64_t block = ROWS_BLOCK / G * each;
                launch_kernel(k_scores_rows<T, P, decltype(best)::value, G, E>, grid_of((rows + block - 1) / block), ROWS_BLOCK, ROWS_BLOCK * top * sizeof(uint2), q, false, a,
                              in_pieces(G, classes) && starts_on_16(x, row_stride, type), static_cast<int>(each));
            };
            if (top > 0 && classes <= MOST_OF_LANES_TOP) return with_lanes<MOST_OF_LANES_TOP>(classes, [&](auto lanes, auto values) { launch_rows(std::true_type{}, lanes, values); });
            if (top == 0 && classes <= MOST_OF_LANES) return with_lanes<MOST_OF_LANES>(classes, [&](auto lanes, auto values) { launch_rows(std::false_type{}, lanes, values); });
            const int blocks     = blocks_of_row(rows, classes, type);
            const int64_t pieces = classes * static_cast<int64_t>(sizeof(T)) / 16;
            const auto launch = [&](auto best) {
                constexpr bool TOP = decltype(best)::value;
                if (blocks > 1) launch_cluster(k_scores_stream<T, P, TOP, STREAM_BLOCK, true>, grid_of(rows * blocks), blocks, q, a);
                else if (pieces <= STREAM_BLOCK || (pieces <= WARP_UP_TO && rows >= WARPS_FROM)) launch_kernel(k_scores_stream<T, P, TOP, WARP, false>, grid_of(rows), WARP, 0, q, false, a, 1);
                else if (rows < HALF_BLOCKS_FROM) launch_kernel(k_scores_stream<T, P, TOP, STREAM_BLOCK, false>, grid_of(rows), STREAM_BLOCK, 0, q, false, a, 1);
                else launch_kernel(k_scores_stream<T, P, TOP, STREAM_BLOCK / 2, false>, grid_of(rows), STREAM_BLOCK / 2, 0, q, false, a, 1);
            };
            if (top > 0) launch(std::true_type{});
            else launch(std::false_type{});
        });
    }
    catch (const std::string& refused) {
        return fail(VM_ERR_INVALID_ARGUMENT, refused);
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
        if (!words_aligned({entropy, log_sum, d_log_prob, d_entropy, d_log_sum})) return fail(VM_ERR_INVALID_ARGUMENT, "an input is not aligned to its elements");
        if (d_log_prob != nullptr && labels == nullptr) return fail(VM_ERR_INVALID_ARGUMENT, "d_log_prob without labels");
        if (d_entropy != nullptr && entropy == nullptr) return fail(VM_ERR_INVALID_ARGUMENT, "d_entropy without entropy");
        const OnDevice on(device);
        const ScoresGradArgs a{x, rows, classes, row_stride, labels, (flags & VM_LABELS_64) != 0, entropy, log_sum, d_log_prob, d_entropy, d_log_sum, dx, dx_row_stride};
        const auto q       = static_cast<cudaStream_t>(stream);
        with_values(type, flags, [&](auto kind, auto probabilities) {
            using T = decltype(kind);
            constexpr bool P = decltype(probabilities)::value;
            if (classes <= MOST_OF_THREAD) {
                const bool dense = dx_row_stride == classes && aligned(dx, 16);
                with_classes(classes, [&](auto c) {
                    launch_kernel(k_scores_grad_own_row<T, P, decltype(c)::value>, grid_of((rows + ROW_BLOCK - 1) / ROW_BLOCK), ROW_BLOCK, 0, q, false, a,
                                  starts_on_row(x, row_stride, classes, type), dense);
                });
                return;
            }
            if (classes <= MOST_OF_LANES_GRADIENT) {
                const bool wide = starts_on_16(x, row_stride, type) && starts_on_16(dx, dx_row_stride, type);
                with_lanes<MOST_OF_LANES_GRADIENT>(classes, [&](auto lanes, auto values) {
                    constexpr int G = decltype(lanes)::value, E = decltype(values)::value;
                    launch_kernel(k_scores_grad_rows<T, P, G, E>, grid_of((rows * G + ROW_BLOCK - 1) / ROW_BLOCK), ROW_BLOCK, 0, q, false, a, wide && in_pieces(G, classes));
                });
                return;
            }
            constexpr int PIECES = STREAM_BLOCK * STREAM_AHEAD;
            const int64_t pieces = classes / (16 / static_cast<int64_t>(sizeof(T))) + 2;  // one more where a row begins inside a piece
            const int64_t blocks = (pieces + PIECES - 1) / PIECES;
            launch_kernel(k_scores_grad_stream<T, P>, grid_of(rows * blocks), STREAM_BLOCK, 0, q, false, a, static_cast<int>(blocks));
        });
    }
    catch (const std::string& refused) {
        return fail(VM_ERR_INVALID_ARGUMENT, refused);
    }
    catch (...) {
        return status_of_exception();
    }
    return VM_OK;
}

}  // extern "C"
