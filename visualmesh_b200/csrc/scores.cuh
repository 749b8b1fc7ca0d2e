// Scores of rows of answers: log of the sum, log probability of a label, entropy, the largest values; and their gradient.
//
// With m = max_j v_j, t_j = v_j - m and e_j = exp t_j:
//   log_sum = m + log sum e_j,   entropy = log sum e_j - (sum e_j t_j) / (sum e_j),   log p_j = v_j - log_sum
// All of it in 32 bits: t_j <= 0, so no e_j overflows, and the largest is 1, so the sum is at least 1.
#pragma once

#include <cstdint>

#include "element.cuh"

namespace vm {
namespace answers {

constexpr int WARP = 32;

struct ScoresArgs {
    const void* x;
    int64_t rows;
    int32_t classes;
    int64_t row_stride;
    const void* labels;
    bool labels_64;
    int32_t top;
    float* log_prob;
    float* entropy;
    float* log_sum;
    float* top_log_prob;
    int32_t* top_index;
};

struct ScoresGradArgs {
    const void* x;
    int64_t rows;
    int32_t classes;
    int64_t row_stride;
    const void* labels;
    bool labels_64;
    const float* entropy;
    const float* log_sum;
    const float* d_log_prob;
    const float* d_entropy;
    const float* d_log_sum;
    void* dx;
    int64_t dx_row_stride;
};

__device__ __forceinline__ int64_t label_of(const void* labels, bool wide, int64_t row) {
    return wide ? static_cast<const int64_t*>(labels)[row] : static_cast<const int32_t*>(labels)[row];
}

template <bool PROBABILITIES>
__device__ __forceinline__ float value_of(float x) {
    return PROBABILITIES ? logf(x) : x;
}

// An order of all floats in which larger values have larger keys, equal ones (0 and -0 too) the lower index the larger key, and NaN
// the largest: 32 bits of value above 32 bits of index. No key is 0 or has all bits set.
__device__ __forceinline__ uint64_t key_of(float x, int32_t index) {
    const uint32_t bits  = __float_as_uint(x + 0.0f);
    const uint32_t order = x != x ? 0xFFFFFFFEu : (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
    return static_cast<uint64_t>(order) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ int32_t index_of_key(uint64_t key) {
    return static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(key));
}

// log p = (v - m) - log sum e: from the difference, not from log_sum, whose rounding grows with m. A class that is masked (-infinity)
// stays that, whatever the rest of the row.
__device__ __forceinline__ float log_prob_of(float v, float m, float log_of_sum) {
    return v == -INFINITY && m < INFINITY ? -INFINITY : (v - m) - log_of_sum;
}

__device__ __forceinline__ float warp_max(float v) {
    for (int d = WARP / 2; d > 0; d /= 2) {
        const float o = __shfl_xor_sync(~0u, v, d);
        v = (o > v || o != o) ? o : v;
    }
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
    for (int d = WARP / 2; d > 0; d /= 2) v += __shfl_xor_sync(~0u, v, d);
    return v;
}

// A warp per row.
template <typename T, bool PROBABILITIES>
__global__ void __launch_bounds__(256) k_scores(const ScoresArgs a) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / WARP) + threadIdx.x / WARP;
    if (row >= a.rows) return;
    const int lane = threadIdx.x % WARP;
    const T* x     = static_cast<const T*>(a.x) + row * a.row_stride;

    float m = -INFINITY;
    for (int32_t j = lane; j < a.classes; j += WARP) {
        const float v = value_of<PROBABILITIES>(to_float(x[j]));
        m = (v > m || v != v) ? v : m;
        if (m != m) break;
    }
    m = warp_max(m);
    float sum = 0.0f, weighted = 0.0f;
    if (m > -INFINITY && m < INFINITY) {
        for (int32_t j = lane; j < a.classes; j += WARP) {
            const float v = value_of<PROBABILITIES>(to_float(x[j]));
            if (v == -INFINITY) continue;
            const float t = fmaxf(v - m, -1000.0f), e = __expf(t);  // e is 0 there, and 0 * -infinity would not be
            sum += e;
            weighted = fmaf(e, t, weighted);
        }
        sum      = warp_sum(sum);
        weighted = warp_sum(weighted);
    }
    float l = 0.0f, log_sum = -INFINITY, entropy = 0.0f;
    if (!(m < INFINITY)) l = log_sum = entropy = NAN;
    else if (m > -INFINITY) {
        l       = logf(sum);
        log_sum = m + l;
        entropy = l - weighted / sum;
    }
    if (lane == 0) {
        if (a.log_sum != nullptr) a.log_sum[row] = log_sum;
        if (a.entropy != nullptr) a.entropy[row] = entropy;
        if (a.log_prob != nullptr) {
            const int64_t label = label_of(a.labels, a.labels_64, row);
            float lp = 0.0f;
            if (label != -1) lp = label < 0 || label >= a.classes ? NAN : log_prob_of(value_of<PROBABILITIES>(to_float(x[label])), m, l);
            a.log_prob[row] = lp;
        }
    }
    uint64_t below = ~0ull;
    for (int k = 0; k < a.top; ++k) {
        uint64_t best = 0;
        for (int32_t j = lane; j < a.classes; j += WARP) {
            const uint64_t key = key_of(to_float(x[j]), j);
            if (key < below && key > best) best = key;
        }
        for (int d = WARP / 2; d > 0; d /= 2) {
            const uint64_t o = __shfl_xor_sync(~0u, best, d);
            best = o > best ? o : best;
        }
        below = best;
        if (lane == 0) {
            const int32_t j = index_of_key(best);
            a.top_index[row * a.top + k]    = j;
            a.top_log_prob[row * a.top + k] = log_prob_of(value_of<PROBABILITIES>(to_float(x[j])), m, l);
        }
    }
}

// The gradient is one pass over the elements once the row's sums are known.
template <typename T, bool PROBABILITIES>
__global__ void __launch_bounds__(256) k_scores_grad(const ScoresGradArgs a) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / WARP) + threadIdx.x / WARP;
    if (row >= a.rows) return;
    const int lane = threadIdx.x % WARP;
    const T* x     = static_cast<const T*>(a.x) + row * a.row_stride;
    T* dx          = static_cast<T*>(a.dx) + row * a.dx_row_stride;

    const float log_sum = a.log_sum[row];
    float d_label = 0.0f;
    int64_t label = -1;
    if (a.d_log_prob != nullptr) {
        label = label_of(a.labels, a.labels_64, row);
        if (label != -1) d_label = label < 0 || label >= a.classes ? NAN : a.d_log_prob[row];
    }
    const float d_entropy = a.d_entropy != nullptr ? a.d_entropy[row] : 0.0f;
    const float entropy   = a.d_entropy != nullptr ? a.entropy[row] : 0.0f;
    const float constant  = log_sum != log_sum ? NAN : (a.d_log_sum != nullptr ? a.d_log_sum[row] : 0.0f) - d_label;
    const float one_over  = PROBABILITIES ? 1.0f / __expf(log_sum) : 0.0f;
    for (int32_t j = lane; j < a.classes; j += WARP) {
        const float p = to_float(x[j]);
        const float v = value_of<PROBABILITIES>(p);
        float d = 0.0f;
        if (v != -INFINITY) {
            const float lp = fmaxf(v - log_sum, -1000.0f);  // p is 0 there, and 0 * -infinity would not be
            d = (constant - d_entropy * (lp + entropy)) * (PROBABILITIES ? one_over : __expf(lp));
            if (j == label) d += PROBABILITIES ? d_label / p : d_label;
        }
        dx[j] = from_float<T>(d);
    }
}

}  // namespace answers
}  // namespace vm
