// Scores of rows of answers: log of the sum, log probability of a label, entropy, the largest values; and their gradient.
//
// With m = max_j v_j, t_j = v_j - m and e_j = exp t_j:
//   log_sum = m + log sum e_j,   entropy = log sum e_j - (sum e_j t_j) / (sum e_j),   log p_j = v_j - log_sum
// All of it in 32 bits: t_j <= 0, so no e_j overflows, and the largest is 1, so the sum is at least 1. Probabilities need no maximum and
// no exponential: with s = sum x_j, log p_j = log x_j - log s and entropy = log s - (sum x_j log x_j) / s.
#pragma once

#include <cooperative_groups.h>

#include <cstdint>
#include <cstring>
#include <type_traits>

#include "../../include/vmcuda.h"
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
// SCALE x log x for the sum of an entropy: the fast logarithm is off by 2^-21.4 near 1 and by two units in the last place elsewhere, which times
// a probability is what rounding the entropy would be. (Log probabilities themselves need all of their digits near 1.)
constexpr float SCALE = 16777216.0f;  // 2^24: a product with a number below the normal ones would lose its digits
__device__ __forceinline__ float times_log(float x) {
    return x == 0.0f ? 0.0f : SCALE * x * __logf(x);
}

// An order of all floats in which larger values have larger numbers, 0 and -0 the same, and NaN the largest (adding 0 makes one zero of both
// and one NaN, 0x7FFFFFFF, of all). No value has 0. With the index below it, the lower the larger: an order of a row's classes.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t bits = __float_as_uint(x + 0.0f);
    return bits ^ (static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of_order(uint32_t order) {
    return __uint_as_float(order ^ (~static_cast<uint32_t>(static_cast<int32_t>(order) >> 31) | 0x80000000u));
}
__device__ __forceinline__ uint64_t key_of(float x, int32_t index) {
    return static_cast<uint64_t>(order_of(x)) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ int32_t index_of_key(uint64_t key) {
    return static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(key));
}

// What a row's values come to. Logits: m their maximum, s = sum e^t and w = sum e^t t with t = v - m. Probabilities: m = 0, s = sum x,
// w = SCALE sum x log x. A value that makes the row no distribution leaves NaN in s or w.
struct Sums {
    float m, s, w;
};
constexpr float NO_EXPONENT = -1000.0f;  // e^t is 0 there, and 0 times -infinity would not be
__device__ __forceinline__ float bounded(float t) {
    return fmaxf(t, NO_EXPONENT);
}
__device__ __forceinline__ float bounded_or_nan(float t) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(t), "f"(NO_EXPONENT));
    return r;
}
// The results of a row from its sums; log p of one of its values.
struct Row {
    float m, l, log_sum, entropy;
};
template <bool PROBABILITIES>
__device__ __forceinline__ Row row_of(const Sums& q) {
    Row r{q.m, 0.0f, -INFINITY, 0.0f};
    // a sum of probabilities that leaves room for SCALE and for a logarithm
    if (!(q.s <= (PROBABILITIES ? 7.92281625e28f : 3.402823466e38f)) || q.w != q.w) r.m = r.l = r.log_sum = r.entropy = NAN;
    else if (q.s > 0.0f) {
        // a softmax's sum is one but for roundings, d: the next term of the series is d^4 / 4
        const float d = q.s - 1.0f;
        r.l           = PROBABILITIES && fabsf(d) < 0.00390625f ? d * fmaf(d, fmaf(d, 0.333333333f, -0.5f), 1.0f) : logf(q.s);
        r.log_sum     = q.m + r.l;
        r.entropy     = r.l - __fdividef(q.w, PROBABILITIES ? SCALE * q.s : q.s);
    }
    return r;
}
// log p = (v - m) - log s: from the difference, not from log_sum, whose rounding grows with m. m is finite in a row that has a distribution,
// so a class that is masked (-infinity) stays that.
__device__ __forceinline__ float log_prob_of(float v, const Row& r) {
    return (v - r.m) - r.l;
}
template <typename T, bool PROBABILITIES>
__device__ __forceinline__ void write_row(const ScoresArgs& a, int64_t row, const T* x, const Row& r) {
    if (a.log_sum != nullptr) a.log_sum[row] = r.log_sum;
    if (a.entropy != nullptr) a.entropy[row] = r.entropy;
    if (a.log_prob != nullptr) {
        const int64_t label = label_of(a.labels, a.labels_64, row);
        float lp = 0.0f;
        if (label != -1) lp = label < 0 || label >= a.classes ? NAN : log_prob_of(value_of<PROBABILITIES>(to_float(x[label])), r);
        a.log_prob[row] = lp;
    }
}
template <bool PROBABILITIES>
__device__ __forceinline__ void write_top(const ScoresArgs& a, int64_t row, int k, uint32_t order, int32_t index, const Row& r) {
    a.top_index[row * a.top + k]    = index;
    a.top_log_prob[row * a.top + k] = log_prob_of(value_of<PROBABILITIES>(value_of_order(order)), r);
}

constexpr int ROW_BLOCK = 256, ROWS_BLOCK = 128;

// ---- up to 8 classes: a thread per row -----------------------------------------------------------------------------------------
// C values in registers, every loop over them unrolled. Bound by instructions rather than bytes (48 bytes a row of three classes with
// their two best are 2.1 cycles of an SM's share of the memory, 270 instructions of its lanes), so each logarithm is taken once, for the sum, the
// label and the best classes alike, and a class's place in the order is counted (C (C - 1) / 2 comparisons) instead of searched for.
// 4,480,064 rows of three floats with two best: 46 us, 33 at the memory's rate.
template <typename T, int C>
__device__ __forceinline__ void load_row(const T* x, bool wide, float (&to)[C]) {
    T e[C];
    constexpr int BYTES = C * sizeof(T);
    if constexpr (BYTES == 8 || BYTES % 16 == 0) {
        if (wide) {
            if constexpr (BYTES == 8) {
                const uint2 raw = *reinterpret_cast<const uint2*>(x);
                memcpy(e, &raw, 8);
            }
            else {
#pragma unroll
                for (int i = 0; i < BYTES / 16; ++i) {
                    const uint4 raw = reinterpret_cast<const uint4*>(x)[i];
                    memcpy(reinterpret_cast<unsigned char*>(e) + 16 * i, &raw, 16);
                }
            }
#pragma unroll
            for (int k = 0; k < C; ++k) to[k] = to_float(e[k]);
            return;
        }
    }
#pragma unroll
    for (int k = 0; k < C; ++k) to[k] = to_float(x[k]);
}

template <typename T, bool PROBABILITIES, int C>
__global__ void __launch_bounds__(ROW_BLOCK) k_scores_own_row(const ScoresArgs a, bool wide, bool pairs) {
    __shared__ uint2 tops[C > 2 ? ROW_BLOCK * C : 1];
    const int first_row = blockIdx.x * ROW_BLOCK, row = first_row + threadIdx.x;  // rows < 2^31, and so are those of the last block
    const int rows      = static_cast<int>(a.rows - first_row < ROW_BLOCK ? a.rows - first_row : ROW_BLOCK);
    if (row < a.rows) {
        float x[C], v[C];
        load_row<T, C>(static_cast<const T*>(a.x) + row * a.row_stride, wide, x);
        const int64_t label = a.log_prob != nullptr ? label_of(a.labels, a.labels_64, row) : -1;
        const int labelled  = label >= 0 && label < C ? static_cast<int>(label) : label == -1 ? -1 : -2;

        Sums q{0.0f, 0.0f, 0.0f};
        if constexpr (PROBABILITIES) {
#pragma unroll
            for (int k = 0; k < C; ++k) {
                v[k] = logf(x[k]);
                q.s += x[k];
                q.w = fmaf(SCALE * x[k], bounded_or_nan(v[k]), q.w);
            }
        }
        else {
            q.m = -INFINITY;
#pragma unroll
            for (int k = 0; k < C; ++k) v[k] = x[k], q.m = fmaxf(q.m, v[k]);
            if (q.m == -INFINITY) q.m = 0.0f;  // then nothing is left, or only NaN
#pragma unroll
            for (int k = 0; k < C; ++k) {
                const float t = v[k] - q.m, e = exp_of(t);
                q.s += e;
                q.w = fmaf(e, bounded(t), q.w);
            }
        }
        const Row r = row_of<PROBABILITIES>(q);
        if (a.log_sum != nullptr) a.log_sum[row] = r.log_sum;
        if (a.entropy != nullptr) a.entropy[row] = r.entropy;
#pragma unroll
        for (int k = 0; k < C; ++k) v[k] = log_prob_of(v[k], r);
        if (a.log_prob != nullptr) {
            float lp = labelled == -1 ? 0.0f : NAN;
#pragma unroll
            for (int k = 0; k < C; ++k)
                if (labelled == k) lp = v[k];
            a.log_prob[row] = lp;
        }
        if (a.top > 0) {
            uint32_t order[C];
            if (PROBABILITIES && r.l == r.l) {
#pragma unroll
                for (int k = 0; k < C; ++k) order[k] = __float_as_uint(x[k] + 0.0f);  // no negative ones in a row that has a distribution
            }
            else {
#pragma unroll
                for (int k = 0; k < C; ++k) order[k] = order_of(x[k]);
            }
            int place[C];
#pragma unroll
            for (int k = 0; k < C; ++k) place[k] = 0;
#pragma unroll
            for (int k = 0; k < C; ++k) {
#pragma unroll
                for (int j = k + 1; j < C; ++j) {
                    const bool behind = order[j] > order[k];
                    place[k] += behind, place[j] += !behind;
                }
            }
            const int64_t first = static_cast<int64_t>(row) * a.top;
            if (a.top <= 2) {
                float lp[2];
                int index[2];
#pragma unroll
                for (int k = 0; k < C; ++k) {
                    if (place[k] == 0) lp[0] = v[k], index[0] = k;
                    if (place[k] == 1) lp[1] = v[k], index[1] = k;
                }
                if (pairs) {  // two at once: half of the stores, which are what bounds rows of few classes
                    *reinterpret_cast<float2*>(a.top_log_prob + first) = make_float2(lp[0], lp[1]);
                    *reinterpret_cast<int2*>(a.top_index + first)      = make_int2(index[0], index[1]);
                }
                else {
                    a.top_log_prob[first] = lp[0], a.top_index[first] = index[0];
                    if (a.top == 2) a.top_log_prob[first + 1] = lp[1], a.top_index[first + 1] = index[1];
                }
            }
            else if constexpr (C > 2) {  // every class puts itself where it stands in the order
#pragma unroll
                for (int k = 0; k < C; ++k)
                    if (place[k] < a.top) tops[threadIdx.x * a.top + place[k]] = make_uint2(__float_as_uint(v[k]), k);
            }
        }
    }
    if (C > 2 && a.top > 2) {  // the rows of a block lie side by side, and so do their best classes
        __syncthreads();
        const int64_t first = static_cast<int64_t>(first_row) * a.top;
        for (int i = threadIdx.x; i < rows * a.top; i += ROW_BLOCK) a.top_log_prob[first + i] = __uint_as_float(tops[i].x), a.top_index[first + i] = static_cast<int32_t>(tops[i].y);
    }
}

// ---- up to 256 classes (gradients 1024): G lanes per row, E values a lane in registers ---------------------------------------------------------
// Lane l of a row has the values l, l + G, l + 2 G, ..., or (wide, rows that begin on 16 bytes) the same with pieces of 16 bytes. 8 and 16 lanes
// never do: their code for both would hold more registers (64 floats with two best 111 -> 125 us), and they gain 10 % at most.
template <typename T, int G, int E>
struct RowLoad {
    static constexpr int PIECE = 16 / sizeof(T);
    static constexpr bool MAY  = G <= 4 || G == WARP;
    __device__ static __forceinline__ int index(bool wide, int lane, int i) {
        return MAY && wide ? (i / PIECE * G + lane) * PIECE + i % PIECE : i * G + lane;
    }
    __device__ static __forceinline__ void load(const T* x, int classes, bool wide, int lane, float (&to)[E]) {
        if constexpr (MAY) {
            if (wide) {
#pragma unroll
                for (int i = 0; i < E; i += PIECE) {
                    const int j = index(true, lane, i);
                    T e[PIECE];
                    if (j + PIECE <= classes) {
                        const uint4 raw = *reinterpret_cast<const uint4*>(x + j);
                        memcpy(e, &raw, 16);
#pragma unroll
                        for (int k = 0; k < PIECE; ++k) to[i + k] = to_float(e[k]);
                    }
                    else {
#pragma unroll
                        for (int k = 0; k < PIECE; ++k) to[i + k] = j + k < classes ? to_float(x[j + k]) : 0.0f;
                    }
                }
                return;
            }
        }
#pragma unroll
        for (int i = 0; i < E; ++i) to[i] = i * G + lane < classes ? to_float(x[i * G + lane]) : 0.0f;
    }
};

template <int G, typename F>
__device__ __forceinline__ void over_lanes(F f) {
#pragma unroll
    for (int d = G / 2; d > 0; d /= 2) f(d);
}

// Order and index of up to 256 values of a 16-bit type in one number: such a value has no more than the upper 19 bits of a float. Never 0.
__device__ __forceinline__ uint32_t short_key_of(float x, int index) {
    return ((order_of(x) >> 5) & 0x07FFFF00u) | (255u - static_cast<uint32_t>(index));
}
__device__ __forceinline__ uint32_t order_of_short_key(uint32_t key) {
    const uint32_t upper = (key & 0x07FFFF00u) << 5;
    return (upper & 0x80000000u) ? upper : upper | 0x1FFFu;  // those of negative values are inverted, with ones below
}

// The lanes of a row take `each` rows one after another (G of them: a warp has 32 neighbouring rows; few rows: 1), and every lane keeps the sums
// of one: what follows the sums (logarithms, labels, results) is then done once for all of them by all lanes, and the results lie side by
// side. The next rows are read meanwhile.
// The best classes are taken one by one, the largest of the lanes' (value, index) each time; of 16-bit values both are one number of 32 bits.
// Bound by instructions: 100,000 rows of 128 floats 15 us (8 at the memory's rate), with five best 50. `each` rows instead of one: 300,000 rows of
// 60 floats 27 -> 19 us, with two best 54 -> 38.
template <typename T, bool PROBABILITIES, bool TOP, int G, int E>
__global__ void __launch_bounds__(ROWS_BLOCK) k_scores_rows(const ScoresArgs a, bool wide, int each) {
    extern __shared__ uint2 tops[];  // [warps][32][top]: order and index
    const int64_t warp = static_cast<int64_t>(blockIdx.x) * (ROWS_BLOCK / WARP) + threadIdx.x / WARP;
    const int lane = threadIdx.x % WARP, l = lane % G;
    const int64_t first = (warp * (WARP / G) + lane / G) * each;  // of the rows of these lanes
    uint2* const warp_tops = tops + threadIdx.x / WARP * WARP * a.top;
    using Load             = RowLoad<T, G, E>;
    const auto load        = [&](int i, float (&to)[E]) {
        const int64_t row = first + i;
        Load::load(static_cast<const T*>(a.x) + (row < a.rows ? row : 0) * a.row_stride, row < a.rows ? a.classes : 0, wide, l, to);
    };
    Sums mine{0.0f, 0.0f, 0.0f};
    float v[E];
    load(0, v);
    for (int i = 0; i < each; ++i) {
        float next[E];
        if (i + 1 < each) load(i + 1, next);
        Sums q{0.0f, 0.0f, 0.0f};
        if constexpr (PROBABILITIES) {
#pragma unroll
            for (int j = 0; j < E; ++j) {
                if (Load::index(wide, l, j) < a.classes) {
                    q.s += v[j];
                    q.w += times_log(v[j]);
                }
            }
        }
        else {
            q.m = -INFINITY;
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (Load::index(wide, l, j) < a.classes) q.m = fmaxf(q.m, v[j]);
            over_lanes<G>([&](int d) { q.m = fmaxf(q.m, __shfl_xor_sync(~0u, q.m, d)); });
            if (q.m == -INFINITY) q.m = 0.0f;  // then nothing is left, or only NaN
#pragma unroll
            for (int j = 0; j < E; ++j) {
                if (Load::index(wide, l, j) < a.classes) {
                    const float t = v[j] - q.m, e = exp_of(t);
                    q.s += e;
                    q.w = fmaf(e, bounded(t), q.w);
                }
            }
        }
        over_lanes<G>([&](int d) {
            q.s += __shfl_xor_sync(~0u, q.s, d);
            q.w += __shfl_xor_sync(~0u, q.w, d);
        });
        if (l == i) mine = q;

        if constexpr (TOP) {
            uint2* const to = warp_tops + (lane / G * each + i) * a.top;
            // the first is a value that equals the maximum (but in a row with NaN, which the maximum does not show)
            int k = 0;
            if (!PROBABILITIES && sizeof(T) == 4 && a.top == 1 && !__any_sync(~0u, q.s != q.s)) {
                const float m = q.s > 0.0f ? q.m : -INFINITY;
                int at        = INT32_MAX;
#pragma unroll
                for (int j = E - 1; j >= 0; --j)
                    if (v[j] == m && Load::index(wide, l, j) < a.classes) at = Load::index(wide, l, j);
                if constexpr (G == WARP) at = __reduce_min_sync(~0u, at);
                else over_lanes<G>([&](int d) { at = min(at, __shfl_xor_sync(~0u, at, d)); });
                if (l == 0) to[0] = make_uint2(order_of(m), at);
                k = 1;
            }
            if (k < a.top) {
                uint32_t key[E];  // 0: not there, or taken
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    const int at = Load::index(wide, l, j);
                    key[j]       = at >= a.classes ? 0 : sizeof(T) == 2 ? short_key_of(v[j], at) : order_of(v[j]);
                }
                for (; k < a.top; ++k) {
                    uint32_t best = key[0];
#pragma unroll
                    for (int j = 1; j < E; ++j) best = max(best, key[j]);
                    if constexpr (G == WARP) best = __reduce_max_sync(~0u, best);
                    else over_lanes<G>([&](int d) { best = max(best, __shfl_xor_sync(~0u, best, d)); });
                    if constexpr (sizeof(T) == 2) {
#pragma unroll
                        for (int j = 0; j < E; ++j)
                            if (key[j] == best) key[j] = 0;
                        if (l == 0) to[k] = make_uint2(order_of_short_key(best), 255u - (best & 255u));
                    }
                    else {
                        int at = INT32_MAX;
#pragma unroll
                        for (int j = E - 1; j >= 0; --j)  // a lane's indices rise with j: the first of equals stays
                            if (key[j] == best) at = Load::index(wide, l, j);
                        if constexpr (G == WARP) at = __reduce_min_sync(~0u, at);
                        else over_lanes<G>([&](int d) { at = min(at, __shfl_xor_sync(~0u, at, d)); });
#pragma unroll
                        for (int j = 0; j < E; ++j)
                            if (Load::index(wide, l, j) == at) key[j] = 0;
                        if (l == 0) to[k] = make_uint2(best, at);
                    }
                }
            }
        }
        if (i + 1 < each) {
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = next[j];
        }
    }
    __syncwarp();
    const int64_t row = first + l;
    if (l < each && row < a.rows) {
        const Row r = row_of<PROBABILITIES>(mine);
        write_row<T, PROBABILITIES>(a, row, static_cast<const T*>(a.x) + row * a.row_stride, r);
        uint2* const own = warp_tops + (lane / G * each + l) * a.top;
        for (int k = 0; TOP && k < a.top; ++k) own[k].x = __float_as_uint(log_prob_of(value_of<PROBABILITIES>(value_of_order(own[k].x)), r));
    }
    if constexpr (TOP) {  // the rows of a warp lie side by side, and so do their best classes
        __syncwarp();
        const int64_t begin = warp * (WARP / G) * each, rows = min(static_cast<int64_t>(WARP / G * each), a.rows - begin);
        for (int i = lane; i < rows * a.top; i += WARP) {
            a.top_log_prob[begin * a.top + i] = __uint_as_float(warp_tops[i].x);
            a.top_index[begin * a.top + i]    = static_cast<int32_t>(warp_tops[i].y);
        }
    }
}

// ---- more classes: blocks per row ----------------------------------------------------------------------------------------------
// One pass over the row in pieces of 16 bytes (the row's first and last may be shorter): a thread keeps its running maximum with the sums
// below it, and which of its pieces held the maximum. The `top` largest then need no second pass: with the threads' maxima in order (by
// value, then by place), every one of the row's `top` largest values lies in a thread whose maximum is among the first `top`, and is at
// least the last of those. So `top` threads' pieces are read again (from the cache), what is that large is
// collected and the largest of it taken. Where that is more than there is room for (many of the largest in one thread's pieces) or the row holds
// NaN, the row is searched `top` times instead.
// Few rows: a cluster of blocks shares a row, and the first of them joins their results through its shared memory.
// 4099 rows of 32771 bf16: 62 us, with five best 72, 41 at the memory's rate; a plain sum over the same rows takes 59. Two thirds of the issue
// slots and of the exponentials' pipe are taken; loads a step ahead in registers moved it by -4 to +2 % (fewer blocks fit). 4 x 131072 fp16 with
// 20 best: 12.3 us, of which 4 are a launch and 4 the cluster's two barriers and the joining.
constexpr int STREAM_BLOCK = 256;
constexpr int STREAM_AHEAD = 4;    // pieces that a thread has under way
constexpr int CANDIDATES   = 256;  // top * (values of a piece) at least: that many can tie
constexpr int MOST_BLOCKS  = 8;    // of a cluster
static_assert(VM_MAX_TOP * 8 <= CANDIDATES && VM_MAX_TOP * MOST_BLOCKS <= CANDIDATES, "room for ties within pieces, and for every block's best");

template <typename T>
struct Pieces {
    static constexpr int N = 16 / sizeof(T);
    const T* x;     // the row
    int classes;
    int before;     // values of piece 0 that lie in front of the row
    int64_t count;  // pieces that hold values of the row
    __device__ __forceinline__ Pieces(const T* row, int n) : x(row), classes(n) {
        before = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
        count  = (static_cast<int64_t>(before) + n + N - 1) / N;
    }
    // index of the first value of a piece in the row; those outside 0..classes-1 are not the row's
    __device__ __forceinline__ int64_t first(int64_t piece) const {
        return piece * N - before;
    }
    __device__ __forceinline__ uint4 load(int64_t piece, T outside) const {
        const int64_t j = first(piece);
        if (j >= 0 && j + N <= classes) return *reinterpret_cast<const uint4*>(x + j);
        T e[N];
#pragma unroll
        for (int k = 0; k < N; ++k) e[k] = j + k >= 0 && j + k < classes ? x[j + k] : outside;
        uint4 raw;
        memcpy(&raw, e, 16);
        return raw;
    }
};
template <typename T>
__device__ __forceinline__ void values_of(const uint4& raw, float (&to)[16 / sizeof(T)]) {
    T e[16 / sizeof(T)];
    memcpy(e, &raw, 16);
#pragma unroll
    for (int k = 0; k < 16 / static_cast<int>(sizeof(T)); ++k) to[k] = to_float(e[k]);
}

// The `top` largest of `n` different keys (0: none) in shared memory, in order, by one warp: every lane sorts its own, and the largest of their
// first is taken away `top` times.
template <int K>
__device__ __forceinline__ void largest_of_lanes(const uint64_t* keys, int n, int top, uint64_t* into) {
    const int lane = threadIdx.x % WARP;
    uint64_t held[K];
#pragma unroll
    for (int i = 0; i < K; ++i) held[i] = i * WARP + lane < n ? keys[i * WARP + lane] : 0;
    if constexpr (K == 4) {  // Batcher's merge sort, of four and of eight
        constexpr int PAIRS[5][2] = {{0, 1}, {2, 3}, {0, 2}, {1, 3}, {1, 2}};
#pragma unroll
        for (int i = 0; i < 5; ++i) {
            const uint64_t x = held[PAIRS[i][0]], y = held[PAIRS[i][1]];
            held[PAIRS[i][0]] = x > y ? x : y;
            held[PAIRS[i][1]] = x > y ? y : x;
        }
    }
    else if constexpr (K > 1) {
        static_assert(K == 8, "the pairs below sort eight");
        constexpr int PAIRS[19][2] = {{0, 1}, {2, 3}, {4, 5}, {6, 7}, {0, 2}, {1, 3}, {4, 6}, {5, 7}, {1, 2}, {5, 6}, {0, 4}, {1, 5}, {2, 6}, {3, 7}, {2, 4}, {3, 5}, {1, 2}, {3, 4}, {5, 6}};
#pragma unroll
        for (int i = 0; i < 19; ++i) {
            const uint64_t x = held[PAIRS[i][0]], y = held[PAIRS[i][1]];
            held[PAIRS[i][0]] = x > y ? x : y;
            held[PAIRS[i][1]] = x > y ? y : x;
        }
    }
    for (int k = 0; k < top; ++k) {
        const uint32_t high = __reduce_max_sync(~0u, static_cast<uint32_t>(held[0] >> 32));
        const bool equal    = static_cast<uint32_t>(held[0] >> 32) == high;
        const uint32_t low  = __reduce_max_sync(~0u, equal ? static_cast<uint32_t>(held[0]) : 0);
        if (equal && static_cast<uint32_t>(held[0]) == low) {
            into[k] = held[0];
#pragma unroll
            for (int i = 0; i + 1 < K; ++i) held[i] = held[i + 1];
            held[K - 1] = 0;
        }
    }
}
__device__ __forceinline__ void largest_keys(const uint64_t* keys, int n, int top, uint64_t* into) {
    if (n <= WARP) largest_of_lanes<1>(keys, n, top, into);
    else if (n <= 4 * WARP) largest_of_lanes<4>(keys, n, top, into);
    else largest_of_lanes<CANDIDATES / WARP>(keys, n, top, into);
}

struct StreamShared {
    Sums warps[STREAM_BLOCK / WARP];
    uint64_t keys[CANDIDATES];      // the threads' maxima, then what may be among the largest
    uint64_t best[VM_MAX_TOP];      // of this block
    uint64_t searched[STREAM_BLOCK / WARP];
    int found;
    // of the cluster, in its first block
    Sums sums[MOST_BLOCKS];
    uint64_t bests[MOST_BLOCKS * VM_MAX_TOP];
};
static_assert(STREAM_BLOCK <= CANDIDATES, "the threads' maxima are chosen from as candidates are");

// The sums of long rows of logits are kept in powers of two, for pairs of values: with M = m L, L = log2 e in 32 bits, t_j = x_j L - M (one rounding
// for a pair), s = sum 2^t_j and w = sum 2^t_j t_j. What rounding m L to M moved, rho = m L - M, is put right in the row's results:
// log sum e^(x_j - m) = log s - rho log 2. That holds while rho is small: it grows with m, to 2^-7 at BELOW, and at 10^10 2^rho is infinite. So no
// maximum counts that lies outside of ABOVE..BELOW, a thread's own no more than the row's: maxima begin at START, below which a thread that has
// seen nothing but masked values stays, values are not let below LOW, where 2^t is 0 beside any of them, and a row whose maximum is not inside
// (padding, or all masked by a finite number) is summed again in the way of the short rows: 4 x 131072 bf16, one of them padding, 43 us instead of 8;
// 4099 x 32771, a quarter padding, 97 instead of 64.
constexpr float LOG2_E = 1.44269504f, LOG_2 = 0.693147181f;
template <typename T>
struct Range {  // numbers of the type
    static constexpr float LOW = -131072.0f, START = -65536.0f, ABOVE = START, BELOW = 131072.0f;
};
template <>
struct Range<__half> {
    static constexpr float LOW = -65504.0f, START = LOW, ABOVE = -64000.0f, BELOW = 131072.0f;
};
__device__ __forceinline__ Sums joined_by_two(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m), da = a.m * LOG2_E - m * LOG2_E, db = b.m * LOG2_E - m * LOG2_E, fa = exp2_of(da), fb = exp2_of(db);
    return Sums{m, fmaf(a.s, fa, b.s * fb), fmaf(fmaf(a.s, da, a.w), fa, fmaf(b.s, db, b.w) * fb)};
}
template <bool PROBABILITIES>
__device__ __forceinline__ Sums joined_stream(const Sums& a, const Sums& b) {
    return PROBABILITIES ? Sums{0.0f, a.s + b.s, a.w + b.w} : joined_by_two(a, b);
}
__device__ __forceinline__ Row row_by_two(const Sums& q) {
    if (!(q.s < INFINITY) || q.w != q.w) return Row{NAN, NAN, NAN, NAN};
    const float rho = fmaf(q.m, LOG2_E, -(q.m * LOG2_E)), l = logf(q.s) - rho * LOG_2;
    return Row{q.m, l, q.m + l, l - (__fdividef(q.w, q.s) - rho) * LOG_2};
}

// Of a warp's lanes, for all of them.
template <int LANES, typename Join>
__device__ __forceinline__ Sums joined_lanes(Sums q, Join join) {
    over_lanes<LANES>([&](int d) { q = join(q, Sums{__shfl_xor_sync(~0u, q.m, d), __shfl_xor_sync(~0u, q.s, d), __shfl_xor_sync(~0u, q.w, d)}); });
    return q;
}

// A row of logits in the way of the short rows, by all threads of a block: first its maximum, then its sums. `warps`: a place for each warp.
template <typename T, int BLOCK>
__device__ __noinline__ Row row_again(const Pieces<T>& pieces, Sums* warps) {
    constexpr int N = Pieces<T>::N;
    const auto over = [&](auto f) {
        for (int64_t p = threadIdx.x; p < pieces.count; p += BLOCK) {
            float v[N];
            values_of<T>(pieces.load(p, from_float<T>(-INFINITY)), v);
            for (int k = 0; k < N; ++k) f(v[k]);
        }
    };
    const auto joined = [&](Sums q, auto join) {
        q = joined_lanes<WARP>(q, join);
        if (BLOCK == WARP) return q;
        __syncthreads();  // what stood there is read
        if (threadIdx.x % WARP == 0) warps[threadIdx.x / WARP] = q;
        __syncthreads();
        return joined_lanes<BLOCK / WARP>(warps[threadIdx.x % (BLOCK / WARP)], join);
    };
    float m = -INFINITY;
    over([&](float v) { m = fmaxf(m, v); });
    m = joined(Sums{m, 0.0f, 0.0f}, [](const Sums& a, const Sums& b) { return Sums{fmaxf(a.m, b.m), 0.0f, 0.0f}; }).m;
    Sums q{m == -INFINITY ? 0.0f : m, 0.0f, 0.0f};  // nothing is left: any number will do
    over([&](float v) {
        const float t = v - q.m, e = exp_of(t);
        q.s += e;
        q.w = fmaf(e, bounded(t), q.w);
    });
    return row_of<false>(joined(q, [](const Sums& a, const Sums& b) { return Sums{a.m, a.s + b.s, a.w + b.w}; }));
}

template <typename T, bool PROBABILITIES, bool TOP, int BLOCK, bool CLUSTER>
__global__ void __launch_bounds__(BLOCK) k_scores_stream(const ScoresArgs a, int blocks) {
    namespace cg = cooperative_groups;
    __shared__ StreamShared shared;
    const int rank    = CLUSTER ? blockIdx.x % blocks : 0;
    const int64_t row = CLUSTER ? blockIdx.x / blocks : blockIdx.x;
    const int lane = threadIdx.x % WARP, warp = threadIdx.x / WARP;
    const T* x = static_cast<const T*>(a.x) + row * a.row_stride;
    const Pieces<T> pieces(x, a.classes);
    constexpr int N     = Pieces<T>::N;
    const int64_t share = CLUSTER ? (pieces.count + blocks - 1) / blocks : pieces.count;
    const int64_t begin = rank * share, end = begin + share < pieces.count ? begin + share : pieces.count;
    const T outside     = from_float<T>(PROBABILITIES ? 0.0f : -INFINITY);
    if constexpr (CLUSTER) cg::this_cluster().barrier_arrive();  // this block runs: the others may write to it

    Sums q{PROBABILITIES ? 0.0f : Range<T>::START, 0.0f, 0.0f};
    float best = PROBABILITIES ? -1.0f : -INFINITY;
    int held   = static_cast<int>(begin) + threadIdx.x;  // the piece with the maximum
    float2 s2 = make_float2(0.0f, 0.0f), w2 = s2;
    for (int64_t p = begin + threadIdx.x; p < end; p += BLOCK * STREAM_AHEAD) {
        using P2 = Pair<T>;
        typename P2::type v[STREAM_AHEAD][N / 2];
#pragma unroll
        for (int u = 0; u < STREAM_AHEAD; ++u) {
            uint4 raw;
            if (p + u * BLOCK < end) raw = pieces.load(p + u * BLOCK, outside);
            else {
                T e[N];
#pragma unroll
                for (int k = 0; k < N; ++k) e[k] = outside;
                memcpy(&raw, e, 16);
            }
            memcpy(v[u], &raw, 16);
        }
        float most = -INFINITY;
#pragma unroll
        for (int u = 0; u < STREAM_AHEAD; ++u) {
            typename P2::type larger = v[u][0];
#pragma unroll
            for (int k = 1; k < N / 2; ++k) larger = P2::larger(larger, v[u][k]);
            const float2 f  = P2::floats(larger);
            const float top = fmaxf(f.x, f.y);
            if (TOP && top > best) best = top, held = static_cast<int>(p) + u * BLOCK;
            most = fmaxf(most, top);
        }
        if constexpr (PROBABILITIES) {
#pragma unroll
            for (int u = 0; u < STREAM_AHEAD; ++u) {
#pragma unroll
                for (int k = 0; k < N / 2; ++k) {
                    const float2 f = P2::floats(v[u][k]);
                    q.s += f.x + f.y;
                    q.w += times_log(f.x) + times_log(f.y);
                }
            }
        }
        else {
            const float m = fmaxf(q.m, most), M = m * LOG2_E, d = q.m * LOG2_E - M, f = exp2_of(d);
            w2  = mul2(fma2(s2, make_float2(d, d), w2), make_float2(f, f));
            s2  = mul2(s2, make_float2(f, f));
            q.m = m;
            const auto low = P2::both(Range<T>::LOW);
#pragma unroll
            for (int u = 0; u < STREAM_AHEAD; ++u) {
#pragma unroll
                for (int k = 0; k < N / 2; ++k) {
                    const float2 t = fma2(P2::floats(P2::bounded(v[u][k], low)), make_float2(LOG2_E, LOG2_E), make_float2(-M, -M));
                    const float2 e = make_float2(exp2_of(t.x), exp2_of(t.y));
                    s2 = add2(s2, e);
                    w2 = fma2(e, t, w2);
                }
            }
        }
    }
    if constexpr (!PROBABILITIES) q.s = s2.x + s2.y, q.w = w2.x + w2.y;
    if (TOP && threadIdx.x == 0) shared.found = 0;
    if (TOP) shared.keys[threadIdx.x] = begin + threadIdx.x < end ? static_cast<uint64_t>(order_of(best)) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(held)) : 0;
    q = joined_lanes<WARP>(q, joined_stream<PROBABILITIES>);
    if (BLOCK > WARP && lane == 0) shared.warps[warp] = q;
    const auto out_of_range = [&] { return !PROBABILITIES && !(q.m > Range<T>::ABOVE && q.m < Range<T>::BELOW); };
    bool search = false;
    if (TOP || CLUSTER) search = __syncthreads_or(q.s != q.s || q.w != q.w);  // NaN, or an infinity: its maxima were no maxima
    else {
        // The warps behind the first stay only for a row that is summed again: where one of the warps' maxima is beyond BELOW (all lanes count), or
        // none is above ABOVE (one lane each). To have them all join the sums for that took 3 to 6 % more.
        const int ways = __syncthreads_count(!PROBABILITIES && (q.m >= Range<T>::BELOW || (q.m > Range<T>::ABOVE && lane == 0)));
        if (warp != 0 && (PROBABILITIES || (ways > 0 && ways < WARP))) return;
    }
    if (BLOCK > WARP) q = joined_lanes<BLOCK / WARP>(shared.warps[lane % (BLOCK / WARP)], joined_stream<PROBABILITIES>);

    if constexpr (TOP) {
        if (warp == 0) largest_keys(shared.keys, BLOCK, a.top, shared.best);
        __syncthreads();
        const uint64_t least = shared.best[a.top - 1];
        if (!search) {
            const uint32_t least_order  = static_cast<uint32_t>(least >> 32);
            const int64_t least_piece   = 0xFFFFFFFFu - static_cast<uint32_t>(least);
            const auto collect = [&](int64_t p) {
                float v[N];
                values_of<T>(pieces.load(p, outside), v);
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const int64_t j      = pieces.first(p) + k;
                    const uint32_t order = order_of(v[k]);
                    if (j < 0 || j >= a.classes || order < least_order || (order == least_order && p > least_piece)) continue;
                    const int at = atomicAdd(&shared.found, 1);
                    if (at < CANDIDATES) shared.keys[at] = key_of(v[k], static_cast<int32_t>(j));
                }
            };
            if ((end - begin + BLOCK - 1) / BLOCK * (BLOCK / WARP) <= a.top) {  // few pieces a thread: every one of those threads reads its own
                const uint64_t own = static_cast<uint64_t>(order_of(best)) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(held));
                for (int64_t p = begin + threadIdx.x; p < end && own >= least; p += BLOCK) collect(p);
            }
            else {
                for (int i = warp; i < a.top; i += BLOCK / WARP) {
                    const int64_t piece = 0xFFFFFFFFu - static_cast<uint32_t>(shared.best[i]);
                    const int64_t first = begin + (piece - begin) % BLOCK;
                    for (int64_t p = first + lane * BLOCK; p < end; p += WARP * BLOCK) collect(p);
                }
            }
            __syncthreads();
            search = shared.found > CANDIDATES;
            if (!search && warp == 0) largest_keys(shared.keys, shared.found, a.top, shared.best);
        }
        if (search) {
            uint64_t below = 0;
            for (int k = 0; k < a.top; ++k) {
                uint64_t most = 0;
                for (int64_t p = begin + threadIdx.x; p < end; p += BLOCK) {
                    float v[N];
                    values_of<T>(pieces.load(p, outside), v);
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const int64_t j    = pieces.first(p) + i;
                        const uint64_t key = j >= 0 && j < a.classes ? key_of(v[i], static_cast<int32_t>(j)) : 0;
                        if ((k == 0 || key < below) && key > most) most = key;
                    }
                }
                over_lanes<WARP>([&](int d) {
                    const uint64_t o = __shfl_xor_sync(~0u, most, d);
                    most = o > most ? o : most;
                });
                __syncthreads();
                if (lane == 0) shared.searched[warp] = most;
                __syncthreads();
                below = shared.searched[0];
                for (int w = 1; w < BLOCK / WARP; ++w) below = shared.searched[w] > below ? shared.searched[w] : below;
                if (threadIdx.x == 0) shared.best[k] = below;
            }
        }
        __syncthreads();
    }

    if constexpr (CLUSTER) {
        const cg::cluster_group cluster = cg::this_cluster();
        cluster.barrier_wait();
        StreamShared* first = cluster.map_shared_rank(&shared, 0);
        if (threadIdx.x == 0) first->sums[rank] = q;
        if (TOP && threadIdx.x < a.top) first->bests[rank * a.top + threadIdx.x] = shared.best[threadIdx.x];
        cluster.sync();
        if (rank != 0) return;
        q = shared.sums[0];
        for (int b = 1; b < blocks; ++b) q = joined_stream<PROBABILITIES>(q, shared.sums[b]);
        if (TOP && warp == 0) largest_keys(shared.bests, blocks * a.top, a.top, shared.best);
    }
    if (warp != 0 && !out_of_range()) return;
    __syncwarp();
    Row r;
    if constexpr (PROBABILITIES) r = row_of<true>(q);
    else r = out_of_range() ? row_again<T, BLOCK>(pieces, shared.warps) : row_by_two(q);
    if (warp != 0) return;
    if (lane == 0) write_row<T, PROBABILITIES>(a, row, x, r);
    if (TOP && lane < a.top) write_top<PROBABILITIES>(a, row, lane, static_cast<uint32_t>(shared.best[lane] >> 32), index_of_key(shared.best[lane]), r);
}

// ---- gradients -----------------------------------------------------------------------------------------------------------------
// One pass over the elements once the row's sums are known. 16 x 68101 rows of five floats, forward and backward: 26.6 us (two launches, 15 at the
// memory's rate for both passes); 2048 x 50021 bf16: 128, of which this is 79 (its 410 MB at 5.2 TB/s; 63 at the memory's rate).
//
// The probabilities come from log p = v - log_sum, off by what log_sum was rounded by when it was written: half a step of it. Beyond FAR that is
// more than a result should lose (2^-19 of p; with 16 bits 2^-15, a sixteenth of their half step), and a row of the type's lowest value would
// have p = 1 for every class. There the row's maximum m and log sum e^(v - m) are computed again, and v - m stands for v. That is done
// behind what is done for every row, and written over it: a branch in front cost the other rows 5 to 14 % of their time, this costs up to 5
// (4096 x 2000 floats 14.0 us, with every fourth row far 20.7; 4099 x 32771 bf16 101 and 218).
template <typename T>
constexpr float FAR = sizeof(T) == 4 ? 64.0f : 1024.0f;
template <typename T>
__device__ __forceinline__ bool is_far(float log_sum) {
    return fabsf(log_sum) >= FAR<T> && fabsf(log_sum) < INFINITY;
}
template <int G>
__device__ __forceinline__ unsigned lanes_of_row() {
    return G == WARP ? ~0u : ((1u << G % WARP) - 1) << (threadIdx.x % WARP / G * G);
}
// Maximum and log sum of a row, by its G lanes.
template <typename T, int G>
__device__ __forceinline__ float2 near_row(const T* x, int classes, int lane) {
    const unsigned lanes = lanes_of_row<G>();
    float m = -INFINITY, s = 0.0f;
#pragma unroll 1
    for (int j = lane; j < classes; j += G) m = fmaxf(m, to_float(x[j]));
    over_lanes<G>([&](int d) { m = fmaxf(m, __shfl_xor_sync(lanes, m, d)); });
#pragma unroll 1
    for (int j = lane; j < classes; j += G) s += exp_of(to_float(x[j]) - m);
    over_lanes<G>([&](int d) { s += __shfl_xor_sync(lanes, s, d); });
    return make_float2(m, logf(s));
}
// v - m, -infinity for a masked class alone
__device__ __forceinline__ float less(float v, float m) {
    return v == -INFINITY ? v : fmaxf(v - m, -3.402823466e38f);
}
template <bool PROBABILITIES>
struct RowGrad {
    float log_sum, d_label, d_entropy, offset, one_over_sum;
    int label_at;  // -1: nowhere
    __device__ __forceinline__ RowGrad(const ScoresGradArgs& a, int64_t row) : log_sum(a.log_sum[row]), d_label(0.0f), label_at(-1) {
        if (a.d_log_prob != nullptr) {
            const int64_t label = label_of(a.labels, a.labels_64, row);
            const bool inside   = label >= 0 && label < a.classes;
            if (inside) label_at = static_cast<int>(label);
            if (label != -1) d_label = inside ? a.d_log_prob[row] : NAN;
        }
        d_entropy = a.d_entropy != nullptr ? a.d_entropy[row] : 0.0f;
        offset    = (a.d_log_sum != nullptr ? a.d_log_sum[row] : 0.0f) - d_label - (a.d_entropy != nullptr ? d_entropy * a.entropy[row] : 0.0f);
        if (log_sum != log_sum) offset = NAN;
        one_over_sum = PROBABILITIES ? exp_of(-log_sum) : 0.0f;
    }
    // of N neighbouring classes, the first of them number j
    template <int N>
    __device__ __forceinline__ void of(const float (&x)[N], int64_t j, float (&to)[N]) const {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float v  = value_of<PROBABILITIES>(x[k]);
            const float lp = bounded(v - log_sum);  // a masked class: p is 0, and so is its gradient
            const float d  = fmaf(-d_entropy, lp, offset);
            to[k]          = PROBABILITIES ? (v == -INFINITY ? 0.0f : d * one_over_sum) : d * exp_of(lp);
        }
        if (!(fabsf(offset) < INFINITY) || (label_at >= j && label_at < j + N)) {  // the row's label is one of these, or the row has no distribution
#pragma unroll
            for (int k = 0; k < N; ++k) {
                if (j + k == label_at) to[k] += label_gradient(x[k]);
                if (x[k] == (PROBABILITIES ? 0.0f : -INFINITY)) to[k] = 0.0f;
            }
        }
    }
    // what the label's own class gets besides
    __device__ __forceinline__ float label_gradient(float x) const {
        return PROBABILITIES ? d_label / x : x == -INFINITY ? 0.0f : d_label;
    }
};

// Every `step`-th element from `begin` on of a row that is far from 0, of which grad holds the log sum of what is less its maximum m.
template <typename T>
__device__ __forceinline__ void far_elements(const RowGrad<false>& grad, const T* x, float m, int64_t begin, int64_t end, int step, T* dx) {
#pragma unroll 1
    for (int64_t j = begin; j < end; j += step) {
        const float v[1] = {less(to_float(x[j]), m)};
        float d[1];
        grad.of(v, j, d);
        dx[j] = from_float<T>(d[0]);
    }
}

// A row that is far from 0, by its G lanes (staged: where the block's rows are gathered, or NULL). A function that is called and looks everything up
// for itself: what it needs would otherwise be held in registers for all rows.
template <typename T, int G>
__device__ __noinline__ void far_row(const ScoresGradArgs& a, T* staged) {
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * ROW_BLOCK + threadIdx.x) / G;
    const int lane    = threadIdx.x % G;
    const T* x        = static_cast<const T*>(a.x) + row * a.row_stride;
    const float2 r    = near_row<T, G>(x, a.classes, lane);
    RowGrad<false> grad(a, row);
    grad.log_sum = r.y;
    __syncwarp(lanes_of_row<G>());  // what the row's lanes wrote before comes before what they write now
    far_elements<T>(grad, x, r.x, lane, a.classes, G, staged != nullptr ? staged + threadIdx.x * a.classes : static_cast<T*>(a.dx) + row * a.dx_row_stride);
}

// Up to 8 classes: a thread per row. The results go through shared memory, so that a block writes its rows, which lie side by side (dense),
// in one piece.
template <typename T, bool PROBABILITIES, int C>
__global__ void __launch_bounds__(ROW_BLOCK) k_scores_grad_own_row(const __grid_constant__ ScoresGradArgs a, bool wide, bool dense) {
    __shared__ alignas(16) T staged[ROW_BLOCK * C];
    const int first = blockIdx.x * ROW_BLOCK, row = first + threadIdx.x;
    if (row < a.rows) {
        float x[C], d[C];
        load_row<T, C>(static_cast<const T*>(a.x) + row * a.row_stride, wide, x);
        const RowGrad<PROBABILITIES> grad(a, row);
        T* const dx = dense ? staged + threadIdx.x * C : static_cast<T*>(a.dx) + row * a.dx_row_stride;
            grad.of(x, 0, d);
#pragma unroll
        for (int k = 0; k < C; ++k) dx[k] = from_float<T>(d[k]);
        if constexpr (!PROBABILITIES) {
            if (is_far<T>(grad.log_sum)) far_row<T, 1>(a, dense ? staged : nullptr);
        }
    }
    if (dense) {
        __syncthreads();
        const int values    = static_cast<int>(a.rows - first < ROW_BLOCK ? a.rows - first : ROW_BLOCK) * C;
        T* const to         = static_cast<T*>(a.dx) + static_cast<int64_t>(first) * C;
        constexpr int PIECE = 16 / sizeof(T);
        for (int i = threadIdx.x; i < values / PIECE; i += ROW_BLOCK) reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(staged)[i];
        for (int i = values / PIECE * PIECE + threadIdx.x; i < values; i += ROW_BLOCK) to[i] = staged[i];
    }
}

// Up to 1024 classes, G lanes per row as above.
template <typename T, bool PROBABILITIES, int G, int E>
__global__ void __launch_bounds__(ROW_BLOCK) k_scores_grad_rows(const __grid_constant__ ScoresGradArgs a, bool wide) {
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * ROW_BLOCK + threadIdx.x) / G;
    const int lane    = threadIdx.x % G;
    if (row >= a.rows) return;
    T* dx      = static_cast<T*>(a.dx) + row * a.dx_row_stride;
    using Load = RowLoad<T, G, E>;
    float v[E];
    Load::load(static_cast<const T*>(a.x) + row * a.row_stride, a.classes, wide, lane, v);
    const RowGrad<PROBABILITIES> grad(a, row);
    if constexpr (Load::MAY) {
        if (wide) {
#pragma unroll
            for (int i = 0; i < E; i += Load::PIECE) {
                const int j = Load::index(true, lane, i);
                float x[Load::PIECE], d[Load::PIECE];
                T e[Load::PIECE];
#pragma unroll
                for (int k = 0; k < Load::PIECE; ++k) x[k] = v[i + k];
                grad.of(x, j, d);
#pragma unroll
                for (int k = 0; k < Load::PIECE; ++k) e[k] = from_float<T>(d[k]);
                if (j + Load::PIECE <= a.classes) {
                    uint4 raw;
                    memcpy(&raw, e, 16);
                    *reinterpret_cast<uint4*>(dx + j) = raw;
                }
                else {
#pragma unroll
                    for (int k = 0; k < Load::PIECE; ++k)
                        if (j + k < a.classes) dx[j + k] = e[k];
                }
            }
        }
    }
    if (!(Load::MAY && wide)) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int j = i * G + lane;
            if (j < a.classes) {
                const float x[1] = {v[i]};
                float d[1];
                grad.of(x, j, d);
                dx[j] = from_float<T>(d[0]);
            }
        }
    }
    if constexpr (!PROBABILITIES) {
        if (is_far<T>(grad.log_sum)) far_row<T, G>(a, nullptr);
    }
}

// The same for a block of a long row, whose blocks each go over the whole row for themselves. Its barriers come between the two results.
template <typename T>
__device__ __noinline__ void far_block(const ScoresGradArgs& a, int blocks) {
    __shared__ float warps[2][STREAM_BLOCK / WARP];
    const int64_t row = a.rows - 1 - blockIdx.x / blocks;
    const T* x        = static_cast<const T*>(a.x) + row * a.row_stride;
    const Pieces<T> pieces(x, a.classes);
    constexpr int N = Pieces<T>::N;
    const int lane = threadIdx.x % WARP, warp = threadIdx.x / WARP;
    const auto over = [&](auto f) {
        for (int64_t p = threadIdx.x; p < pieces.count; p += STREAM_BLOCK) {
            float v[N];
            values_of<T>(pieces.load(p, from_float<T>(-INFINITY)), v);
            for (int k = 0; k < N; ++k) f(v[k]);
        }
    };
    float m = -INFINITY, s = 0.0f;
    over([&](float v) { m = fmaxf(m, v); });
    over_lanes<WARP>([&](int d) { m = fmaxf(m, __shfl_xor_sync(~0u, m, d)); });
    if (lane == 0) warps[0][warp] = m;
    __syncthreads();
    m = warps[0][lane % (STREAM_BLOCK / WARP)];
    over_lanes<STREAM_BLOCK / WARP>([&](int d) { m = fmaxf(m, __shfl_xor_sync(~0u, m, d)); });
    over([&](float v) { s += exp_of(v - m); });
    over_lanes<WARP>([&](int d) { s += __shfl_xor_sync(~0u, s, d); });
    if (lane == 0) warps[1][warp] = s;
    __syncthreads();
    s = warps[1][lane % (STREAM_BLOCK / WARP)];
    over_lanes<STREAM_BLOCK / WARP>([&](int d) { s += __shfl_xor_sync(~0u, s, d); });
    RowGrad<false> grad(a, row);
    grad.log_sum = logf(s);
    const int64_t first = pieces.first(static_cast<int64_t>(blockIdx.x % blocks) * (STREAM_BLOCK * STREAM_AHEAD)), end = first + STREAM_BLOCK * STREAM_AHEAD * N;
    far_elements<T>(grad, x, m, (first < 0 ? 0 : first) + threadIdx.x, end < a.classes ? end : a.classes, STREAM_BLOCK, static_cast<T*>(a.dx) + row * a.dx_row_stride);
}

// Longer rows: a block for STREAM_BLOCK * STREAM_AHEAD pieces of a row. The last rows come first: they are what the cache still holds of
// the pass that made the sums.
// The bound holds the 16-bit kernels of logits to the 48 registers of five blocks an SM: with 57 they took 79 and 85 us instead of 75 and 73 (2048 x
// 50021 bf16, 20000 x 2055 fp16).
template <typename T, bool PROBABILITIES>
__global__ void __launch_bounds__(STREAM_BLOCK, !PROBABILITIES && sizeof(T) == 2 ? 5 : 0) k_scores_grad_stream(const __grid_constant__ ScoresGradArgs a, int blocks) {
    const int64_t row = a.rows - 1 - blockIdx.x / blocks;
    const T* x        = static_cast<const T*>(a.x) + row * a.row_stride;
    T* dx             = static_cast<T*>(a.dx) + row * a.dx_row_stride;
    const Pieces<T> pieces(x, a.classes);
    constexpr int N      = Pieces<T>::N;
    const bool together  = reinterpret_cast<uintptr_t>(dx) % 16 == reinterpret_cast<uintptr_t>(x) % 16;
    const int64_t begin  = static_cast<int64_t>(blockIdx.x % blocks) * (STREAM_BLOCK * STREAM_AHEAD) + threadIdx.x;
    const T outside      = from_float<T>(0.0f);
    uint4 raw[STREAM_AHEAD];
#pragma unroll
    for (int u = 0; u < STREAM_AHEAD; ++u)
        if (begin + u * STREAM_BLOCK < pieces.count) raw[u] = pieces.load(begin + u * STREAM_BLOCK, outside);
    const RowGrad<PROBABILITIES> grad(a, row);
    // Logits, in powers of two and by pairs as above: with S = log_sum L rounded, t = x L - S and rho = log_sum L - S, log p = (t - rho) log 2
    // and p = 2^(t - rho), so that rho joins the factors of the row. Values are not let below log_sum - 1000, where p is 0; of a row that is not
    // far from 0 that is well below log_sum in every type.
    const float S = grad.log_sum * LOG2_E, rho = fmaf(grad.log_sum, LOG2_E, -S), back = exp2_of(-rho);
    const float slope = -grad.d_entropy * LOG_2 * back, level = fmaf(grad.d_entropy * LOG_2, rho, grad.offset) * back;
    const bool quick  = !PROBABILITIES && fabsf(grad.log_sum) < INFINITY && fabsf(grad.offset) < INFINITY;
    const auto low    = Pair<T>::both(grad.log_sum - 1000.0f);
#pragma unroll
    for (int u = 0; u < STREAM_AHEAD; ++u) {
        const int64_t p = begin + u * STREAM_BLOCK;
        if (p >= pieces.count) break;
        const int64_t j = pieces.first(p);
        T e[N];
        if (quick) {
            typename Pair<T>::type v[N / 2];
            memcpy(v, &raw[u], 16);
#pragma unroll
            for (int k = 0; k < N / 2; ++k) {
                const float2 t = fma2(Pair<T>::floats(Pair<T>::bounded(v[k], low)), make_float2(LOG2_E, LOG2_E), make_float2(-S, -S));
                const float2 d = mul2(fma2(t, make_float2(slope, slope), make_float2(level, level)), make_float2(exp2_of(t.x), exp2_of(t.y)));
                e[2 * k] = from_float<T>(d.x), e[2 * k + 1] = from_float<T>(d.y);
            }
            if (static_cast<unsigned>(grad.label_at - static_cast<int>(j)) < N) {  // the row's label is one of these
                float x[N], d[N];
                values_of<T>(raw[u], x);
                grad.of(x, j, d);
#pragma unroll
                for (int k = 0; k < N; ++k) e[k] = from_float<T>(d[k]);
            }
        }
        else {
            float v[N], d[N];
            values_of<T>(raw[u], v);
            grad.of(v, j, d);
#pragma unroll
            for (int k = 0; k < N; ++k) e[k] = from_float<T>(d[k]);
        }
        if (together && j >= 0 && j + N <= a.classes) {
            uint4 out;
            memcpy(&out, e, 16);
            *reinterpret_cast<uint4*>(dx + j) = out;
        }
        else {
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (j + k >= 0 && j + k < a.classes) dx[j + k] = e[k];
        }
    }
    if constexpr (!PROBABILITIES) {
        if (is_far<T>(grad.log_sum)) far_block<T>(a, blocks);
    }
}

}  // namespace answers
}  // namespace vm
