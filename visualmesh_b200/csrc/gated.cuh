// A gated linear recurrence over sequences, h_t = f_t h_(t-1) + u_t x_t with f = 1 / (1 + exp -g) and u = 1 - f = 1 / (1 + exp g), its
// gradient and its single step. u is computed from g, not from f: near f = 1 the difference would lose its digits.
//
// Gradient: with c_T = d_last and, from the last step to the first,  l_t = dy_t + c_(t+1),  c_t = f_t l_t:
//   dx_t = u_t l_t,   dg_t = f_t u_t (h_(t-1) - x_t) l_t,   d_h0 = c_0
// The states h_(t-1) are computed again from those that the forward pass kept every KEEP steps: exact to 32 bits, and fewer bytes than
// reading the (rounded) outputs would be.
//
// A factor of exactly 0 drops what it multiplies, NaN and infinities included.
#pragma once

#include <cstdint>

#include "../../include/vmcuda.h"
#include "element.cuh"

namespace vm {
namespace answers {

constexpr int KEEP = VM_GATED_KEEP;

// A vm_sequence (data, strides of batch, step and channel in elements); data NULL: absent.
struct Sequence {
    void* data;
    int64_t b, t, c;
};

struct GatedArgs {
    int64_t batch, steps, channels;
    Sequence x, gate, y;  // backward: y is dy
    const float* h0;
    const int32_t* lengths;
    float* last;
    float* states;
    const float* d_last;
    Sequence dx, d_gate;
    float* d_h0;
};

struct StepArgs {
    int64_t rows, slots, channels;
    float* state;
    int64_t state_stride;
    Sequence x, gate, y;
    const int32_t* index;
    uint32_t* first;  // per slot the first row that names it (with index)
};

struct Factors {
    float f, u;
};
__device__ __forceinline__ Factors factors_of(float g) {
    const float e = __expf(-fabsf(g)), r = 1.0f / (1.0f + e), s = e * r;  // e <= 1: nothing overflows
    return g >= 0.0f ? Factors{r, s} : Factors{s, r};
}
// a * b, where a of 0 drops b
__device__ __forceinline__ float gated(float a, float b) {
    return a == 0.0f ? 0.0f : a * b;
}

__device__ __forceinline__ int64_t length_of(const GatedArgs& a, int64_t b) {
    if (a.lengths == nullptr) return a.steps;
    const int64_t n = a.lengths[b];
    return n < 0 ? 0 : n > a.steps ? a.steps : n;
}

// A thread per sequence of one channel.
template <typename T>
__global__ void __launch_bounds__(256) k_gated_scan(const GatedArgs a) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (at >= a.batch * a.channels) return;
    const int64_t b = at / a.channels, c = at % a.channels;
    const T* x = static_cast<const T*>(a.x.data) + b * a.x.b + c * a.x.c;
    const T* g = static_cast<const T*>(a.gate.data) + b * a.gate.b + c * a.gate.c;
    T* y       = a.y.data != nullptr ? static_cast<T*>(a.y.data) + b * a.y.b + c * a.y.c : nullptr;
    float h    = a.h0 != nullptr ? a.h0[at] : 0.0f;
    const int64_t n = length_of(a, b), kept = (a.steps + KEEP - 1) / KEEP;
    for (int64_t t = 0; t < a.steps; ++t) {
        if (a.states != nullptr && t % KEEP == 0) a.states[(b * kept + t / KEEP) * a.channels + c] = h;
        if (t < n) {
            const Factors k = factors_of(to_float(g[t * a.gate.t]));
            h = gated(k.f, h) + gated(k.u, to_float(x[t * a.x.t]));
        }
        if (y != nullptr) y[t * a.y.t] = from_float<T>(t < n ? h : 0.0f);
    }
    if (a.last != nullptr) a.last[at] = h;
}

template <typename T>
__global__ void __launch_bounds__(256) k_gated_scan_grad(const GatedArgs a) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (at >= a.batch * a.channels) return;
    const int64_t b = at / a.channels, c = at % a.channels;
    const T* x  = static_cast<const T*>(a.x.data) + b * a.x.b + c * a.x.c;
    const T* g  = static_cast<const T*>(a.gate.data) + b * a.gate.b + c * a.gate.c;
    const T* dy = a.y.data != nullptr ? static_cast<const T*>(a.y.data) + b * a.y.b + c * a.y.c : nullptr;
    T* dx       = a.dx.data != nullptr ? static_cast<T*>(a.dx.data) + b * a.dx.b + c * a.dx.c : nullptr;
    T* dg       = a.d_gate.data != nullptr ? static_cast<T*>(a.d_gate.data) + b * a.d_gate.b + c * a.d_gate.c : nullptr;
    float carry = a.d_last != nullptr ? a.d_last[at] : 0.0f;
    const int64_t n = length_of(a, b), kept = (a.steps + KEEP - 1) / KEEP;
    float before[KEEP];
    for (int64_t k = kept - 1; k >= 0; --k) {
        const int64_t first = k * KEEP;
        const int count     = static_cast<int>(a.steps - first < KEEP ? a.steps - first : KEEP);
        float h             = a.states[(b * kept + k) * a.channels + c];
        for (int i = 0; i < count; ++i) {
            before[i] = h;
            if (first + i < n) {
                const Factors q = factors_of(to_float(g[(first + i) * a.gate.t]));
                h = gated(q.f, h) + gated(q.u, to_float(x[(first + i) * a.x.t]));
            }
        }
        for (int i = count - 1; i >= 0; --i) {
            const int64_t t = first + i;
            float to_x = 0.0f, to_g = 0.0f;
            if (t < n) {
                const Factors q   = factors_of(to_float(g[t * a.gate.t]));
                const float total = (dy != nullptr ? to_float(dy[t * a.y.t]) : 0.0f) + carry;
                to_x  = gated(q.u, total);
                to_g  = gated(q.f * q.u, (before[i] - to_float(x[t * a.x.t])) * total);
                carry = gated(q.f, total);
            }
            if (dx != nullptr) dx[t * a.dx.t] = from_float<T>(to_x);
            if (dg != nullptr) dg[t * a.d_gate.t] = from_float<T>(to_g);
        }
    }
    if (a.d_h0 != nullptr) a.d_h0[at] = carry;
}

__global__ void __launch_bounds__(256) k_first_rows(const StepArgs a) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (row >= a.rows) return;
    const int32_t slot = a.index[row];
    if (slot >= 0 && slot < a.slots) atomicMin(a.first + slot, static_cast<uint32_t>(row));
}

template <typename T>
__global__ void __launch_bounds__(256) k_gated_step(const StepArgs a) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (at >= a.rows * a.channels) return;
    const int64_t row = at / a.channels, c = at % a.channels;
    int64_t slot = row;
    if (a.index != nullptr) {
        slot = a.index[row];
        if (slot < 0 || slot >= a.slots || a.first[slot] != row) slot = -1;
    }
    float h = 0.0f;
    if (slot >= 0) {
        const Factors k = factors_of(to_float(static_cast<const T*>(a.gate.data)[row * a.gate.b + c * a.gate.c]));
        float* state    = a.state + slot * a.state_stride + c;
        h = gated(k.f, *state) + gated(k.u, to_float(static_cast<const T*>(a.x.data)[row * a.x.b + c * a.x.c]));
        *state = h;
    }
    if (a.y.data != nullptr) static_cast<T*>(a.y.data)[row * a.y.b + c * a.y.c] = from_float<T>(h);
}

}  // namespace answers
}  // namespace vm
