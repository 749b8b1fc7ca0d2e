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

#include <cooperative_groups.h>

#include <cstdint>
#include <cstring>
#include <type_traits>

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
    bool small;  // batch * channels < 2^32
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
// e^-|g| as the square of a half of it: e^(-|g| / 2) is a normal number wherever e^-|g| is a number of 32 bits at all, normal or not, and one
// multiplication is less than what an exponential of the full range takes. From |g| = 104 on it is 0.
// 4 x 4096 x 2048 bf16 forward and backward 148.3 -> 148.9 us, 60 calls 0.5 % in the mean.
__device__ __forceinline__ Factors factors_of(float g) {
    const float half = exp2_of(-0.721347520f * fabsf(g)), e = half * half, r = one_over(1.0f + e), s = e * r;  // e <= 1: nothing overflows
    return g >= 0.0f ? Factors{r, s} : Factors{s, r};
}
// a * b, where a of 0 drops b
__device__ __forceinline__ float gated(float a, float b) {
    return a == 0.0f ? 0.0f : a * b;
}

// a * b + c, where a of 0 drops b
__device__ __forceinline__ float gated(float a, float b, float c) {
    return a == 0.0f ? c : fmaf(a, b, c);
}
// The factor of two runs of steps. It is 0 only where a step's is: what 32 bits cannot hold becomes their smallest number, so that an infinity or NaN
// goes on through a long run as it does step by step, and of a state at the end of the range 5e-7 stay.
constexpr float SMALLEST = 1.40129846e-45f;
__device__ __forceinline__ float product(float a, float b) {
    const float r = a * b;
    return a == 0.0f || b == 0.0f ? 0.0f : r < SMALLEST ? SMALLEST : r;
}

// Of all sequences number `at`: its batch (a division in 32 bits is a quarter of one in 64).
__device__ __forceinline__ int64_t batch_of(const GatedArgs& a, int64_t at) {
    return a.small ? static_cast<uint32_t>(at) / static_cast<uint32_t>(a.channels) : at / a.channels;
}

__device__ __forceinline__ int64_t length_of(const GatedArgs& a, int64_t b) {
    if (a.lengths == nullptr) return a.steps;
    const int64_t n = a.lengths[b];
    return n < 0 ? 0 : n > a.steps ? a.steps : n;
}

// ---- tiles -------------------------------------------------------------------------------------------------------------------
// A block of W warps owns CHANNELS = 4 W neighbouring channels and walks over time in tiles: a thread holds V channels of L consecutive
// steps, CHANNELS / V threads lie along the channels, the others along time. A step h -> f h + v is an affine map, and so is every run of
// steps (A, H): h -> A h + H. A tile is three things: the maps of the threads' own steps, a scan of the maps over the threads along time
// (shuffles inside a warp, shared memory between the warps), and the states of the own steps from the one that the scan gives. Every element
// is read once and written once.
//
// Whether a factor of 0 meets an infinity or NaN is not asked step by step: an infinity or NaN leaves H without a finite value (0 times it is
// NaN), and only then the thread goes over its steps again, with the rule.
//
// Two barriers a tile: behind the first the warps' maps lie in shared memory and one thread for every channel folds them, from the state that
// it carries; behind the second the states in front of every warp are there, and the ring's next tile.
//
// W is 8 where a block walks alone (the more threads along time, the fewer tiles), 4 where a cluster shares a sequence: narrower blocks are
// more of them, and a cluster need not be as large (3 x 1021 x 515 floats, forward and backward: 33 us and 29).
// Bound by the instructions: 32 for an element forward and 65 backward (an exponential, a reciprocal, conversions, one map or two, the scan's
// share), which take 66 to 71 % of the active issue slots with 16 warps an SM (128 registers), the rest being barriers and the ring's wait. 4 x 4096 x
// 2048 forward / backward: bf16 51 / 96 us (31 / 51 at the memory's rate), float 66 / 115 (61 / 102). Clusters were slower wherever blocks fill the
// SMs (the same in clusters of 2: 66 / 123), as were pairs of floats in one instruction (moves into even registers cost what they save).
template <int W>
struct Shape {
    static constexpr int THREADS = 32 * W, CHANNELS = 4 * W;
};

template <int BYTES>
struct RawOf;
template <>
struct RawOf<2> {
    using type = uint16_t;
};
template <>
struct RawOf<4> {
    using type = uint32_t;
};
template <>
struct RawOf<8> {
    using type = uint2;
};
template <>
struct RawOf<16> {
    using type = uint4;
};
template <typename T, int V>
using Raw = typename RawOf<V * sizeof(T)>::type;

template <typename T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V>& raw, float (&to)[V]) {
    T e[V];
    memcpy(e, &raw, sizeof(raw));
#pragma unroll
    for (int k = 0; k < V; ++k) to[k] = to_float(e[k]);
}
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> pack(const float (&from)[V]) {
    T e[V];
#pragma unroll
    for (int k = 0; k < V; ++k) e[k] = from_float<T>(from[k]);
    Raw<T, V> raw;
    memcpy(&raw, e, sizeof(raw));
    return raw;
}
// V neighbouring 32-bit floats at a place that is aligned to all of them
template <int V>
__device__ __forceinline__ void load_floats(const float* from, float (&to)[V]) {
    const Raw<float, V> raw = *reinterpret_cast<const Raw<float, V>*>(from);
    memcpy(to, &raw, sizeof(raw));
}
template <int V>
__device__ __forceinline__ void store_floats(float* to, const float (&from)[V]) {
    Raw<float, V> raw;
    memcpy(&raw, from, sizeof(raw));
    *reinterpret_cast<Raw<float, V>*>(to) = raw;
}

template <int V, int W>
struct Place {
    static constexpr int TX = Shape<W>::CHANNELS / V, SEGMENTS = 32 / TX;  // threads along the channels, along time in a warp
    int warp, lane, tx, ty;
    int64_t at, b, c;  // first of the thread's channels: of all, its batch, within that
    bool there;
    __device__ __forceinline__ Place(const GatedArgs& a) {
        warp  = threadIdx.x / 32;
        lane  = threadIdx.x % 32;
        tx    = lane % TX;
        ty    = warp * SEGMENTS + lane / TX;
        at    = (static_cast<int64_t>(blockIdx.x) * TX + tx) * V;
        there = at < a.batch * a.channels;
        b     = there ? batch_of(a, at) : 0;
        c     = there ? at - b * a.channels : 0;
    }
};

// Maps of the warps of a block, and the states in front of them.
template <int V, int W>
struct alignas(16) Between {
    static constexpr int CHANNELS = Shape<W>::CHANNELS;
    float before[W][CHANNELS];
    float2 totals[W][CHANNELS];
};

// Whether a factor is 0, or came to it.
template <int V>
__device__ __forceinline__ bool has_zero(const float (&A)[V]) {
    bool zero = false;
#pragma unroll
    for (int k = 0; k < V; ++k) zero = zero || A[k] == 0.0f;
    return zero;
}
// The factor of L steps, 0 only where one of theirs is.
template <int V, int L>
__device__ __forceinline__ void products(const float (&f)[L][V], float (&A)[V]) {
#pragma unroll
    for (int k = 0; k < V; ++k) A[k] = f[0][k];
#pragma unroll
    for (int i = 1; i < L; ++i) {
#pragma unroll
        for (int k = 0; k < V; ++k) A[k] = product(f[i][k], A[k]);
    }
}
template <int V>
__device__ __forceinline__ bool finite(const float (&v)[V]) {
    bool ok = true;
#pragma unroll
    for (int k = 0; k < V; ++k) ok = ok && fabsf(v[k]) < INFINITY;
    return ok;
}

// Scan over the lanes along time, in their order or (REVERSE) against it. In: every thread's map (A, H). Out: the map of all threads
// before it in its own warp, and that of the whole warp in `shared`. careful: in one of the lanes a factor is 0 or a value not finite.
template <int V, int W, bool REVERSE>
__device__ __forceinline__ void scan_warp(const Place<V, W>& at, float (&A)[V], float (&H)[V], bool careful, Between<V, W>& shared) {
    constexpr int TX = Place<V, W>::TX;
    const auto from = [](float v, int d) { return REVERSE ? __shfl_down_sync(~0u, v, d) : __shfl_up_sync(~0u, v, d); };
    const auto scan = [&](auto care) {
#pragma unroll
        for (int d = TX; d < 32; d *= 2) {
            const bool has = REVERSE ? at.lane + d < 32 : at.lane >= d;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float pa = from(A[k], d), ph = from(H[k], d);
                if (has) {
                    if constexpr (decltype(care)::value) {
                        H[k] = gated(A[k], ph, H[k]);
                        A[k] = product(A[k], pa);
                    }
                    else {
                        H[k] = fmaf(A[k], ph, H[k]);
                        A[k] = fmaxf(A[k] * pa, SMALLEST);
                    }
                }
            }
        }
    };
    if (__any_sync(~0u, careful)) scan(std::true_type{});
    else scan(std::false_type{});
    if (REVERSE ? at.lane < TX : at.lane >= 32 - TX) {
#pragma unroll
        for (int k = 0; k < V; ++k) shared.totals[at.warp][at.tx * V + k] = make_float2(A[k], H[k]);
    }
    const bool first = REVERSE ? at.lane >= 32 - TX : at.lane < TX;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        if constexpr (TX < 32) {
            const float pa = from(A[k], TX), ph = from(H[k], TX);
            A[k] = first ? 1.0f : pa;
            H[k] = first ? 0.0f : ph;
        }
        else A[k] = 1.0f, H[k] = 0.0f;
    }
}
// One thread for a channel, between two barriers: the states in front of every warp, from the one in front of the block (carry), which
// becomes the one behind it.
template <int V, int W, bool REVERSE>
__device__ __forceinline__ void fold_warps(Between<V, W>& shared, int channel, float& carry) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const int w              = REVERSE ? W - 1 - i : i;
        const float2 q           = shared.totals[w][channel];
        shared.before[w][channel] = carry;
        carry                    = gated(q.x, carry, q.y);
    }
}
// The state in front of the thread's own steps.
template <int V, int W>
__device__ __forceinline__ void state_before(const Place<V, W>& at, const Between<V, W>& shared, const float (&A)[V], const float (&H)[V], float (&h)[V]) {
    float before[V];
    load_floats<V>(&shared.before[at.warp][at.tx * V], before);
#pragma unroll
    for (int k = 0; k < V; ++k) h[k] = gated(A[k], before[k], H[k]);
}

template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
    static_assert(BYTES == 4 || BYTES == 16, "pieces of the ring");
    const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to));
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at), "l"(from) : "memory");
}

// A gate that keeps the state: what stands for steps that are not there (with a value of 0).
template <typename T>
__device__ __forceinline__ T kept_gate() {
    return from_float<T>(INFINITY);
}
constexpr int STAGES = 3;  // tiles of the ring
enum { X = 0, GATE = 1, DY = 2 };  // which of the sequences of a kernel
template <typename T, int PIECE>
__device__ __forceinline__ typename RawOf<PIECE>::type filled(bool gate) {
    T e[PIECE / sizeof(T)];
#pragma unroll
    for (int i = 0; i < PIECE / static_cast<int>(sizeof(T)); ++i) e[i] = gate ? kept_gate<T>() : from_float<T>(0.0f);
    typename RawOf<PIECE>::type raw;
    memcpy(&raw, e, PIECE);
    return raw;
}

// How many of a thread's L steps from t on come before `stop`.
template <int L>
__device__ __forceinline__ int steps_before(int64_t stop, int64_t t) {
    return stop - t >= L ? L : stop > t ? static_cast<int>(stop - t) : 0;
}
// The tiles of N sequences on their way through a ring in shared memory (asynchronous copies hold no registers while they are under way), a
// row of the block's channels for a step. A thread copies pieces of PIECE bytes (16 where the sequences' places allow it) for channels of its
// own, and after a barrier every thread reads what it works on. Rows at and behind a sequence's stop are filled instead. A row of 16-bit
// elements is half as wide as the banks, so that the rows of every other thread along time begin in their other half (a gap behind every L
// rows). Copies by the whole block in pieces of 16 bytes instead of every thread's own pairs: 4 x 4096 x 2048 bf16 forward and backward
// 222 -> 150 us.
// PIECE == 0: no ring, every thread reads its own (single) elements into registers, a tile ahead: an asynchronous copy has 4 bytes at least.
template <typename T, int V, int L, int N, int PIECE, int W>
struct Tiles {
    static constexpr int THREADS = Shape<W>::THREADS, CHANNELS = Shape<W>::CHANNELS, TX = CHANNELS / V, TILE = THREADS / TX * L;
    static constexpr int ROW   = CHANNELS * sizeof(T), GAP = ROW < 128 ? ROW : 0;
    static constexpr int BYTES = TILE * ROW + TILE / L * GAP;  // of a tile of one sequence
    static constexpr int SHARED = PIECE > 0 ? STAGES * N * BYTES : 0;
    static constexpr int ACROSS = PIECE > 0 ? ROW / (PIECE > 0 ? PIECE : 1) : 1, ROWS = THREADS / ACROSS;  // pieces of a row; rows copied side by side
    static_assert(PIECE == 0 || THREADS % ACROSS == 0, "a thread's channels are the same in every row");

    unsigned char* ring;
    const T* from[N];
    int64_t stride[N];
    int64_t next, left;  // the step that the next tile begins with, and how many tiles are still to be asked for
    int put, at;
    T held[N][PIECE > 0 ? 1 : L], coming[N][PIECE > 0 ? 1 : L];

    __device__ __forceinline__ static int offset(int row) {
        return row * ROW + row / L * GAP;
    }
    // by: steps from tile to tile
    __device__ __forceinline__ void ask(int64_t by, const int64_t (&stop)[N]) {
        if (left-- > 0) {
            const int first = threadIdx.x / ACROSS;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int rows     = steps_before<TILE>(stop[n], next);  // of the tile that are there
                const T* p         = from[n];
                unsigned char* to  = ring + (put * N + n) * BYTES + threadIdx.x % ACROSS * PIECE;
#pragma unroll
                for (int k = 0; k < TILE / ROWS; ++k) {
                    const int row = first + k * ROWS;
                    if (row < rows) copy_async<PIECE>(to + offset(row), p);
                    else *reinterpret_cast<typename RawOf<PIECE>::type*>(to + offset(row)) = filled<T, PIECE>(n == GATE);
                    p += ROWS * stride[n];
                }
                from[n] += by * stride[n];
            }
        }
        next += by;
        put = put + 1 == STAGES ? 0 : put + 1;
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // next: the thread's own step
    __device__ __forceinline__ void read(int64_t by, const int64_t (&stop)[N], T (&to)[N][PIECE > 0 ? 1 : L]) {
        if (left-- <= 0) return;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int there = steps_before<L>(stop[n], next);
            const T* p      = from[n];
#pragma unroll
            for (int i = 0; i < L; ++i, p += stride[n]) {
                to[n][i] = n == GATE ? kept_gate<T>() : from_float<T>(0.0f);
                if (i < there) to[n][i] = *p;
            }
            from[n] += by * stride[n];
        }
        next += by;
    }
    // The first tiles; `from` are the first elements of the first tile that the thread copies (PIECE == 0: that it works on, in that tile).
    __device__ __forceinline__ void begin(void* shared, int64_t by, int64_t first, int64_t tiles, const int64_t (&stop)[N]) {
        at = 0;
        if constexpr (PIECE == 0) {
            next = first + threadIdx.x / TX * L, left = tiles;
            read(by, stop, held);
        }
        if constexpr (PIECE > 0) {
            ring = static_cast<unsigned char*>(shared), next = first, left = tiles, put = 0;
#pragma unroll
            for (int s = 0; s + 1 < STAGES; ++s) ask(by, stop);
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        }
    }
    // In a tile, between two barriers that all threads come to with what they read of the tile before it: the tile behind it is there after
    // the second of them.
    __device__ __forceinline__ void ahead(int64_t by, const int64_t (&stop)[N]) {
        if constexpr (PIECE > 0) {
            ask(by, stop);
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        }
        else read(by, stop, coming);
    }
    // Behind the last use of a tile.
    __device__ __forceinline__ void advance() {
        if constexpr (PIECE > 0) at = at + 1 == STAGES ? 0 : at + 1;
        else memcpy(held, coming, sizeof(held));
    }
    // step number i of the thread's (ty along time, tx along the channels) in sequence n
    __device__ __forceinline__ void get(int n, int i, int tx, int ty, float (&to)[V]) const {
        T e[V];
        if constexpr (PIECE > 0) {
            const Raw<T, V> raw = *reinterpret_cast<const Raw<T, V>*>(ring + (at * N + n) * BYTES + offset(ty * L) + i * ROW + tx * V * sizeof(T));
            memcpy(e, &raw, sizeof(raw));
        }
        else e[0] = held[n][i];
#pragma unroll
        for (int k = 0; k < V; ++k) to[k] = to_float(e[k]);
    }
};

// The part of time that a block of a split launch has: whole tiles of `run` steps, the last as long as there are steps.
struct Split {
    int64_t run;      // steps of a part, a multiple of a tile's; all of them where nothing is split
    int32_t parts;
    float2* summary;  // [parts][batch * channels]: the map of every part
};

// The tiles of a block, in the order it takes them: a part of the sequence, or (CLUSTER) every so manieth tile of all of it.
template <int TILE, bool CLUSTER, bool REVERSE>
struct Walk {
    int64_t first, by, tiles, end;  // the step that the first tile begins with (maybe behind the end), steps from tile to tile, how many, and the end of the steps
    __device__ __forceinline__ Walk(const GatedArgs& a, const Split& s) {
        const int64_t begin = CLUSTER ? 0 : blockIdx.y * s.run;
        end                 = CLUSTER || begin + s.run > a.steps ? a.steps : begin + s.run;
        const int64_t all   = (end - begin + TILE - 1) / TILE;
        const int ranks     = CLUSTER ? gridDim.y : 1;  // a power of two
        tiles               = (all + ranks - 1) >> (__ffs(ranks) - 1);
        first               = begin + ((REVERSE && tiles > 0 ? tiles - 1 : 0) * ranks + (CLUSTER ? blockIdx.y : 0)) * TILE;
        by                  = (REVERSE ? -TILE : TILE) * ranks;
    }
};

// Sequence number n of a kernel, from step `first` on: where the thread's copies begin, and (returned) behind which step of first..end-1 there
// is nothing. What a thread copies belongs to other channels than what it works on, maybe of another batch.
template <typename T, int V, int L, int N, int PIECE, int W>
__device__ __forceinline__ int64_t set_up(Tiles<T, V, L, N, PIECE, W>& io, int n, const Sequence& q, const GatedArgs& a, const Place<V, W>& at, int64_t first, int64_t end) {
    using IO             = Tiles<T, V, L, N, PIECE, W>;
    const int64_t copied = PIECE > 0 ? blockIdx.x * int64_t(IO::CHANNELS) + threadIdx.x % IO::ACROSS * (PIECE / int(sizeof(T))) : at.at;
    io.stride[n]         = q.t;
    io.from[n]           = nullptr;
    if (copied >= a.batch * a.channels || q.data == nullptr) return 0;
    const int64_t b = batch_of(a, copied), length = length_of(a, b);
    io.from[n] = static_cast<const T*>(q.data) + b * q.b + (copied - b * a.channels) * q.c + (first + (PIECE > 0 ? threadIdx.x / IO::ACROSS : at.ty * L)) * q.t;
    return end < length ? end : length;
}

// The state in front of part `part` of a split sequence (or, REVERSE, behind it), from the one at the sequence's end: a thread along
// time takes its share of the parts on that side one after another, several loads at a time, and the threads are joined as in a tile: 129 parts
// in as many rounds of joined threads as it takes cost 3 us more, 194 parts of 12381 x 2 floats 7.
// channel: the one whose state the thread carries, or -1.
template <int V, int W, bool REVERSE>
__device__ __forceinline__ void join_parts(const GatedArgs& a, const Split& s, const Place<V, W>& at, int part, int channel, float& carry, Between<V, W>& shared) {
    constexpr int TY = W * Place<V, W>::SEGMENTS, TOGETHER = 4;
    const int64_t all = a.batch * a.channels;
    cudaGridDependencySynchronize();  // the summaries are there
    const int begin = REVERSE ? part + 1 : 0, end = REVERSE ? s.parts : part;
    const int each  = (end - begin + TY - 1) / TY;
    float A[V], H[V];
#pragma unroll
    for (int k = 0; k < V; ++k) A[k] = 1.0f, H[k] = 0.0f;
    for (int first = 0; first < each; first += TOGETHER) {
        float2 q[TOGETHER][V];
#pragma unroll
        for (int i = 0; i < TOGETHER; ++i) {
            const int j = begin + at.ty * each + (REVERSE ? each - 1 - first - i : first + i);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                q[i][k] = make_float2(1.0f, 0.0f);
                if (at.there && first + i < each && j < end) q[i][k] = s.summary[j * all + at.at + k];
            }
        }
#pragma unroll
        for (int i = 0; i < TOGETHER; ++i) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                H[k] = gated(q[i][k].x, H[k], q[i][k].y);
                A[k] = product(q[i][k].x, A[k]);
            }
        }
    }
    scan_warp<V, W, REVERSE>(at, A, H, !finite<V>(H) || has_zero<V>(A), shared);
    __syncthreads();
    if (channel >= 0) fold_warps<V, W, REVERSE>(shared, channel, carry);
    __syncthreads();
}

// Blocks of a cluster that share their channels, a tile of time each: maps of all their tiles, told to all of them.
constexpr int MOST_RANKS = 8;
template <int W, bool CLUSTER>
struct Exchange {
    float2 maps[CLUSTER ? 2 : 1][CLUSTER ? MOST_RANKS : 1][CLUSTER ? Shape<W>::CHANNELS : 1];
};
// Between the two barriers of a tile, by all threads of a block: the map of its tile, which the thread of a channel makes of its warps', goes to every
// block of the cluster, and comes back as the state in front of this block's tile (here) and the one behind the whole cluster's (carry).
template <int V, int W, bool REVERSE>
__device__ __forceinline__ void tell_cluster(Exchange<W, true>& shared, const Between<V, W>& between, int window, int ranks, int channel, float& carry, float& here) {
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const int rank                  = blockIdx.y;
    float2(*maps)[Shape<W>::CHANNELS] = shared.maps[window & 1];
    if (window == 0) cluster.barrier_wait();  // all blocks run
    if (channel >= 0) {
        float2 whole = make_float2(1.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float2 q = between.totals[REVERSE ? W - 1 - i : i][channel];
            whole          = make_float2(product(q.x, whole.x), gated(q.x, whole.y, q.y));
        }
        for (int to = 0; to < ranks; ++to) *cluster.map_shared_rank(&maps[rank][channel], to) = whole;
    }
    cluster.sync();
    if (channel >= 0) {
        for (int i = 0; i < ranks; ++i) {
            const int from = REVERSE ? ranks - 1 - i : i;
            if (from == rank) here = carry;
            const float2 q = maps[from][channel];
            carry          = gated(q.x, carry, q.y);
        }
    }
}

// Maps of the parts of a split sequence, of the recurrence or (REVERSE) of its gradient. The pass behind it reads the inputs once more, mostly from
// the cache; it starts while this one ends. 65537 x 64 bf16 (129 parts): 16.4 us for both (two more one after the other), 3.8 at the memory's rate
// and 6 for two empty launches.
template <typename T, int V, int L, int PIECE, bool REVERSE>
__global__ void __launch_bounds__(Shape<8>::THREADS) k_gated_summary(const GatedArgs a, const Split s) {
    constexpr int W = 8;
    using IO        = Tiles<T, V, L, 2, PIECE, W>;
    constexpr int TILE = IO::TILE, CHANNELS = IO::CHANNELS;
    extern __shared__ uint4 ring[];
    __shared__ Between<V, W> shared;
    cudaTriggerProgrammaticLaunchCompletion();  // the kernel behind this one reads its first tiles meanwhile
    const Place<V, W> at(a);
    const Walk<TILE, false, REVERSE> walk(a, s);
    const int64_t end = walk.end, tiles = walk.tiles, first = walk.first, by = walk.by;
    IO io;
    const int64_t stops[2] = {set_up(io, X, REVERSE ? a.y : a.x, a, at, first, end), set_up(io, GATE, a.gate, a, at, first, end)};
    io.begin(ring, by, first, tiles, stops);
    const int channel = threadIdx.x < CHANNELS ? threadIdx.x : -1;
    float carry = 0.0f, whole = 1.0f;
    __syncthreads();
    for (int64_t tile = 0; tile < tiles; ++tile) {
        float A[V], H[V];
        const auto pass = [&](auto careful) {
            constexpr bool CAREFUL = decltype(careful)::value;
#pragma unroll
            for (int k = 0; k < V; ++k) A[k] = 1.0f, H[k] = 0.0f;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                float x[V], g[V];
                io.get(X, i, at.tx, at.ty, x);
                io.get(GATE, i, at.tx, at.ty, g);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const Factors w = factors_of(g[k]);
                    if constexpr (!REVERSE) H[k] = CAREFUL ? gated(w.f, H[k], gated(w.u, x[k])) : fmaf(w.f, H[k], w.u * x[k]);
                    A[k] = CAREFUL ? product(w.f, A[k]) : w.f * A[k];
                    if constexpr (REVERSE) H[k] = CAREFUL ? gated(A[k], x[k], H[k]) : fmaf(A[k], x[k], H[k]);
                }
            }
        };
        pass(std::false_type{});
        const bool careful = !finite<V>(H) || has_zero<V>(A);
        if (careful) pass(std::true_type{});
        scan_warp<V, W, REVERSE>(at, A, H, careful, shared);
        __syncthreads();
        io.ahead(by, stops);
        if (channel >= 0) {
#pragma unroll
            for (int w = 0; w < W; ++w) whole = product(shared.totals[w][channel].x, whole);
            fold_warps<V, W, REVERSE>(shared, channel, carry);
        }
        __syncthreads();
        io.advance();
    }
    const int64_t of_channel = static_cast<int64_t>(blockIdx.x) * CHANNELS + channel, all = a.batch * a.channels;
    if (channel >= 0 && of_channel < all) s.summary[blockIdx.y * all + of_channel] = make_float2(whole, carry);
}

// y, the last state and the kept ones. Bounds of registers: 16 warps an SM for pairs (16 steps of 16-bit ones a thread), 24 for single elements.
template <typename T, int V, int L, int PIECE, bool CLUSTER>
__global__ void __launch_bounds__(CLUSTER ? 128 : 256, (V == 1 ? 3 : 2) * (CLUSTER ? 2 : 1)) k_gated_scan(const GatedArgs a, const Split s) {
    constexpr int W = CLUSTER ? 4 : 8;
    using IO        = Tiles<T, V, L, 2, PIECE, W>;
    constexpr int TILE = IO::TILE, CHANNELS = IO::CHANNELS;
    extern __shared__ uint4 ring[];
    __shared__ Between<V, W> shared;
    __shared__ Exchange<W, CLUSTER> exchange;
    if constexpr (CLUSTER) cooperative_groups::this_cluster().barrier_arrive();
    const Place<V, W> at(a);
    const int64_t n     = at.there ? length_of(a, at.b) : 0, kept = (a.steps + KEEP - 1) / KEEP;
    const Walk<TILE, CLUSTER, false> walk(a, s);
    const int64_t begin = walk.first, end = walk.end, tiles = walk.tiles, stop = end < n ? end : n;
    const int64_t by    = walk.by;  // steps from tile to tile
    IO io;
    const int64_t stops[2] = {set_up(io, X, a.x, a, at, begin, end), set_up(io, GATE, a.gate, a, at, begin, end)};
    io.begin(ring, by, begin, tiles, stops);
    int64_t t         = begin + at.ty * L;
    T* y              = static_cast<T*>(a.y.data) + at.b * a.y.b + at.c * a.y.c + t * a.y.t;
    const bool writes = at.there && a.y.data != nullptr;
    const int64_t of_channel = static_cast<int64_t>(blockIdx.x) * CHANNELS + threadIdx.x;
    const int channel        = threadIdx.x < CHANNELS ? threadIdx.x : -1;
    const bool carries       = channel >= 0 && of_channel < a.batch * a.channels;
    float carry              = carries && a.h0 != nullptr ? a.h0[of_channel] : 0.0f;
    if (!CLUSTER && s.parts > 1) join_parts<V, W, false>(a, s, at, blockIdx.y, channel, carry, shared);
    __syncthreads();
    for (int64_t tile = 0; tile < tiles; ++tile, t += by, y += by * a.y.t) {
        const int left = steps_before<L>(stop, t), room = steps_before<L>(end, t);
        float f[L][V], v[L][V], A[V], H[V], h[V];
        const auto pass = [&](auto careful) {
            constexpr bool CAREFUL = decltype(careful)::value;
#pragma unroll
            for (int k = 0; k < V; ++k) A[k] = 1.0f, H[k] = 0.0f;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                io.get(X, i, at.tx, at.ty, v[i]);
                io.get(GATE, i, at.tx, at.ty, f[i]);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const Factors q = factors_of(f[i][k]);
                    f[i][k] = q.f;
                    v[i][k] = CAREFUL ? gated(q.u, v[i][k]) : q.u * v[i][k];
                    H[k]    = CAREFUL ? gated(q.f, H[k], v[i][k]) : fmaf(q.f, H[k], v[i][k]);
                    A[k]    = CAREFUL ? product(q.f, A[k]) : q.f * A[k];
                }
            }
        };
        pass(std::false_type{});
        const bool careful = !finite<V>(H), zero = has_zero<V>(A);
        if (careful) pass(std::true_type{});
        else if (zero) products<V, L>(f, A);
        scan_warp<V, W, false>(at, A, H, careful || zero, shared);
        __syncthreads();
        if constexpr (CLUSTER) {
            float here = 0.0f;
            tell_cluster<V, W, false>(exchange, shared, static_cast<int>(tile), gridDim.y, channel, carry, here);
            if (channel >= 0) fold_warps<V, W, false>(shared, channel, here);
        }
        else if (channel >= 0) fold_warps<V, W, false>(shared, channel, carry);
        io.ahead(by, stops);
        __syncthreads();
        io.advance();
        state_before<V, W>(at, shared, A, H, h);
        if (a.states != nullptr && at.there && room > 0 && t % KEEP == 0) store_floats<V>(a.states + (at.b * kept + t / KEEP) * a.channels + at.c, h);
        if (careful || !finite<V>(h)) {
#pragma unroll
            for (int i = 0; i < L; ++i) {
#pragma unroll
                for (int k = 0; k < V; ++k) v[i][k] = h[k] = gated(f[i][k], h[k], v[i][k]);
            }
        }
        else {
#pragma unroll
            for (int i = 0; i < L; ++i) {
#pragma unroll
                for (int k = 0; k < V; ++k) v[i][k] = h[k] = fmaf(f[i][k], h[k], v[i][k]);
            }
        }
        T* to = y;
        if (writes && left == L) {
#pragma unroll
            for (int i = 0; i < L; ++i, to += a.y.t) *reinterpret_cast<Raw<T, V>*>(to) = pack<T, V>(v[i]);
        }
        else if (writes) {
#pragma unroll
            for (int i = 0; i < L; ++i, to += a.y.t)
                if (i < room) *reinterpret_cast<Raw<T, V>*>(to) = i < left ? pack<T, V>(v[i]) : Raw<T, V>{};
        }
    }
    if (a.last != nullptr && carries && blockIdx.y + 1 == gridDim.y) a.last[of_channel] = carry;
}

// Many short sequences: a thread walks along time alone, AHEAD steps' loads in front of itself. Bound by the loads' latency: 64 x 204303 floats 33
// us, 24 at the memory's rate; 64 x 204304 bf16 in pairs 23 (by single elements 28), 12 at the memory's rate.
constexpr int SERIAL_BLOCK = 128, AHEAD = 8;

template <int BLOCK, int V>
struct Serial {
    int64_t at, b, c, n, kept;
    __device__ __forceinline__ explicit Serial(const GatedArgs& a) : at((static_cast<int64_t>(blockIdx.x) * BLOCK + threadIdx.x) * V), b(0), c(0), n(0), kept((a.steps + KEEP - 1) / KEEP) {
        if (at < a.batch * a.channels) b = batch_of(a, at), c = at - b * a.channels, n = length_of(a, b);
    }
    template <typename T>
    __device__ __forceinline__ T* of(const Sequence& s, int64_t t = 0) const {
        return static_cast<T*>(s.data) + b * s.b + c * s.c + t * s.t;
    }
};

template <typename T, int V>
__global__ void __launch_bounds__(SERIAL_BLOCK) k_gated_serial(const GatedArgs a) {
    const Serial<SERIAL_BLOCK, V> q(a);
    if (q.at >= a.batch * a.channels) return;
    const T* x = q.template of<const T>(a.x);
    const T* g = q.template of<const T>(a.gate);
    T* y       = q.template of<T>(a.y);
    Raw<T, V> rx[AHEAD], rg[AHEAD];
    const auto load = [&](int64_t t) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (t + i < q.n) rx[i] = *reinterpret_cast<const Raw<T, V>*>(x), rg[i] = *reinterpret_cast<const Raw<T, V>*>(g);
            x += a.x.t, g += a.gate.t;
        }
    };
    float h[V] = {};
    if (a.h0 != nullptr) load_floats<V>(a.h0 + q.at, h);
    load(0);
    for (int64_t t = 0; t < a.steps; t += AHEAD) {
        float f[AHEAD][V], v[AHEAD][V];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            float xs[V], gs[V];
            unpack<T, V>(rx[i], xs);
            unpack<T, V>(rg[i], gs);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const bool on   = t + i < q.n;
                const Factors w = factors_of(on ? gs[k] : 0.0f);
                f[i][k] = on ? w.f : 1.0f;
                v[i][k] = on ? gated(w.u, xs[k]) : 0.0f;
            }
        }
        load(t + AHEAD);
        if (a.states != nullptr && t % KEEP == 0) store_floats<V>(a.states + (q.b * q.kept + t / KEEP) * a.channels + q.c, h);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
#pragma unroll
            for (int k = 0; k < V; ++k) h[k] = gated(f[i][k], h[k], v[i][k]);
            if (a.y.data != nullptr && t + i < a.steps) *reinterpret_cast<Raw<T, V>*>(y) = t + i < q.n ? pack<T, V>(h) : Raw<T, V>{};
            y += a.y.t;
        }
    }
    if (a.last != nullptr) store_floats<V>(a.last + q.at, h);
}

// The gradient of few steps: forward through them from the kept state, with half of h_(t-1) - x_t and the gates left in shared memory (every thread
// has its own column: no two of a warp share a bank, nothing waits), then backward. Bound by latency: shared memory holds 7 blocks of 64
// threads an SM. 64 x 204304: bf16 57 us (20 at the memory's rate), floats 75 (40); 16 x 204304 17 and 15. Pairs were no faster (58 and 101).
constexpr int SERIAL_GRAD_BLOCK = 64;
inline size_t serial_shared(int64_t steps, size_t element) {
    return static_cast<size_t>(steps) * SERIAL_GRAD_BLOCK * (sizeof(float) + element);
}

template <typename T>
__global__ void __launch_bounds__(SERIAL_GRAD_BLOCK) k_gated_serial_grad(const GatedArgs a) {
    extern __shared__ uint4 columns[];
    const int steps    = static_cast<int>(a.steps);  // KEEP at most
    float* const apart = reinterpret_cast<float*>(columns) + threadIdx.x;
    T* const gates     = reinterpret_cast<T*>(reinterpret_cast<float*>(columns) + steps * SERIAL_GRAD_BLOCK) + threadIdx.x;
    const Serial<SERIAL_GRAD_BLOCK, 1> q(a);
    if (q.at >= a.batch * a.channels) return;
    const int n = static_cast<int>(q.n);
    {
        const T* x = q.template of<const T>(a.x);
        const T* g = q.template of<const T>(a.gate);
        T rx[AHEAD], rg[AHEAD], nx[AHEAD], ng[AHEAD];
        const auto load = [&](int t) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i, x += a.x.t, g += a.gate.t)
                if (t + i < n) nx[i] = *x, ng[i] = *g;
        };
        float h = n > 0 ? a.states[q.at] : 0.0f;
        load(0);
        for (int t = 0; t < n; t += AHEAD) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) rx[i] = nx[i], rg[i] = ng[i];
            load(t + AHEAD);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                if (t + i >= n) break;
                const Factors w = factors_of(to_float(rg[i]));
                const float xt  = to_float(rx[i]);
                apart[(t + i) * SERIAL_GRAD_BLOCK] = fmaf(0.5f, h, -0.5f * xt);
                gates[(t + i) * SERIAL_GRAD_BLOCK] = rg[i];
                h = gated(w.f, h, gated(w.u, xt));
            }
        }
    }
    T* dx = q.template of<T>(a.dx, steps - 1);
    T* dg = q.template of<T>(a.d_gate, steps - 1);
    for (int t = steps - 1; t >= n; --t, dx -= a.dx.t, dg -= a.d_gate.t) {
        if (a.dx.data != nullptr) *dx = from_float<T>(0.0f);
        if (a.d_gate.data != nullptr) *dg = from_float<T>(0.0f);
    }
    const T* dy = q.template of<const T>(a.y, n - 1);
    T rd[AHEAD], nd[AHEAD];
    const auto load = [&](int t) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i, dy -= a.y.t) {
            nd[i] = from_float<T>(0.0f);
            if (a.y.data != nullptr && t - i >= 0) nd[i] = *dy;
        }
    };
    float c = a.d_last != nullptr ? a.d_last[q.at] : 0.0f;
    load(n - 1);
    for (int t = n - 1; t >= 0; t -= AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) rd[i] = nd[i];
        load(t - AHEAD);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i, dx -= a.dx.t, dg -= a.d_gate.t) {
            if (t - i < 0) break;
            const Factors w   = factors_of(to_float(gates[(t - i) * SERIAL_GRAD_BLOCK]));
            const float total = to_float(rd[i]) + c;
            if (a.dx.data != nullptr) *dx = from_float<T>(gated(w.u, total));
            if (a.d_gate.data != nullptr) *dg = from_float<T>(gated(w.f * w.u, apart[(t - i) * SERIAL_GRAD_BLOCK]) * (total + total));
            c = gated(w.f, total);
        }
    }
    if (a.d_h0 != nullptr) a.d_h0[q.at] = c;
}

// The gradient's walk goes from the last tile to the first. Its own scan runs against time beside the recurrence's, which starts in every
// tile from a kept state. x and dy are read from the ring twice: 8 steps of all that a thread has to hold would spill at 128 registers (260 us
// instead of 222 for 4 x 4096 x 2048 forward and backward, before the copies by the whole block).
template <typename T, int V, int L, int PIECE, bool CLUSTER>
__global__ void __launch_bounds__(CLUSTER ? 128 : 256, CLUSTER ? 4 : 2) k_gated_scan_grad(const GatedArgs a, const Split s) {
    constexpr int W = CLUSTER ? 4 : 8;
    using IO        = Tiles<T, V, L, 3, PIECE, W>;
    constexpr int TILE = IO::TILE, CHANNELS = IO::CHANNELS, THREADS = IO::THREADS;
    extern __shared__ uint4 ring[];
    __shared__ Between<V, W> shared, shared_back;
    __shared__ Exchange<W, CLUSTER> exchange;
    if constexpr (CLUSTER) cooperative_groups::this_cluster().barrier_arrive();
    const Place<V, W> at(a);
    const int64_t kept = (a.steps + KEEP - 1) / KEEP;
    const Walk<TILE, CLUSTER, true> walk(a, s);
    const int64_t end = walk.end, tiles = walk.tiles, by = walk.by;
    int64_t t0 = walk.first, t = t0 + at.ty * L;
    IO io;
    const int64_t stops[3] = {set_up(io, X, a.x, a, at, t0, end), set_up(io, GATE, a.gate, a, at, t0, end), set_up(io, DY, a.y, a, at, t0, end)};
    io.begin(ring, by, t0, tiles, stops);
    T* dx = static_cast<T*>(a.dx.data) + at.b * a.dx.b + at.c * a.dx.c + t * a.dx.t;
    T* dg = static_cast<T*>(a.d_gate.data) + at.b * a.d_gate.b + at.c * a.d_gate.c + t * a.d_gate.t;
    const bool writes_x = at.there && a.dx.data != nullptr, writes_g = at.there && a.d_gate.data != nullptr;
    // the first threads carry the recurrence's states, the last ones the gradient's
    static_assert(2 * CHANNELS <= THREADS, "a thread carries one state");
    const int channel = threadIdx.x < CHANNELS ? threadIdx.x : -1, channel_back = static_cast<int>(threadIdx.x) - (THREADS - CHANNELS);
    const int64_t of_channel = static_cast<int64_t>(blockIdx.x) * CHANNELS + (channel >= 0 ? channel : channel_back), all = a.batch * a.channels;
    const bool carries = channel >= 0 && of_channel < all, carries_back = channel_back >= 0 && of_channel < all;
    const float* states = a.states;
    if (carries) states += of_channel + batch_of(a, of_channel) * (kept - 1) * a.channels;
    float next = carries && tiles > 0 && t0 < a.steps ? states[t0 / KEEP * a.channels] : 0.0f;  // the state in front of the tile to come
    float back = carries_back && a.d_last != nullptr ? a.d_last[of_channel] : 0.0f;
    if (!CLUSTER && s.parts > 1) join_parts<V, W, true>(a, s, at, blockIdx.y, channel_back, back, shared_back);
    __syncthreads();
    for (int64_t tile = 0; tile < tiles; ++tile, t0 += by, t += by, dx += by * a.dx.t, dg += by * a.d_gate.t) {
        float carry = next;
        if (carries && tile + 1 < tiles) next = states[(t0 + by) / KEEP * a.channels];
        const int room = steps_before<L>(end, t);
        float f[L][V], u[L][V], w[L][V], A[V], H[V], AR[V], R[V], h[V], c[V];
        // x and dy are read from the ring twice, here and behind the scan, instead of being held
        const auto pass = [&](auto careful) {
            constexpr bool CAREFUL = decltype(careful)::value;
#pragma unroll
            for (int k = 0; k < V; ++k) A[k] = 1.0f, H[k] = 0.0f, R[k] = 0.0f;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                float x[V], d[V], g[V];
                io.get(X, i, at.tx, at.ty, x);
                io.get(GATE, i, at.tx, at.ty, g);
                io.get(DY, i, at.tx, at.ty, d);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const Factors q = factors_of(g[k]);
                    f[i][k] = q.f;
                    u[i][k] = q.u;
                    H[k]    = CAREFUL ? gated(q.f, H[k], gated(q.u, x[k])) : fmaf(q.f, H[k], q.u * x[k]);
                    A[k]    = CAREFUL ? product(q.f, A[k]) : q.f * A[k];
                    R[k]    = CAREFUL ? gated(A[k], d[k], R[k]) : fmaf(A[k], d[k], R[k]);
                }
            }
        };
        pass(std::false_type{});
        bool careful    = !finite<V>(H) || !finite<V>(R);
        const bool zero = has_zero<V>(A);
        if (careful) pass(std::true_type{});
        else if (zero) products<V, L>(f, A);
#pragma unroll
        for (int k = 0; k < V; ++k) AR[k] = A[k];
        scan_warp<V, W, false>(at, A, H, careful || zero, shared);
        scan_warp<V, W, true>(at, AR, R, careful || zero, shared_back);
        __syncthreads();
        if (channel >= 0) fold_warps<V, W, false>(shared, channel, carry);
        if constexpr (CLUSTER) {
            float here = 0.0f;
            tell_cluster<V, W, true>(exchange, shared_back, static_cast<int>(tile), gridDim.y, channel_back, back, here);
            if (channel_back >= 0) fold_warps<V, W, true>(shared_back, channel_back, here);
        }
        else if (channel_back >= 0) fold_warps<V, W, true>(shared_back, channel_back, back);
        io.ahead(by, stops);
        __syncthreads();
        state_before<V, W>(at, shared, A, H, h);
        state_before<V, W>(at, shared_back, AR, R, c);
        careful = careful || !finite<V>(h) || !finite<V>(c);
        // w: f u (h_(t-1) - x), then the gradient of the gate; u: to the gradient of x
        const auto grads = [&](auto care) {
            constexpr bool CAREFUL = decltype(care)::value;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                float x[V];
                io.get(X, i, at.tx, at.ty, x);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float fu = f[i][k] * u[i][k];  // a quarter at most: h and x beside it stay in the range, and a factor of 0 drops them
                    if constexpr (CAREFUL) w[i][k] = gated(fu, h[k]) - gated(fu, x[k]);
                    else w[i][k] = fmaf(fu, h[k], -(fu * x[k]));
                    h[k] = CAREFUL ? gated(f[i][k], h[k], gated(u[i][k], x[k])) : fmaf(f[i][k], h[k], u[i][k] * x[k]);
                }
            }
#pragma unroll
            for (int i = L - 1; i >= 0; --i) {
                float d[V];
                io.get(DY, i, at.tx, at.ty, d);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float total = d[k] + c[k];
                    w[i][k] = CAREFUL && f[i][k] * u[i][k] == 0.0f ? 0.0f : w[i][k] * total;
                    c[k]    = CAREFUL ? gated(f[i][k], total) : f[i][k] * total;
                    u[i][k] = CAREFUL ? gated(u[i][k], total) : u[i][k] * total;
                }
            }
        };
        if (careful) grads(std::true_type{});
        else grads(std::false_type{});
        io.advance();
        T* to_x = dx;
        T* to_g = dg;
        if (writes_x && writes_g && room == L) {
#pragma unroll
            for (int i = 0; i < L; ++i, to_x += a.dx.t, to_g += a.d_gate.t) {
                *reinterpret_cast<Raw<T, V>*>(to_x) = pack<T, V>(u[i]);
                *reinterpret_cast<Raw<T, V>*>(to_g) = pack<T, V>(w[i]);
            }
        }
        else {
#pragma unroll
            for (int i = 0; i < L; ++i, to_x += a.dx.t, to_g += a.d_gate.t) {
                if (writes_x && i < room) *reinterpret_cast<Raw<T, V>*>(to_x) = pack<T, V>(u[i]);
                if (writes_g && i < room) *reinterpret_cast<Raw<T, V>*>(to_g) = pack<T, V>(w[i]);
            }
        }
    }
    if (a.d_h0 != nullptr && carries_back && blockIdx.y == 0) a.d_h0[of_channel] = back;
}

// ---- single steps ------------------------------------------------------------------------------------------------------------
// A thread has V channels of a row. Of the rows that name a slot the first is the one that counts: a slot is one row's, whatever order they
// run in. With few rows every block looks through the index for itself; with many, a table with the first row of every slot is made before.
// Bound by launches: 64 rows of 2048 bf16 channels 4.7 us and 68100 of 3 floats, with the table, 7.3, where an empty call takes 4; 0.3 and 0.7
// at the memory's rate.
constexpr int STEP_BLOCK = 256;

// The table is not cleared before: what stands in it counts where it is a row that names the slot, which is true whoever wrote it and when.
__global__ void __launch_bounds__(STEP_BLOCK) k_first_rows(const StepArgs a) {
    cudaTriggerProgrammaticLaunchCompletion();
    const uint32_t row = blockIdx.x * STEP_BLOCK + threadIdx.x;
    if (row >= a.rows) return;
    const int32_t slot = a.index[row];
    if (slot < 0 || slot >= a.slots) return;
    uint32_t held = *static_cast<volatile uint32_t*>(a.first + slot);
    while (!(held <= row && a.index[held] == slot)) {  // each round that fails found another row's entry, and those only fall
        const uint32_t was = atomicCAS(a.first + slot, held, row);
        if (was == held) break;
        held = was;
    }
}

enum Slots { ROW_IS_SLOT, LOOK_THROUGH, TABLE };

template <typename T, int V, Slots SLOTS>
__global__ void __launch_bounds__(STEP_BLOCK) k_gated_step(const StepArgs a) {
    const int64_t each = a.channels / V, all = a.rows * each;  // V divides the channels
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * STEP_BLOCK, at = begin + threadIdx.x;
    const auto row_at   = [&](int64_t i) -> int64_t { return all <= UINT32_MAX ? static_cast<uint32_t>(i) / static_cast<uint32_t>(each) : i / each; };
    const bool there    = at < all;
    const int64_t row   = row_at(there ? at : all - 1), c = there ? (at - row * each) * V : 0;
    int64_t slot        = SLOTS == ROW_IS_SLOT ? row : a.index[row];
    if (slot < 0 || slot >= a.slots || !there) slot = -1;
    // everything is on its way before it is known whether the row counts
    Raw<T, V> rx{}, rg{};
    float h[V];
#pragma unroll
    for (int k = 0; k < V; ++k) h[k] = 0.0f;
    float* const state = a.state + (slot >= 0 ? slot * a.state_stride + c : 0);
    if (slot >= 0) {
        rx = *reinterpret_cast<const Raw<T, V>*>(static_cast<const T*>(a.x.data) + row * a.x.b + c * a.x.c);
        rg = *reinterpret_cast<const Raw<T, V>*>(static_cast<const T*>(a.gate.data) + row * a.gate.b + c * a.gate.c);
        load_floats<V>(state, h);
    }
    if constexpr (SLOTS == LOOK_THROUGH) {
        __shared__ int32_t slots[STEP_BLOCK], taken[STEP_BLOCK];  // of the block's rows
        const int low   = static_cast<int>(row_at(begin));
        const int count = static_cast<int>(row_at(begin + STEP_BLOCK < all ? begin + STEP_BLOCK - 1 : all - 1)) - low + 1;
        if (threadIdx.x < count) {
            slots[threadIdx.x] = a.index[low + threadIdx.x];
            taken[threadIdx.x] = 0;
        }
        __syncthreads();
        for (int j = threadIdx.x; j < low + count - 1; j += STEP_BLOCK) {
            const int32_t earlier = a.index[j];
            for (int r = j < low ? 0 : j - low + 1; r < count; ++r)
                if (slots[r] == earlier) taken[r] = 1;
        }
        __syncthreads();
        if (taken[row - low] != 0) slot = -1;
    }
    if constexpr (SLOTS == TABLE) {
        cudaGridDependencySynchronize();
        if (slot >= 0 && a.first[slot] != row) slot = -1;
    }
    if (!there) return;
    if (slot >= 0) {
        float x[V], g[V];
        unpack<T, V>(rx, x);
        unpack<T, V>(rg, g);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const Factors q = factors_of(g[k]);
            h[k]            = gated(q.f, h[k], gated(q.u, x[k]));
        }
        store_floats<V>(state, h);
    }
    else {
#pragma unroll
        for (int k = 0; k < V; ++k) h[k] = 0.0f;
    }
    if (a.y.data != nullptr) *reinterpret_cast<Raw<T, V>*>(static_cast<T*>(a.y.data) + row * a.y.b + c * a.y.c) = pack<T, V>(h);
}

}  // namespace answers
}  // namespace vm
