// vm_gated_scan, vm_gated_scan_backward and vm_gated_step: checks and launches of the kernels in gated.cuh.
#include <algorithm>
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "device_call.hpp"
#include "gated.cuh"

namespace {

using namespace vm;
using namespace vm::answers;

constexpr int64_t MOST = INT64_MAX >> 4;  // no offset in bytes comes near the end of 64 bits

bool sizes_fit(int64_t batch, int64_t steps, int64_t channels) {
    if (batch < 0 || steps < 0 || channels < 0 || batch > INT32_MAX || steps > INT32_MAX || channels > INT32_MAX) return false;
    return batch * channels <= (int64_t(1) << 38);
}

// An output needs a place of its own for every index: strides that nest, in the order that their sizes give.
bool nests(const vm_sequence& s, const int64_t (&sizes)[3]) {
    int64_t stride[3] = {s.batch_stride, s.step_stride, s.channel_stride}, size[3] = {sizes[0], sizes[1], sizes[2]};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (stride[j] < stride[i]) {
                std::swap(stride[i], stride[j]);
                std::swap(size[i], size[j]);
            }
    int64_t reach = 1;
    for (int i = 0; i < 3; ++i) {
        if (size[i] <= 1) continue;
        if (stride[i] < reach) return false;
        reach = stride[i] * (size[i] - 1) + reach;
    }
    return true;
}

// Whether s (NULL: absent, where that is allowed) can be addressed; throws the message otherwise.
void check_sequence(const vm_sequence* s, const char* name, int32_t type, const int64_t (&sizes)[3], bool needed, bool output) {
    if (s == nullptr || s->data == nullptr) {
        if (needed) throw std::string("null ") + name;
        return;
    }
    if (!aligned(s->data, element_size(type))) throw std::string(name) + " is not aligned to its elements";
    const int64_t stride[3] = {s->batch_stride, s->step_stride, s->channel_stride};
    int64_t reach = 0;
    for (int i = 0; i < 3; ++i) {
        if (stride[i] < 0) throw std::string(name) + ": strides must not be negative";
        if (sizes[i] > 1 && stride[i] > MOST / sizes[i]) throw std::string(name) + ": stride out of range";
        reach += sizes[i] > 1 ? stride[i] * (sizes[i] - 1) : 0;
        if (reach > MOST) throw std::string(name) + ": strides out of range";
    }
    if (output && !nests(*s, sizes)) throw std::string(name) + ": elements of an output share a place";
}

Sequence sequence(const vm_sequence* s) {
    if (s == nullptr) return Sequence{nullptr, 0, 0, 0};
    return Sequence{s->data, s->batch_stride, s->step_stride, s->channel_stride};
}

// Whether every block looks for earlier rows of its slots in the index itself: few rows, or rows of so many channels that a block has few of
// them. By blocks / with a table of first rows, us: 256 rows of 3 channels 6.3 / 7.1, 512 10.4 / 6.9; 1024 of 64 6.5 / 7.0, of 512 6.2 / 7.1;
// 2048 of 512 8.4 / 7.0.
constexpr int64_t MOST_LOOKED_THROUGH = 256;
bool looks_through(int64_t rows, int64_t channels) {
    return rows <= MOST_LOOKED_THROUGH || (rows <= 4 * MOST_LOOKED_THROUGH && channels >= 64);
}

unsigned blocks_of(int64_t threads, int block) {
    const int64_t n = (threads + block - 1) / block;
    if (n > INT32_MAX) throw std::string("too many elements for one call");
    return static_cast<unsigned>(n);
}

void check_sizes(int32_t type, int64_t batch, int64_t steps, int64_t channels) {
    if (!known_type(type)) throw std::string("unknown element type");
    if (!sizes_fit(batch, steps, channels)) throw std::string("batch, steps and channels must be 0..2^31-1 (batch * channels at most 2^38)");
}

// ---- how a scan is laid out ----------------------------------------------------------------------------------------------
constexpr int SMS = 148;  // of a B200; which launch is taken depends on it, no result

// A thread takes pairs of channels where they lie side by side, else single ones; a block 32 channels either way. Steps of a thread in the
// forward and in the backward pass: what its 128 registers hold (but for a few outside of the loops), with two blocks an SM. Half the steps in 80
// registers with three blocks an SM were slower: 4 x 4096 x 2048 forward / backward bf16 53 / 97 and 60 / 142 us, float 67 / 118 and 84 / 164.
constexpr int forward_steps(int vector, bool wide_type) {
    return vector == 2 && !wide_type ? 16 : 8;
}
constexpr int backward_steps(int vector, bool wide_type) {
    return vector == 2 && wide_type ? 4 : 8;
}
// Blocks of 16 channels that an SM's registers hold.
constexpr int forward_resident(int vector) {
    return vector == 2 ? 4 : 6;
}
constexpr int BACKWARD_RESIDENT = 4;
// Whether every sequence gets a thread of its own, which walks along time alone: many short ones, of which a tile over time would be mostly
// empty. Tiles / a thread each, us: forward 64 x 204304 bf16 95 / 24, float 76 / 33; 512 x 100000 81 / 84 and 111 / 114;
// 200 x 40000 23 / 27. Backward 64 x 204304 107 / 58 and 97 / 77, 128 x 80000 49 / 58 and 58 / 67. 64 steps of 40000 sequences forward
// 21 / 11, backward 23 / 17; of 10000 10 / 8 and 11 / 13.
bool serial(int64_t all, int64_t steps, bool backward) {
    constexpr int64_t FEW = 16384, MANY = 75776, LONG = 512;
    return (steps <= KEEP && all >= FEW) || (!backward && steps <= LONG && all >= MANY);
}

struct Plan {
    int64_t blocks;  // along the channels
    int64_t run;     // steps of a part
    int64_t parts;
    bool cluster;    // the parts are blocks of a cluster, which take every so manieth tile, instead
};

// `vector` elements and `length` steps a thread, `resident` blocks of a cluster's kind on an SM at a time.
//
// Blocks of 32 channels that fill the SMs take their sequences whole. Fewer share each: with clusters of blocks of 16 channels, which read
// everything once, or, where clusters of 8 would still leave SMs without a block and each block more than 4 tiles, as parts, which are read
// twice. A cluster grows while all of the call's blocks run together: its blocks wait for each other's tiles, and a second round of
// clusters costs as much as the first. Forward / backward on B200, us:
//   3 x 1021 x 515 (97 blocks of 16, float): clusters of 4  13 / 15, of 8  10 / 20 (of which 6 and 4 blocks fit an SM)
//   3 x 4096 x 1024 (192): clusters of 2  41 / 76, of 4  44 / 88, whole  42 / 77
//   1 x 65537 x 64 (4): 8 parts in a cluster 40, 129 parts 16.4
Plan plan_of(int64_t all, int64_t steps, int vector, int length, int resident) {
    const auto blocks_of = [&](int channels) { return (all + channels - 1) / channels; };
    const int64_t tile = 8 * vector * length, tiles = (steps + tile - 1) / tile;  // whatever the block: 32 W threads for 4 W / vector of them along the channels
    Plan p{blocks_of(Shape<8>::CHANNELS), steps, 1, false};
    if (p.blocks >= SMS || tiles <= 1) return p;
    const int64_t narrow = blocks_of(Shape<4>::CHANNELS);
    int64_t ranks        = 2;
    while (ranks < MOST_RANKS && ranks < tiles && narrow * ranks * 2 <= resident * SMS) ranks *= 2;
    if (narrow * ranks >= 2 * SMS || tiles <= 4 * ranks) return Plan{narrow, steps, ranks, true};
    const int64_t wanted = std::min(tiles, (2 * SMS + p.blocks - 1) / p.blocks);
    p.run                = (tiles + wanted - 1) / wanted * tile;
    p.parts              = (steps + p.run - 1) / p.run;
    return p;
}

// Whether `vector` neighbouring channels of s lie side by side at a place that one load or store can take.
bool takes(const vm_sequence* s, int32_t type, int vector, const int64_t (&sizes)[3]) {
    if (s == nullptr || s->data == nullptr) return true;
    const size_t size = element_size(type);
    return s->channel_stride == 1 && aligned(s->data, vector * size) && (sizes[0] <= 1 || s->batch_stride % vector == 0) && (sizes[1] <= 1 || s->step_stride % vector == 0);
}

// How a thread takes elements (vector) and copies them (piece, in bytes; 0: not through the ring).
struct Access {
    int vector, piece;
};
// f(a value of the element type, elements of a thread, bytes of a copy), as constants
template <typename F>
void with_access(int32_t type, const Access& access, F f) {
    using std::integral_constant;
    with_type(type, [&](auto kind) {
        if (access.piece == 16) f(kind, integral_constant<int, 2>{}, integral_constant<int, 16>{});
        else if constexpr (sizeof(kind) == 2) {
            if (access.vector == 2) f(kind, integral_constant<int, 2>{}, integral_constant<int, 4>{});
            else f(kind, integral_constant<int, 1>{}, integral_constant<int, 0>{});
        }
        else f(kind, integral_constant<int, 1>{}, integral_constant<int, 0>{});
    });
}
bool in_pairs(int32_t type, int64_t channels, const int64_t (&sizes)[3], std::initializer_list<const vm_sequence*> sequences) {
    return channels % 2 == 0 && std::all_of(sequences.begin(), sequences.end(), [&](const vm_sequence* s) { return takes(s, type, 2, sizes); });
}
// Inputs are read through the ring in pieces, outputs are written by a thread's vectors. Where no piece of 16 bytes fits, single elements go
// through registers, but pairs of 16 bits through the ring where blocks are few. Forward / backward by pairs and by single elements, us:
// bf16 8 x 40462 x 74 117 / 165 and 155 / 201, 1 x 65536 x 66 32 / 42 and 36 / 38, but 6 x 3216 x 1710 130 / 181 and 87 / 163; float
// 3 x 4096 x 1022 58 / 141 and 50 / 93, 1 x 16384 x 514 56 / 90 and 47 / 58.
Access access_of(int32_t type, int64_t channels, const int64_t (&sizes)[3], std::initializer_list<const vm_sequence*> inputs, std::initializer_list<const vm_sequence*> outputs, const float* states) {
    const int wide = 16 / static_cast<int>(element_size(type));
    if (!in_pairs(type, channels, sizes, inputs) || !in_pairs(type, channels, sizes, outputs) || !aligned(states, 8)) return {1, 0};
    if (channels % wide == 0 && std::all_of(inputs.begin(), inputs.end(), [&](const vm_sequence* s) { return takes(s, type, wide, sizes); })) return {2, 16};
    if (type != VM_F32 && sizes[0] * channels < SMS * Shape<8>::CHANNELS) return {2, 4};
    return {1, 0};
}

// Launches one kernel (early: while the one in front of it runs, whose results it waits for itself), which is told once for a device that it
// may take more shared memory than every kernel may.
template <auto KERNEL>
void launch_tiles(dim3 grid, int threads, int ranks, bool early, int shared, cudaStream_t q, const GatedArgs& a, const Split& s) {
    static LaunchPlans plans;
    if (shared > 0) {
        plans.get([&](int) {
            VM_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, shared));
            return LaunchPlan{};
        });
    }
    cudaLaunchAttribute attributes[2]{};
    int count = 0;
    if (ranks > 1) {
        cudaLaunchAttribute& cluster = attributes[count++];
        cluster.id                   = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim.x = cluster.val.clusterDim.z = 1;
        cluster.val.clusterDim.y = ranks;
    }
    if (early) {
        cudaLaunchAttribute& programmatic                       = attributes[count++];
        programmatic.id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
        programmatic.val.programmaticStreamSerializationAllowed = 1;
    }
    cudaLaunchConfig_t config{};
    config.gridDim          = grid;
    config.blockDim         = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream           = q;
    config.attrs            = attributes;
    config.numAttrs         = count;
    VM_CUDA(cudaLaunchKernelEx(&config, KERNEL, a, s));
}

Split split_of(const Plan& p, void* workspace) {
    return Split{p.run, static_cast<int32_t>(p.parts), static_cast<float2*>(workspace)};
}

void check_workspace(int64_t batch, int64_t steps, int64_t channels, const void* workspace, size_t bytes) {
    const size_t needed = vm_gated_workspace(batch, steps, channels);
    if (bytes < needed) throw std::string("the workspace is too small");
    if (needed > 0 && (workspace == nullptr || !aligned(workspace, 16))) throw std::string("the workspace is null or not aligned to 16 bytes");
}

dim3 grid_of(const Plan& p) {
    if (p.blocks > INT32_MAX) throw std::string("too many sequences for one call");
    return dim3(static_cast<unsigned>(p.blocks), static_cast<unsigned>(p.parts));
}

}  // namespace

extern "C" {

size_t vm_gated_workspace(int64_t batch, int64_t steps, int64_t channels) {
    if (!sizes_fit(batch, steps, channels) || batch == 0 || channels == 0) return 0;
    const int64_t all = batch * channels;
    int64_t parts     = 1;
    for (const int vector : {1, 2})
        for (const int length : {4, 8, 16})
            for (const int resident : {forward_resident(vector), BACKWARD_RESIDENT}) {
                const Plan p = plan_of(all, steps, vector, length, resident);
                if (!p.cluster) parts = std::max(parts, p.parts);
            }
    return parts > 1 ? static_cast<size_t>(parts * all) * sizeof(float2) : 0;
}

vm_status vm_gated_scan(int device, int32_t type, int64_t batch, int64_t steps, int64_t channels, const vm_sequence* x, const vm_sequence* gate, const float* h0,
                        const int32_t* lengths, const vm_sequence* y, float* last, float* states, void* workspace, size_t workspace_bytes, void* stream) {
    try {
        check_sizes(type, batch, steps, channels);
        if (batch == 0 || channels == 0) return VM_OK;
        const int64_t sizes[3] = {batch, steps, channels};
        check_sequence(x, "x", type, sizes, steps > 0, false);
        check_sequence(gate, "gate", type, sizes, steps > 0, false);
        check_sequence(y, "y", type, sizes, false, true);
        if (!words_aligned({h0, lengths, last, states})) throw std::string("h0, lengths, last or states are not aligned to their elements");
        check_workspace(batch, steps, channels, workspace, workspace_bytes);
        const OnDevice on(device);
        GatedArgs a{};
        a.batch = batch, a.steps = steps, a.channels = channels;
        a.small = batch * channels <= UINT32_MAX;
        a.x = sequence(x), a.gate = sequence(gate), a.y = sequence(y);
        a.h0 = h0, a.lengths = lengths, a.last = last, a.states = states;
        const auto q       = static_cast<cudaStream_t>(stream);
        if (serial(batch * channels, steps, false)) {
            const auto launch = [&](auto kind, auto v) {
                constexpr int V = decltype(v)::value;
                launch_kernel(k_gated_serial<decltype(kind), V>, dim3(blocks_of(batch * channels / V, SERIAL_BLOCK)), SERIAL_BLOCK, 0, q, false, a);
            };
            with_type(type, [&](auto kind) {
                if (in_pairs(type, channels, sizes, {x, gate, y}) && aligned(h0, 8) && aligned(last, 8) && aligned(states, 8)) launch(kind, std::integral_constant<int, 2>{});
                else launch(kind, std::integral_constant<int, 1>{});
            });
            return VM_OK;
        }
        const Access access = access_of(type, channels, sizes, {x, gate}, {y}, states);
        const Plan p    = plan_of(batch * channels, steps, access.vector, forward_steps(access.vector, type == VM_F32), forward_resident(access.vector));
        const Split s   = split_of(p, workspace);
        const dim3 grid = grid_of(p);
        with_access(type, access, [&](auto kind, auto v, auto piece) {
            using T = decltype(kind);
            constexpr int V = decltype(v)::value, PIECE = decltype(piece)::value, L = forward_steps(V, sizeof(T) == 4), SHARED = Tiles<T, V, L, 2, PIECE, 8>::SHARED;
            if (p.cluster) {
                launch_tiles<k_gated_scan<T, V, L, PIECE, true>>(grid, Shape<4>::THREADS, static_cast<int>(p.parts), false, Tiles<T, V, L, 2, PIECE, 4>::SHARED, q, a, s);
                return;
            }
            if (p.parts > 1) launch_tiles<k_gated_summary<T, V, L, PIECE, false>>(grid, Shape<8>::THREADS, 1, false, SHARED, q, a, s);
            launch_tiles<k_gated_scan<T, V, L, PIECE, false>>(grid, Shape<8>::THREADS, 1, p.parts > 1, SHARED, q, a, s);
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

vm_status vm_gated_scan_backward(int device, int32_t type, int64_t batch, int64_t steps, int64_t channels, const vm_sequence* x, const vm_sequence* gate, const float* states,
                                 const int32_t* lengths, const vm_sequence* dy, const float* d_last, const vm_sequence* dx, const vm_sequence* d_gate, float* d_h0,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    try {
        check_sizes(type, batch, steps, channels);
        if (batch == 0 || channels == 0) return VM_OK;
        const int64_t sizes[3] = {batch, steps, channels};
        check_sequence(x, "x", type, sizes, steps > 0, false);
        check_sequence(gate, "gate", type, sizes, steps > 0, false);
        check_sequence(dy, "dy", type, sizes, false, false);
        check_sequence(dx, "dx", type, sizes, false, true);
        check_sequence(d_gate, "d_gate", type, sizes, false, true);
        if (steps > 0 && states == nullptr) throw std::string("null states");
        if (!words_aligned({states, lengths, d_last, d_h0})) throw std::string("states, lengths, d_last or d_h0 are not aligned to their elements");
        check_workspace(batch, steps, channels, workspace, workspace_bytes);
        const OnDevice on(device);
        GatedArgs a{};
        a.batch = batch, a.steps = steps, a.channels = channels;
        a.small = batch * channels <= UINT32_MAX;
        a.x = sequence(x), a.gate = sequence(gate), a.y = sequence(dy);
        a.lengths = lengths, a.states = const_cast<float*>(states), a.d_last = d_last;
        a.dx = sequence(dx), a.d_gate = sequence(d_gate), a.d_h0 = d_h0;
        const auto q = static_cast<cudaStream_t>(stream);
        if (serial(batch * channels, steps, true)) {
            const dim3 grid(blocks_of(batch * channels, SERIAL_GRAD_BLOCK));
            with_type(type, [&](auto kind) { launch_kernel(k_gated_serial_grad<decltype(kind)>, grid, SERIAL_GRAD_BLOCK, serial_shared(steps, element_size(type)), q, false, a); });
            return VM_OK;
        }
        const Access access = access_of(type, channels, sizes, {x, gate, dy}, {dx, d_gate}, nullptr);
        const Plan p     = plan_of(batch * channels, steps, access.vector, backward_steps(access.vector, type == VM_F32), BACKWARD_RESIDENT);
        const Split s    = split_of(p, workspace);
        const dim3 grid  = grid_of(p);
        with_access(type, access, [&](auto kind, auto v, auto piece) {
            using T = decltype(kind);
            constexpr int V = decltype(v)::value, PIECE = decltype(piece)::value, L = backward_steps(V, sizeof(T) == 4);
            if (p.cluster) {
                launch_tiles<k_gated_scan_grad<T, V, L, PIECE, true>>(grid, Shape<4>::THREADS, static_cast<int>(p.parts), false, Tiles<T, V, L, 3, PIECE, 4>::SHARED, q, a, s);
                return;
            }
            if (p.parts > 1) launch_tiles<k_gated_summary<T, V, L, PIECE, true>>(grid, Shape<8>::THREADS, 1, false, Tiles<T, V, L, 2, PIECE, 8>::SHARED, q, a, s);
            launch_tiles<k_gated_scan_grad<T, V, L, PIECE, false>>(grid, Shape<8>::THREADS, 1, p.parts > 1, Tiles<T, V, L, 3, PIECE, 8>::SHARED, q, a, s);
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

size_t vm_gated_step_workspace(int64_t rows, int64_t slots) {
    return rows > MOST_LOOKED_THROUGH && slots > 0 ? static_cast<size_t>(slots) * sizeof(uint32_t) : 0;
}

vm_status vm_gated_step(int device, int32_t type, int64_t rows, int64_t slots, int64_t channels, float* state, int64_t state_stride, const vm_sequence* x,
                        const vm_sequence* gate, const int32_t* index, const vm_sequence* y, void* workspace, size_t workspace_bytes, void* stream) {
    try {
        check_sizes(type, rows, 1, channels);
        if (slots < 0 || slots > INT32_MAX) throw std::string("slots must be 0..2^31-1");
        if (index == nullptr && rows > slots) throw std::string("more rows than slots, and no index");
        if (rows == 0 || channels == 0) return VM_OK;
        const int64_t sizes[3] = {rows, 1, channels};
        check_sequence(x, "x", type, sizes, true, false);
        check_sequence(gate, "gate", type, sizes, true, false);
        check_sequence(y, "y", type, sizes, false, true);
        if (slots > 0 && state == nullptr) throw std::string("null state");
        if (!words_aligned({state, index})) throw std::string("state or index are not aligned to their elements");
        if (state_stride < (slots > 1 ? channels : 0) || state_stride > MOST / (slots > 0 ? slots : 1)) throw std::string("the states of slots overlap");
        const size_t needed = index != nullptr ? vm_gated_step_workspace(rows, slots) : 0;
        if (workspace_bytes < needed || (needed > 0 && (workspace == nullptr || !aligned(workspace, 16)))) throw std::string("the workspace is too small, null or not aligned");
        const OnDevice on(device);
        const auto q = static_cast<cudaStream_t>(stream);
        const StepArgs a{rows, slots, channels, state, state_stride, sequence(x), sequence(gate), sequence(y), index, static_cast<uint32_t*>(workspace)};
        const bool table = needed > 0 && !looks_through(rows, channels);
        if (table) {
            launch_kernel(k_first_rows, dim3(blocks_of(rows, STEP_BLOCK)), STEP_BLOCK, 0, q, false, a);
        }
        const bool vectors = channels % 4 == 0 && takes(x, type, 4, sizes) && takes(gate, type, 4, sizes) && takes(y, type, 4, sizes) && aligned(state, 16) && state_stride % 4 == 0;
        with_type(type, [&](auto kind) {
            using T = decltype(kind);
            const auto launch = [&](auto v) {
                constexpr int V     = decltype(v)::value;
                const unsigned grid = blocks_of(rows * (channels / V), STEP_BLOCK);
                if (index == nullptr || slots == 0) launch_kernel(k_gated_step<T, V, ROW_IS_SLOT>, dim3(grid), STEP_BLOCK, 0, q, false, a);
                else if (!table) launch_kernel(k_gated_step<T, V, LOOK_THROUGH>, dim3(grid), STEP_BLOCK, 0, q, false, a);
                else launch_kernel(k_gated_step<T, V, TABLE>, dim3(grid), STEP_BLOCK, 0, q, true, a);
            };
            if (vectors) launch(std::integral_constant<int, 4>{});
            else launch(std::integral_constant<int, 1>{});
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
