/*
 * vmcuda.h - C ABI of the B200 (sm_100a) Visual Mesh inference engine.
 *
 * The library behind this header replaces, for one path only, what the reference's interchangeable engines do:
 *   visualmesh::engine::cpu::Engine<float>::operator()(mesh, Hoc, lens)                  cpp/visualmesh/engine/cpu/engine.hpp:85-147
 *   visualmesh::engine::cpu::Engine<float>::operator()(mesh, Hoc, lens, image, format)   cpp/visualmesh/engine/cpu/engine.hpp:181-273
 * (the OpenCL engine has the same two calls: cpp/visualmesh/engine/opencl/engine.hpp:283-333, :348-534).
 *
 * Plain pointers and sizes only. All matrices are row-major. Every function returns a vm_status; a failing call
 * leaves a message readable through vm_last_error(). There is no CPU fallback: without a CUDA device every compute
 * entry point fails with VM_ERR_CUDA.
 */
#ifndef VMCUDA_H
#define VMCUDA_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define VM_API __attribute__((visibility("default")))
#else
#define VM_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

typedef enum vm_status {
    VM_OK                     = 0,
    VM_ERR_INVALID_ARGUMENT   = 1,
    /* unknown fourcc; the reference throws std::runtime_error (cpp/visualmesh/engine/cpu/pixel.hpp:100) */
    VM_ERR_UNSUPPORTED_FORMAT = 2,
    /* unknown lens projection; the reference throws std::runtime_error (cpp/visualmesh/utility/projection.hpp:174) */
    VM_ERR_UNSUPPORTED_LENS   = 3,
    /* layer shapes that do not chain: weights rows != (N+1) * previous width, biases != weights columns */
    VM_ERR_NETWORK_SHAPE      = 4,
    VM_ERR_CUDA               = 5,
    VM_ERR_OUT_OF_MEMORY      = 6,
    /* a kernel gave up on a bounded loop and raised its abort flag */
    VM_ERR_DEVICE_ABORT       = 7,
    /* device-side lookup asked for (ranges == NULL) on a mesh that has no BSP uploaded */
    VM_ERR_NO_BSP             = 8
} vm_status;

/* cpp/visualmesh/lens.hpp:28 - same order as enum LensProjection */
enum { VM_RECTILINEAR = 0, VM_EQUISOLID = 1, VM_EQUIDISTANT = 2 };
/* cpp/visualmesh/network_structure.hpp:32-37 - same order as enum ActivationFunction */
enum { VM_SELU = 0, VM_RELU = 1, VM_SOFTMAX = 2, VM_TANH = 3 };

/* Mirrors visualmesh::Lens<float> (cpp/visualmesh/lens.hpp:35-52). k is applied to radii in pixels. */
typedef struct vm_lens {
    int32_t dimensions[2]; /* width, height */
    int32_t projection;    /* VM_RECTILINEAR | VM_EQUISOLID | VM_EQUIDISTANT */
    float focal_length;    /* pixels */
    float centre[2];       /* pixels */
    float k[2];
    float fov;             /* radians */
} vm_lens;

/* One dense layer: visualmesh::Layer<float> (cpp/visualmesh/network_structure.hpp:40-45).
 * weights is row-major [n_in][n_out] exactly as the reference hands them over (:25-27). */
typedef struct vm_layer {
    const float* weights;
    const float* biases;
    int32_t n_in;
    int32_t n_out;
    int32_t activation; /* VM_SELU | VM_RELU | VM_SOFTMAX | VM_TANH */
} vm_layer;

typedef struct vm_engine vm_engine;
typedef struct vm_mesh vm_mesh;

/* One camera frame: the arguments of Engine::operator() (cpp/visualmesh/engine/cpu/engine.hpp:181-185). */
typedef struct vm_frame {
    const vm_mesh* mesh;
    /* n_ranges [start,end) pairs as returned by Mesh::lookup (cpp/visualmesh/mesh.hpp:499-595), or NULL to have
     * the device walk the mesh's BSP itself (needs vm_mesh_set_bsp) */
    const int32_t* ranges;
    int32_t n_ranges;
    float Hoc[16];
    vm_lens lens;
    const void* image; /* NULL: projection only */
    uint32_t format;   /* fourcc code of image */
    int32_t image_on_device;
} vm_frame;

/* Results of a batch, frames concatenated. Frame f has n_f = offsets[f+1] - offsets[f] on-screen points.
 * pixel_coordinates and global_indices hold n_f entries per frame starting at offsets[f].
 * neighbourhood and classifications hold n_f + 1 rows per frame (the last is the off-screen row, as in
 * cpp/visualmesh/engine/cpu/engine.hpp:134-143, :206, :269-272) starting at row offsets[f] + f.
 * Neighbour indices are local to their frame (0..n_f, n_f = off-screen row).
 * Host pointers address pinned memory owned by the engine, valid until its next call. */
typedef struct vm_batch_result {
    int32_t n_frames;
    int32_t n_neighbours;
    int32_t n_classes; /* 0 for projection only */
    int32_t on_device; /* 1: the four data pointers are device pointers */
    const int32_t* offsets; /* host, n_frames + 1 */
    const float* pixel_coordinates;
    const int32_t* global_indices;
    const int32_t* neighbourhood;
    const float* classifications;
} vm_batch_result;

/* flags of vm_run_batch */
enum {
    VM_RESULTS_ON_DEVICE = 1, /* leave results in device memory: no device-to-host copies except offsets */
    VM_TIME_STAGES       = 2  /* bracket every kernel with events; read them with vm_stage_times */
};

/* Replaces the engine constructor Engine(const NetworkStructure<float>&) (cpp/visualmesh/engine/cpu/engine.hpp:57-72,
 * OpenCL: cpp/visualmesh/engine/opencl/engine.hpp:189). layers holds the dense layers of all groups in order;
 * layers_per_group[g] of them belong to ConvolutionalGroup g (cpp/visualmesh/network_structure.hpp:47-52): the first
 * layer of a group consumes the (N+1)-row gather, the others follow without one. n_groups == 0 gives a
 * projection-only engine. device < 0 selects the current device. */
VM_API vm_status vm_engine_create(int device,
                           const vm_layer* layers,
                           const int32_t* layers_per_group,
                           int32_t n_groups,
                           vm_engine** out);
VM_API void vm_engine_destroy(vm_engine* engine);

/* Uploads one mesh (one camera height) once, as the OpenCL engine caches rays per mesh
 * (cpp/visualmesh/engine/opencl/engine.hpp:603-625). rays is n_nodes x 3, neighbours n_nodes x n_neighbours
 * (visualmesh::Node, cpp/visualmesh/node.hpp:40-46); neighbour value n_nodes = no such node. n_neighbours in {4,6,8}. */
VM_API vm_status vm_mesh_upload(vm_engine* engine,
                         const float* rays,
                         const int32_t* neighbours,
                         int32_t n_nodes,
                         int32_t n_neighbours,
                         vm_mesh** out);
/* Adds the mesh's binary space partition (cpp/visualmesh/mesh.hpp:66-83): per element its node range [start,end),
 * its two children (-1,-1 for a leaf) and its bounding cone (axis xyz, cos, sin). With it frames may pass
 * ranges == NULL and Mesh::lookup (cpp/visualmesh/mesh.hpp:499-595) runs on the device. */
VM_API vm_status vm_mesh_set_bsp(vm_engine* engine,
                          vm_mesh* mesh,
                          int32_t n_elements,
                          const int32_t* element_ranges,
                          const int32_t* element_children,
                          const float* element_cones);
/* Counterpart of clear_cache() (cpp/visualmesh/engine/opencl/engine.hpp:559-572) for one mesh. */
VM_API void vm_mesh_release(vm_engine* engine, vm_mesh* mesh);

/* The hot path over a batch of independent frames in one set of kernel launches.
 * All frames of a batch must use meshes with the same n_neighbours. */
VM_API vm_status vm_run_batch(vm_engine* engine, const vm_frame* frames, int32_t n_frames, uint32_t flags, vm_batch_result* out);

/* Single-frame forms of the two reference calls (batches of one).
 * vm_project  = operator()(mesh, Hoc, lens)                cpp/visualmesh/engine/cpu/engine.hpp:85-147
 * vm_classify = operator()(mesh, Hoc, lens, image, format) cpp/visualmesh/engine/cpu/engine.hpp:181-273 */
VM_API vm_status vm_project(vm_engine* engine,
                     const vm_mesh* mesh,
                     const int32_t* ranges,
                     int32_t n_ranges,
                     const float Hoc[16],
                     const vm_lens* lens,
                     vm_batch_result* out);
VM_API vm_status vm_classify(vm_engine* engine,
                      const vm_mesh* mesh,
                      const int32_t* ranges,
                      int32_t n_ranges,
                      const float Hoc[16],
                      const vm_lens* lens,
                      const void* image,
                      uint32_t format,
                      vm_batch_result* out);

/* The reference's calls with their lookup (cpp/visualmesh/engine/opencl/engine.hpp:581): Mesh::lookup runs inside the call, on the
 * device where the mesh's BSP is (vm_mesh_set_bsp), else on the host before it; either finds the same nodes.
 * lookup: the host tables that `mesh` was uploaded from (vm_hostmesh, below); image NULL: projection only. Otherwise vm_classify and
 * vm_project. */
struct vm_hostmesh;
VM_API vm_status vm_call(vm_engine* engine,
                         const vm_mesh* mesh,
                         const struct vm_hostmesh* lookup,
                         const float Hoc[16],
                         const vm_lens* lens,
                         const void* image,
                         uint32_t format,
                         vm_batch_result* out);

/* No counterpart in the reference: the reference's results are the caller's own, the arrays of a vm_batch_result belong to the
 * engine and are overwritten by its next call. vm_results_keep hands the host arrays of the engine's last call over to the caller
 * instead of having them copied: they stay valid until vm_results_release, whatever becomes of the engine, and then serve it again.
 * At most VM_MAX_KEPT_RESULTS are kept per engine; one more fails with VM_ERR_OUT_OF_MEMORY and leaves the results where they
 * are. A set of result arrays is pinned memory for all candidates of the largest batch it served, 12 + 4 * (neighbours + classes)
 * bytes each (its points are not counted when it is made); sets that were given back serve later calls and are freed with the
 * engine, so that an engine holds up to VM_MAX_KEPT_RESULTS + 1 of them. vm_results_release may be called from any thread. */
#define VM_MAX_KEPT_RESULTS 4
typedef struct vm_results vm_results;
VM_API vm_status vm_results_keep(vm_engine* engine, vm_results** kept);
VM_API void vm_results_release(vm_results* kept);

/* No counterpart in the reference.
 * Projection of one frame (operator()(mesh, Hoc, lens) with the lookup on the device) for callers that must not
 * allocate device memory while they run: a camera thread inside a fixed-period control loop, where the driver lock and
 * the implicit device synchronisation of cudaMalloc/cudaFree show up as missed frame deadlines, or a process in which
 * another framework's caching allocator already owns all of the GPU's memory so that a fresh allocation fails.
 * Every intermediate of the call (frame constants, BSP element states, per-candidate pixels and node ids, per-block
 * counts, the node -> point table, the point count) lives in one array that is part of the library image itself,
 * about 4.3 MB, resident on every GPU that loads the library until the process exits. The call makes no
 * cudaMalloc/cudaFree and uses no allocating library routine; inputs (a mesh uploaded earlier with its BSP) and
 * outputs (device buffers of the caller) are passed in.
 * Limits: mesh->n_nodes <= VM_STATIC_MAX_NODES and its BSP <= VM_STATIC_MAX_BSP elements; larger meshes are
 * rejected with VM_ERR_INVALID_ARGUMENT and a message naming the limit.
 * Outputs, all DEVICE pointers sized for the whole mesh: pixel_coordinates n_nodes x 2, global_indices n_nodes,
 * neighbourhood (n_nodes + 1) x n_neighbours; the first n (+1 for neighbourhood) entries are written. n is stored to
 * *d_n_points (device, may be NULL) and to *n_points (host, may be NULL). The call returns after its work has finished.
 * The last-bit correction tables of acosf/sinf/tanf (built, with an allocation, by the first vm_run_batch/vm_project/
 * vm_classify on a device) are used when they already exist and never built here; without them a pixel coordinate can
 * differ from the reference's in its last bit.
 * The first call on a device looks up the array's device address (cudaGetSymbolAddress) - make that first call
 * during set-up, before any stream capture. All calls share the one array and it keeps the previous call's contents
 * (the cells that must start at zero are cleared by each call): two calls whose GPU work overlaps - from two engines,
 * threads or processes' streams on the same device within one process - race on it, so serialise them. */
#define VM_STATIC_MAX_NODES 262144
#define VM_STATIC_MAX_BSP 131072
VM_API vm_status vm_project_static(vm_engine* engine,
                                   const vm_mesh* mesh,
                                   const float Hoc[16],
                                   const vm_lens* lens,
                                   float* d_pixel_coordinates,
                                   int32_t* d_global_indices,
                                   int32_t* d_neighbourhood,
                                   int32_t* d_n_points,
                                   int32_t* n_points);

/* Results that were left on the device are the engine's memory, and its own streams do not wait for others. After this call the
 * engine's calls write there only once everything that `stream` (a cudaStream_t of the engine's device, NULL: the default stream) holds
 * now is done; the host does not wait here, and streams add up. While `stream` is being captured the call does nothing: make it again behind
 * every launch of the graph. */
VM_API vm_status vm_wait_for(vm_engine* engine, void* stream);

/* Stand-alone stages on caller-provided HOST arrays, for testing a stage against the reference function it
 * replaces with identical inputs.
 * vm_sample: cpu::interpolate (cpp/visualmesh/engine/cpu/pixel.hpp:116-144) at n pixel coordinates -> n x 4 floats.
 * vm_network: the gather/dense/activation loop (cpp/visualmesh/engine/cpu/engine.hpp:213-265) over n_rows rows
 *             (last row = off-screen row) of 4 input floats with an n_rows x n_neighbours neighbourhood. */
VM_API vm_status vm_sample(vm_engine* engine,
                    const float* pixel_coordinates,
                    int32_t n,
                    const void* image,
                    int32_t width,
                    int32_t height,
                    uint32_t format,
                    float* out);
VM_API vm_status vm_network(vm_engine* engine,
                     const float* input,
                     const int32_t* neighbourhood,
                     int32_t n_rows,
                     int32_t n_neighbours,
                     float* out);

/* Kernel time of the last vm_run_batch called with VM_TIME_STAGES, one entry per launched kernel in launch order.
 * Returns the number of stages through *n; names[i] points at a static string. */
VM_API vm_status vm_stage_times(vm_engine* engine, const char** names, float* milliseconds, int32_t capacity, int32_t* n);

/* Device-side stopwatch over any number of calls: vm_timer_start records a CUDA event on the engine's first stream
 * (after draining its streams), vm_timer_stop records one that follows all of the engine's streams, waits for it and
 * returns the elapsed device time. */
VM_API vm_status vm_timer_start(vm_engine* engine);
VM_API vm_status vm_timer_stop(vm_engine* engine, float* milliseconds);

/* No counterpart in the reference. Every wait of one thread block on another agent inside the tensor-core kernels (an
 * mbarrier armed by the tensor core or by another warp) polls at most `polls` times, then the kernel raises its abort
 * flag, leaves through its normal tear-down and the call returns VM_ERR_DEVICE_ABORT with the engine still usable.
 * The default (4,000,000 polls, a few seconds) is never reached by a healthy run. 0 makes every such wait give up at
 * once: the way to exercise the error path without hanging or faulting the device. */
VM_API vm_status vm_set_wait_limit(vm_engine* engine, uint32_t polls);

/* Number of kernels launched by this engine since creation. */
VM_API int64_t vm_launch_count(const vm_engine* engine);

/* Pinned host memory for callers that want zero-staging copies of their frames. */
VM_API vm_status vm_host_alloc(void** ptr, size_t bytes);
VM_API void vm_host_free(void* ptr);

/* ------------------------------------------------------------------------------------------------------------------
 * Operators on what a network answered (no counterpart in the reference's engines): how sure it was of every row, and what a
 * sequence of frames adds. All pointers are DEVICE pointers of the caller, on `device` (< 0: the current device; the device that was
 * current is current again when the call returns). The calls enqueue their kernels on `stream` (a cudaStream_t, NULL: the default
 * stream) and return: they neither wait, allocate nor keep anything, so they may be captured into a CUDA graph, from any number of
 * threads. Pointers are aligned to their elements; outputs overlap neither inputs nor one another. What an engine left on the device
 * (VM_RESULTS_ON_DEVICE) is complete when its call returns; before the engine's next call writes there again, `stream` has to be done
 * with it: see vm_wait_for.
 * ------------------------------------------------------------------------------------------------------------------ */

/* element types; sums, logarithms and states are 32-bit floats whatever the type */
enum { VM_F32 = 0, VM_F16 = 1, VM_BF16 = 2 };

enum {
    VM_PROBABILITIES = 1, /* rows hold probabilities (what a softmax layer wrote) instead of logits: v_j = log x_j, else v_j = x_j */
    VM_LABELS_64     = 2  /* labels are int64_t, else int32_t */
};
#define VM_MAX_TOP 32

/* For every row of `classes` values, row_stride elements after the row before it: log_sum = log sum_j exp v_j, with
 * log p_j = v_j - log_sum the log probability of the row's label, entropy = -sum_j p_j log p_j (natural logarithms) and the `top`
 * largest values in descending order with their indices, the lowest index first among equals (top_log_prob and top_index: rows x top).
 * Any output may be NULL; top <= min(classes, VM_MAX_TOP), and top > 0 needs both of its outputs, log_prob needs labels.
 * Label -1: none, log_prob is 0. Any other label outside 0..classes-1: log_prob is NaN.
 * v_j = -infinity (a probability of 0) masks a class: it adds nothing to sum and entropy and its log probability is -infinity. A row
 * with nothing else has log_sum -infinity and entropy 0. A row with NaN or +infinity (or a negative probability, or a sum of
 * probabilities beyond 2^96) has no distribution: its log_sum, entropy and log probabilities are NaN; in the order of the top values
 * NaN comes before +infinity. */
VM_API vm_status vm_scores(int device,
                           const void* x,
                           int32_t type,
                           int64_t rows,
                           int32_t classes,
                           int64_t row_stride,
                           uint32_t flags,
                           const void* labels,
                           int32_t top,
                           float* log_prob,
                           float* entropy,
                           float* log_sum,
                           float* top_log_prob,
                           int32_t* top_index,
                           void* stream);

/* The gradient of x (rows dx_row_stride apart, type as x) from those of log_prob, entropy and log_sum (each NULL: zero), with x, labels,
 * flags, entropy and log_sum as vm_scores had and wrote them (labels and d_log_prob come together; entropy is needed with d_entropy):
 *   logits         dx_j = p_j (d_log_sum - d_log_prob - d_entropy (log p_j + entropy)) + d_log_prob [j = label]
 *   probabilities  dx_j = (the same bracket) / sum_j x_j + d_log_prob [j = label] / x_j
 * A masked class gets the gradient 0, also where it is the label; label -1 counts as d_log_prob 0; the gradient of a row with another
 * label outside 0..classes-1, or without a distribution, is NaN but for its masked classes. */
VM_API vm_status vm_scores_backward(int device,
                                    const void* x,
                                    int32_t type,
                                    int64_t rows,
                                    int32_t classes,
                                    int64_t row_stride,
                                    uint32_t flags,
                                    const void* labels,
                                    const float* entropy,
                                    const float* log_sum,
                                    const float* d_log_prob,
                                    const float* d_entropy,
                                    const float* d_log_sum,
                                    void* dx,
                                    int64_t dx_row_stride,
                                    void* stream);

/* Element (b, t, c) of a sequence is data[b * batch_stride + t * step_stride + c * channel_stride] (in elements, >= 0; 0 repeats an
 * input along that dimension, outputs have an element of their own for every index). */
typedef struct vm_sequence {
    void* data;
    int64_t batch_stride;
    int64_t step_stride;
    int64_t channel_stride;
} vm_sequence;

/* Steps between two states that vm_gated_scan keeps for its backward pass. */
#define VM_GATED_KEEP 64

/* A gated linear recurrence over `steps` of batch x channels sequences: with f = 1 / (1 + exp(-gate)),
 *   h_t = f_t h_(t-1) + (1 - f_t) x_t,   y_t = h_t,   h_(-1) = h0 (NULL: zero),   last = h after the last step.
 * gate = -infinity drops what was before (the sequence begins anew), +infinity drops x_t (nothing was seen), whatever they hold, NaN
 * and infinities included; so do gates beyond -104 and 104, whose factor is 0 in 32 bits. lengths (NULL: all `steps`): sequence b has
 * lengths[b] steps (clamped to 0..steps); y is 0 behind them and last is h after the last of them. x, gate and y have `type`; h0, last and
 * states are 32-bit, batch x channels without gaps.
 * states (may be NULL): batch x ceil(steps / VM_GATED_KEEP) x channels, h before steps 0, 64, 128, ...: what the backward pass starts from.
 * y and last may be NULL. workspace: at least vm_gated_workspace(batch, steps, channels) bytes, aligned to 16, that no other call uses
 * until this one's kernels are done (NULL when that is 0). steps, batch or channels may be 0. */
VM_API vm_status vm_gated_scan(int device,
                               int32_t type,
                               int64_t batch,
                               int64_t steps,
                               int64_t channels,
                               const vm_sequence* x,
                               const vm_sequence* gate,
                               const float* h0,
                               const int32_t* lengths,
                               const vm_sequence* y,
                               float* last,
                               float* states,
                               void* workspace,
                               size_t workspace_bytes,
                               void* stream);

/* The gradients of x, gate and h0 (each may be NULL) from those of y and last (each NULL: zero), with x, gate and lengths as
 * vm_gated_scan had them and the states that it kept. An input that a stride of 0 repeats gets a gradient for every place it was
 * used at: what belongs to the one value is their sum. Behind a sequence's length the gradients of x and gate are 0. Workspace as above. */
VM_API vm_status vm_gated_scan_backward(int device,
                                        int32_t type,
                                        int64_t batch,
                                        int64_t steps,
                                        int64_t channels,
                                        const vm_sequence* x,
                                        const vm_sequence* gate,
                                        const float* states,
                                        const int32_t* lengths,
                                        const vm_sequence* dy,
                                        const float* d_last,
                                        const vm_sequence* dx,
                                        const vm_sequence* d_gate,
                                        float* d_h0,
                                        void* workspace,
                                        size_t workspace_bytes,
                                        void* stream);

/* Bytes of workspace that either of the two needs at these sizes (0 for sizes that they refuse). */
VM_API size_t vm_gated_workspace(int64_t batch, int64_t steps, int64_t channels);

/* One step of the recurrence for rows whose states stand in a table of `slots` rows of `channels` 32-bit floats (state_stride elements
 * apart), updated in place: h = f h + (1 - f) x for the slot index[row] (NULL: slot = row, rows <= slots), y[row] = h.
 * x, gate and y have rows x channels elements of `type`, row and channel strides in batch_stride (step_stride is not used) and
 * channel_stride. A row whose index is outside 0..slots-1, or whose slot an earlier row of the call names too, changes no state and its
 * y is 0. y may be NULL. workspace: as above, at least vm_gated_step_workspace(rows, slots) bytes when index is given. */
VM_API vm_status vm_gated_step(int device,
                               int32_t type,
                               int64_t rows,
                               int64_t slots,
                               int64_t channels,
                               float* state,
                               int64_t state_stride,
                               const vm_sequence* x,
                               const vm_sequence* gate,
                               const int32_t* index,
                               const vm_sequence* y,
                               void* workspace,
                               size_t workspace_bytes,
                               void* stream);
VM_API size_t vm_gated_step_workspace(int64_t rows, int64_t slots);

/* Message of the last failing call on this thread. */
VM_API const char* vm_last_error(void);

/* ------------------------------------------------------------------------------------------------------------------
 * Host-side mesh tables for callers that are not C++ and cannot instantiate the reference's templates:
 * a restatement of visualmesh::Mesh (cpp/visualmesh/mesh.hpp:425-467 construction, :499-595 lookup) over the ring
 * and grid models (cpp/visualmesh/model/) and shapes (cpp/visualmesh/geometry/). Host code only.
 * ------------------------------------------------------------------------------------------------------------------ */
typedef struct vm_hostmesh vm_hostmesh;

/* model: "RING4" "RING6" "RING8", "XYGRID4" "XYGRID6" "XYGRID8", "XMGRID4" "XMGRID6" "XMGRID8", "NMGRID4" "NMGRID6"
 * "NMGRID8" (every model of cpp/visualmesh/model/); shape: "SPHERE" (a = radius), "CIRCLE" (a = radius), "CYLINDER"
 * (a = radius, b = height). */
VM_API vm_status vm_hostmesh_create(const char* model,
                             const char* shape,
                             float shape_a,
                             float shape_b,
                             float h,
                             float k,
                             float max_distance,
                             vm_hostmesh** out);
VM_API void vm_hostmesh_destroy(vm_hostmesh* mesh);
VM_API int32_t vm_hostmesh_n_nodes(const vm_hostmesh* mesh);
VM_API int32_t vm_hostmesh_n_neighbours(const vm_hostmesh* mesh);
VM_API int32_t vm_hostmesh_n_bsp(const vm_hostmesh* mesh);
/* rays: n_nodes x 3, neighbours: n_nodes x n_neighbours */
VM_API vm_status vm_hostmesh_nodes(const vm_hostmesh* mesh, float* rays, int32_t* neighbours);
/* ranges: n_bsp x 2, children: n_bsp x 2, cones: n_bsp x 5 */
VM_API vm_status vm_hostmesh_bsp(const vm_hostmesh* mesh, int32_t* ranges, int32_t* children, float* cones);
/* Mesh::lookup on the host; writes up to capacity pairs, returns the number of ranges through *n_ranges. */
VM_API vm_status vm_hostmesh_lookup(const vm_hostmesh* mesh,
                             const float Hoc[16],
                             const vm_lens* lens,
                             int32_t* ranges,
                             int32_t capacity,
                             int32_t* n_ranges);

#ifdef __cplusplus
}
#endif

#endif /* VMCUDA_H */
