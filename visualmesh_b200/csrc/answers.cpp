// Python's side of the operators on answers (answers.py): checks of the tensors, outputs and workspaces, and the calls of the C ABI,
// without an interpreter's share. The calls of small problems are bound by their way to the GPU: through ctypes and Python's view of the
// tensors one took 15 to 20 us.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/Functions.h>
#include <ATen/core/Tensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <optional>
#include <string>

#include "../../include/vmcuda.h"

namespace {

using at::Tensor;
using Maybe = std::optional<Tensor>;

PyObject* g_error = nullptr;  // VisualMeshError

// A call that is refused here, before the C ABI sees it.
struct Refused {
    std::string message;
};
// The Python error of a status has been set.
struct Raised {};

[[noreturn]] void refuse(const std::string& message) {
    throw Refused{message};
}
void raise_status(int status, const char* message) {
    if (PyObject* error = PyObject_CallFunction(g_error, "is", status, message)) {
        PyErr_SetObject(g_error, error);
        Py_DECREF(error);
    }
}
void check(vm_status status) {
    if (status == VM_OK) return;
    raise_status(status, vm_last_error());
    throw Raised{};
}

const Tensor& tensor_of(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor on the GPU (there is no CPU fallback)");
    return THPVariable_Unpack(o);
}
// No gradient, forward or backward, would be lost, and x holds its own values.
void check_plain(const Tensor& x, const char* name) {
    if (x.unsafeGetTensorImpl()->autograd_meta() != nullptr) {  // plain tensors have none
        if (x.requires_grad() && c10::GradMode::is_enabled()) refuse(std::string(name) + " requires a gradient, which autograd would not get: detach it and call the backward function");
        if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && x._fw_grad(0).defined()) refuse(std::string(name) + " has a tangent, which forward differentiation would lose: unpack it first");
    }
    if (x.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor}))) refuse(std::string(name) + " is a view that holds no values of its own: call resolve_neg() or clone()");
}
// x is on the GPU, has so many dimensions and one of the three types, which is returned
int32_t type_of(const Tensor& x, const char* name, int64_t dimensions) {
    if (!x.is_cuda() || x.layout() != at::kStrided) refuse(std::string(name) + " must be a tensor on the GPU (there is no CPU fallback)");
    if (x.dim() != dimensions) refuse(std::string(name) + " must have " + std::to_string(dimensions) + " dimensions");
    check_plain(x, name);
    switch (x.scalar_type()) {
        case at::kFloat: return VM_F32;
        case at::kHalf: return VM_F16;
        case at::kBFloat16: return VM_BF16;
        default: refuse(std::string(name) + " must be float32, float16 or bfloat16");
    }
}
enum Layout { ANY, DENSE };
void check_like(const Tensor& x, const char* name, at::IntArrayRef shape, at::ScalarType type, const at::Device& device, Layout layout) {
    if (x.device() != device || x.layout() != at::kStrided) refuse(std::string(name) + " must be a tensor on " + device.str());
    if (x.scalar_type() != type || x.sizes() != shape) {
        std::string wanted = std::string(name) + " must be " + c10::toString(type) + " of shape (";
        for (const int64_t n : shape) wanted += std::to_string(n) + ", ";
        refuse(wanted + ")");
    }
    check_plain(x, name);
    if (layout == DENSE && !x.is_contiguous()) refuse(std::string(name) + " must be contiguous");
}
Maybe like(PyObject* o, const char* name, at::IntArrayRef shape, at::ScalarType type, const at::Device& device, Layout layout) {
    if (o == Py_None) return std::nullopt;
    const Tensor& x = tensor_of(o, name);
    check_like(x, name, shape, type, device, layout);
    return x;
}

// x is written in place: autograd's record of what it saved of x is no longer of x. (Tensors of inference mode have no such record.)
void written(const Tensor& x) {
    if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}

Tensor make(at::IntArrayRef shape, at::ScalarType type, const at::Device& device) {
    return at::empty(shape, at::TensorOptions().dtype(type).device(device));
}
// A part of a tensor of bytes as a tensor of its own: the small results of a call share one allocation.
Tensor part_of(const Tensor& bytes, size_t& at, at::IntArrayRef shape, at::ScalarType type) {
    Tensor part      = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(bytes.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::scalarTypeToTypeMeta(type));
    const auto size  = c10::elementSize(type);
    auto* const impl = part.unsafeGetTensorImpl();
    impl->set_storage_offset(static_cast<int64_t>(at / size));
    impl->set_sizes_contiguous(shape);
    at += static_cast<size_t>(impl->numel()) * size;
    return part;
}

template <typename T = void>
T* pointer(const Tensor& x) {
    return static_cast<T*>(x.data_ptr());
}
template <typename T = void>
T* pointer(const Maybe& x) {
    return x ? static_cast<T*>(x->data_ptr()) : nullptr;
}
void* stream_of(const Tensor& x) {
    return c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
}
PyObject* wrap(Maybe x) {
    if (!x) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(*x));
}
PyObject* tuple_of(std::initializer_list<Maybe> values) {
    PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(values.size()));
    if (t == nullptr) throw Raised{};
    Py_ssize_t i = 0;
    for (const Maybe& v : values) {
        PyObject* o = wrap(v);
        if (o == nullptr) {
            Py_DECREF(t);
            throw Raised{};
        }
        PyTuple_SET_ITEM(t, i++, o);
    }
    return t;
}

// What every entry does around its body: the errors.
template <typename F>
PyObject* call(F body, Py_ssize_t given, Py_ssize_t wanted) {
    HANDLE_TH_ERRORS
    if (given != wanted) {
        PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
        return nullptr;
    }
    try {
        return body();
    }
    catch (const Refused& r) {
        raise_status(VM_ERR_INVALID_ARGUMENT, r.message.c_str());
        return nullptr;
    }
    catch (const Raised&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// ---- scores ------------------------------------------------------------------------------------------------------------------
struct Rows {
    Tensor x;
    Maybe labels;
    int32_t type;
    int64_t rows, classes, stride;
    uint32_t flags;
    Rows(PyObject* o, PyObject* l, PyObject* probabilities) : x(tensor_of(o, "x")) {
        type    = type_of(x, "x", 2);
        rows    = x.size(0);
        classes = x.size(1);
        stride  = x.stride(0);
        if (classes > 1 && x.stride(1) != 1) refuse("the classes of a row must lie side by side");
        if (classes > INT32_MAX) refuse("too many classes");
        const int p = PyObject_IsTrue(probabilities);
        if (p < 0) throw Raised{};
        flags = p ? VM_PROBABILITIES : 0;
        if (l != Py_None) {
            const Tensor& t = tensor_of(l, "labels");
            if (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) refuse("labels must be int32 or int64");
            check_like(t, "labels", {rows}, t.scalar_type(), x.device(), DENSE);
            if (t.scalar_type() == at::kLong) flags |= VM_LABELS_64;
            labels = t;
        }
    }
};

// (x, labels, top, probabilities) -> (log_prob, entropy, log_sum, top_log_prob, top_index)
PyObject* scores(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return call([&] {
        const Rows r(args[0], args[1], args[3]);
        const long top = PyLong_AsLong(args[2]);
        if (top == -1 && PyErr_Occurred()) throw Raised{};
        const int64_t most = r.classes < VM_MAX_TOP ? r.classes : VM_MAX_TOP;
        if (top < 0 || top > most) refuse("top must be 0.." + std::to_string(most));
        const at::Device device = r.x.device();
        // the values of the rows are one allocation, the best classes another
        const Tensor values  = make({r.rows * (r.labels ? 12 : 8)}, at::kByte, device);
        size_t at            = 0;
        const Tensor entropy = part_of(values, at, {r.rows}, at::kFloat), log_sum = part_of(values, at, {r.rows}, at::kFloat);
        Maybe log_prob, top_log_prob, top_index;
        if (r.labels) log_prob = part_of(values, at, {r.rows}, at::kFloat);
        if (top > 0) {
            const Tensor best = make({r.rows * top * 8}, at::kByte, device);
            at                = 0;
            top_log_prob      = part_of(best, at, {r.rows, top}, at::kFloat);
            top_index         = part_of(best, at, {r.rows, top}, at::kInt);
        }
        check(vm_scores(device.index(), pointer(r.x), r.type, r.rows, static_cast<int32_t>(r.classes), r.stride, r.flags, pointer(r.labels), static_cast<int32_t>(top),
                        pointer<float>(log_prob), pointer<float>(entropy), pointer<float>(log_sum), pointer<float>(top_log_prob), pointer<int32_t>(top_index), stream_of(r.x)));
        return tuple_of({log_prob, entropy, log_sum, top_log_prob, top_index});
    }, n, 4);
}

// (x, entropy, log_sum, labels, d_log_prob, d_entropy, d_log_sum, probabilities) -> dx
PyObject* scores_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return call([&] {
        const Rows r(args[0], args[3], args[7]);
        const at::Device device = r.x.device();
        const auto row = [&](int i, const char* name) { return like(args[i], name, {r.rows}, at::kFloat, device, DENSE); };
        const Maybe entropy = row(1, "entropy"), log_sum = row(2, "log_sum"), d_log_prob = row(4, "d_log_prob"), d_entropy = row(5, "d_entropy"), d_log_sum = row(6, "d_log_sum");
        if (d_log_prob && !r.labels) refuse("d_log_prob without labels");
        const Tensor dx = make({r.rows, r.classes}, r.x.scalar_type(), device);
        check(vm_scores_backward(device.index(), pointer(r.x), r.type, r.rows, static_cast<int32_t>(r.classes), r.stride, r.flags, pointer(r.labels), pointer<float>(entropy),
                                 pointer<float>(log_sum), pointer<float>(d_log_prob), pointer<float>(d_entropy), pointer<float>(d_log_sum), pointer(dx), r.classes, stream_of(r.x)));
        return wrap(dx);
    }, n, 8);
}

// ---- recurrence ----------------------------------------------------------------------------------------------------------------
vm_sequence sequence(const Tensor& x) {
    return vm_sequence{x.data_ptr(), x.stride(0), x.stride(1), x.stride(2)};
}
vm_sequence row_sequence(const Tensor& x) {
    return vm_sequence{x.data_ptr(), x.stride(0), 0, x.stride(1)};
}
Maybe workspace_of(size_t size, const at::Device& device) {
    return size > 0 ? Maybe(make({static_cast<int64_t>(size)}, at::kByte, device)) : Maybe();
}

struct Sequences {
    Tensor x, gate;
    Maybe lengths;
    int32_t type;
    int64_t batch, steps, channels, kept;
    size_t workspace;
    Sequences(PyObject* o, PyObject* g, PyObject* l) : x(tensor_of(o, "x")), gate(tensor_of(g, "gate")) {
        type = type_of(x, "x", 3);
        check_like(gate, "gate", x.sizes(), x.scalar_type(), x.device(), ANY);
        batch = x.size(0), steps = x.size(1), channels = x.size(2);
        kept      = (steps + VM_GATED_KEEP - 1) / VM_GATED_KEEP;
        lengths   = like(l, "lengths", {batch}, at::kInt, x.device(), DENSE);
        workspace = vm_gated_workspace(batch, steps, channels);
    }
};

// (x, gate, h0, lengths, keep) -> (y, last, states)
PyObject* gated_scan(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return call([&] {
        const Sequences s(args[0], args[1], args[3]);
        const at::Device device = s.x.device();
        const Maybe h0 = like(args[2], "h0", {s.batch, s.channels}, at::kFloat, device, DENSE);
        const int keep = PyObject_IsTrue(args[4]);
        if (keep < 0) throw Raised{};
        const Tensor y = make(s.x.sizes(), s.x.scalar_type(), device), last = make({s.batch, s.channels}, at::kFloat, device);
        Maybe states;
        if (keep) states = make({s.batch, s.kept, s.channels}, at::kFloat, device);
        const Maybe workspace = workspace_of(s.workspace, device);
        const vm_sequence vx = sequence(s.x), vg = sequence(s.gate), vy = sequence(y);
        check(vm_gated_scan(device.index(), s.type, s.batch, s.steps, s.channels, &vx, &vg, pointer<float>(h0), pointer<int32_t>(s.lengths), &vy, pointer<float>(last),
                            pointer<float>(states), pointer(workspace), s.workspace, stream_of(s.x)));
        return tuple_of({y, last, states});
    }, n, 5);
}

// (x, gate, states, dy, d_last, lengths) -> (dx, d_gate, d_h0)
PyObject* gated_scan_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return call([&] {
        const Sequences s(args[0], args[1], args[5]);
        const at::Device device = s.x.device();
        const Tensor& states    = tensor_of(args[2], "states");
        check_like(states, "states", {s.batch, s.kept, s.channels}, at::kFloat, device, DENSE);
        const Maybe dy     = like(args[3], "dy", s.x.sizes(), s.x.scalar_type(), device, ANY);
        const Maybe d_last = like(args[4], "d_last", {s.batch, s.channels}, at::kFloat, device, DENSE);
        const Tensor dx = make(s.x.sizes(), s.x.scalar_type(), device), d_gate = make(s.x.sizes(), s.x.scalar_type(), device), d_h0 = make({s.batch, s.channels}, at::kFloat, device);
        const Maybe workspace = workspace_of(s.workspace, device);
        const vm_sequence vx = sequence(s.x), vg = sequence(s.gate), vdy = dy ? sequence(*dy) : vm_sequence{}, vdx = sequence(dx), vdg = sequence(d_gate);
        check(vm_gated_scan_backward(device.index(), s.type, s.batch, s.steps, s.channels, &vx, &vg, pointer<float>(states), pointer<int32_t>(s.lengths), dy ? &vdy : nullptr,
                                     pointer<float>(d_last), &vdx, &vdg, pointer<float>(d_h0), pointer(workspace), s.workspace, stream_of(s.x)));
        return tuple_of({dx, d_gate, d_h0});
    }, n, 6);
}

// (state, x, gate, index, out) -> y
PyObject* gated_step(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return call([&] {
        const Tensor &state = tensor_of(args[0], "state"), &x = tensor_of(args[1], "x"), &gate = tensor_of(args[2], "gate");
        const int32_t type      = type_of(x, "x", 2);
        const at::Device device = x.device();
        const int64_t rows = x.size(0), channels = x.size(1);
        check_like(gate, "gate", x.sizes(), x.scalar_type(), device, ANY);
        if (state.dim() != 2) refuse("state must have 2 dimensions");
        const int64_t slots = state.size(0);
        check_like(state, "state", {slots, channels}, at::kFloat, device, ANY);
        if (channels > 1 && state.stride(1) != 1) refuse("the channels of a state must lie side by side");
        const Maybe index = like(args[3], "index", {rows}, at::kInt, device, DENSE);
        const Maybe out   = like(args[4], "out", x.sizes(), x.scalar_type(), device, ANY);
        const Tensor y    = out ? *out : make(x.sizes(), x.scalar_type(), device);
        const size_t size = index ? vm_gated_step_workspace(rows, slots) : 0;
        const Maybe workspace = workspace_of(size, device);
        const vm_sequence vx = row_sequence(x), vg = row_sequence(gate), vy = row_sequence(y);
        written(state);
        if (out) written(*out);
        check(vm_gated_step(device.index(), type, rows, slots, channels, pointer<float>(state), state.stride(0), &vx, &vg, pointer<int32_t>(index), &vy, pointer(workspace), size,
                            stream_of(x)));
        return wrap(y);
    }, n, 5);
}

PyMethodDef g_methods[] = {{"scores", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(scores)), METH_FASTCALL, nullptr},
                           {"scores_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(scores_backward)), METH_FASTCALL, nullptr},
                           {"gated_scan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gated_scan)), METH_FASTCALL, nullptr},
                           {"gated_scan_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gated_scan_backward)), METH_FASTCALL, nullptr},
                           {"gated_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gated_step)), METH_FASTCALL, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_answers", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__answers(void) {
    PyObject* abi = PyImport_ImportModule("visualmesh_b200.abi");
    if (abi == nullptr) return nullptr;
    g_error = PyObject_GetAttrString(abi, "VisualMeshError");
    Py_DECREF(abi);
    return g_error == nullptr ? nullptr : PyModule_Create(&g_module);
}
