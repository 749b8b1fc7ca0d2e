"""Operators on what a network answered, for torch tensors on the GPU: how sure it was of every row, and what a sequence of frames adds.

    got = scores(classifications, labels, top=2, probabilities=True)      # vm_scores
    dx = scores_backward(x, got, labels, d_log_prob=...)                  # vm_scores_backward
    got = gated_scan(x, gate, h0, keep=True)                              # vm_gated_scan
    dx, d_gate, d_h0 = gated_scan_backward(x, gate, got.states, dy)       # vm_gated_scan_backward
    y = gated_step(state, x, gate, index)                                 # vm_gated_step

What each computes, masks, lengths and special values included, is written beside its entry point in include/vmcuda.h. The calls
enqueue on torch's current stream of the tensors' device and return without waiting; they may be captured into a CUDA graph. Results and
workspaces are new tensors of every call. Tensors have float32, float16 or bfloat16 elements with any strides that are not negative,
where nothing else is said. Autograd does not see these calls: the gradients are functions of their own, and a tensor that requires a
gradient is refused where gradients are recorded. Refused calls raise VisualMeshError.
"""
import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import abi
from .abi import VisualMeshError

_TYPES = {torch.float32: abi.VM_F32, torch.float16: abi.VM_F16, torch.bfloat16: abi.VM_BF16}


class Scores(NamedTuple):
    """One value (float32) per row, `top` of them for the best; None for what was not asked for."""
    log_prob: Optional[torch.Tensor]
    entropy: torch.Tensor
    log_sum: torch.Tensor
    top_log_prob: Optional[torch.Tensor]
    top_index: Optional[torch.Tensor]


class Scanned(NamedTuple):
    """y as x, last [batch, channels] float32, and what gated_scan_backward starts from (None unless kept)."""
    y: torch.Tensor
    last: torch.Tensor
    states: Optional[torch.Tensor]


def _refuse(message):
    raise VisualMeshError(abi.VM_ERR_INVALID_ARGUMENT, message)


def _type(x, name, dimensions):
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        _refuse(f"{name} must be a tensor on the GPU (there is no CPU fallback)")
    if x.dim() != dimensions:
        _refuse(f"{name} must have {dimensions} dimensions")
    if x.requires_grad and torch.is_grad_enabled():
        _refuse(f"{name} requires a gradient, which autograd would not get: detach it and call the backward function")
    kind = _TYPES.get(x.dtype)
    if kind is None:
        _refuse(f"{name} must be float32, float16 or bfloat16")
    return kind


def _like(x, name, shape, dtype, device, dense=False):
    """x has this shape and type and is on this device; dense: and without gaps."""
    if not isinstance(x, torch.Tensor) or x.device != device:
        _refuse(f"{name} must be a tensor on {device}")
    if x.dtype != dtype or tuple(x.shape) != tuple(shape):
        _refuse(f"{name} must be {dtype} of shape {tuple(shape)}")
    if x.requires_grad and torch.is_grad_enabled():
        _refuse(f"{name} requires a gradient, which autograd would not get: detach it and call the backward function")
    if dense and not x.is_contiguous():
        _refuse(f"{name} must be contiguous")
    return x


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _pointer(x):
    return None if x is None else x.data_ptr()


def _rows(x, labels, probabilities):
    """What both score calls pass on: type, sizes, row stride, flags"""
    kind = _type(x, "x", 2)
    rows, classes = x.shape
    if classes > 1 and x.stride(1) != 1:
        _refuse("the classes of a row must lie side by side")
    flags = abi.VM_PROBABILITIES if probabilities else 0
    if labels is not None:
        if not isinstance(labels, torch.Tensor) or labels.dtype not in (torch.int32, torch.int64):
            _refuse("labels must be int32 or int64")
        _like(labels, "labels", (rows,), labels.dtype, x.device, dense=True)
        if labels.dtype == torch.int64:
            flags |= abi.VM_LABELS_64
    return kind, rows, classes, x.stride(0), flags


def scores(x, labels=None, top=0, probabilities=False) -> Scores:
    """x: [rows, classes], logits or (probabilities) what a softmax wrote; labels: [rows] int32 or int64, -1 where a row has none."""
    kind, rows, classes, stride, flags = _rows(x, labels, probabilities)
    if not 0 <= top <= min(classes, abi.VM_MAX_TOP):
        _refuse(f"top must be 0..{min(classes, abi.VM_MAX_TOP)}")
    device = x.device
    made = torch.empty((3, rows), dtype=torch.float32, device=device)
    log_prob, entropy, log_sum = made.unbind(0)
    if labels is None:
        log_prob = None
    top_log_prob = top_index = None
    if top:
        top_log_prob = torch.empty((rows, top), dtype=torch.float32, device=device)
        top_index = torch.empty((rows, top), dtype=torch.int32, device=device)
    abi.check(abi.load().vm_scores(device.index, x.data_ptr(), kind, rows, classes, stride, flags, _pointer(labels), top, _pointer(log_prob), entropy.data_ptr(),
                                   log_sum.data_ptr(), _pointer(top_log_prob), _pointer(top_index), _stream(device)))
    return Scores(log_prob, entropy, log_sum, top_log_prob, top_index)


def scores_backward(x, scored: Scores, labels=None, d_log_prob=None, d_entropy=None, d_log_sum=None, probabilities=False):
    """The gradient of x from those of the scores that scores(x, labels, probabilities=probabilities) returned (None: zero)."""
    kind, rows, classes, stride, flags = _rows(x, labels, probabilities)
    if d_log_prob is not None and labels is None:
        _refuse("d_log_prob without labels")
    device = x.device
    for name, v in (("entropy", scored.entropy), ("log_sum", scored.log_sum), ("d_log_prob", d_log_prob), ("d_entropy", d_entropy), ("d_log_sum", d_log_sum)):
        if v is not None:
            _like(v, name, (rows,), torch.float32, device, dense=True)
    dx = torch.empty((rows, classes), dtype=x.dtype, device=device)
    abi.check(abi.load().vm_scores_backward(device.index, x.data_ptr(), kind, rows, classes, stride, flags, _pointer(labels), scored.entropy.data_ptr(),
                                            scored.log_sum.data_ptr(), _pointer(d_log_prob), _pointer(d_entropy), _pointer(d_log_sum), dx.data_ptr(), classes,
                                            _stream(device)))
    return dx


def _sequence(x):
    return None if x is None else C.byref(abi.vm_sequence(x.data_ptr(), *x.stride()))


def _sequences(x, gate, lengths):
    kind = _type(x, "x", 3)
    _like(gate, "gate", x.shape, x.dtype, x.device)
    if lengths is not None:
        _like(lengths, "lengths", (x.shape[0],), torch.int32, x.device, dense=True)
    return kind, tuple(x.shape)


def _workspace(size, device):
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def gated_scan(x, gate, h0=None, lengths=None, keep=False) -> Scanned:
    """x, gate: [batch, steps, channels]; h0: [batch, channels] float32; lengths: [batch] int32. A stride of 0 (expand) repeats x or gate.
    keep: also the states that gated_scan_backward needs."""
    kind, shape = _sequences(x, gate, lengths)
    batch, steps, channels = shape
    device, lib = x.device, abi.load()
    if h0 is not None:
        _like(h0, "h0", (batch, channels), torch.float32, device, dense=True)
    y = torch.empty(shape, dtype=x.dtype, device=device)
    last = torch.empty((batch, channels), dtype=torch.float32, device=device)
    states = torch.empty((batch, -(-steps // abi.VM_GATED_KEEP), channels), dtype=torch.float32, device=device) if keep else None
    size = lib.vm_gated_workspace(batch, steps, channels)
    workspace = _workspace(size, device)
    abi.check(lib.vm_gated_scan(device.index, kind, batch, steps, channels, _sequence(x), _sequence(gate), _pointer(h0), _pointer(lengths), _sequence(y),
                                last.data_ptr(), _pointer(states), _pointer(workspace), size, _stream(device)))
    return Scanned(y, last, states)


def gated_scan_backward(x, gate, states, dy=None, d_last=None, lengths=None):
    """(dx, d_gate, d_h0) from the gradients of y and last (None: zero). x, gate and lengths as gated_scan had them, states as it kept them."""
    kind, shape = _sequences(x, gate, lengths)
    batch, steps, channels = shape
    device, lib = x.device, abi.load()
    _like(states, "states", (batch, -(-steps // abi.VM_GATED_KEEP), channels), torch.float32, device, dense=True)
    if dy is not None:
        _like(dy, "dy", shape, x.dtype, device)
    if d_last is not None:
        _like(d_last, "d_last", (batch, channels), torch.float32, device, dense=True)
    dx, d_gate = torch.empty((2,) + shape, dtype=x.dtype, device=device).unbind(0)
    d_h0 = torch.empty((batch, channels), dtype=torch.float32, device=device)
    size = lib.vm_gated_workspace(batch, steps, channels)
    workspace = _workspace(size, device)
    abi.check(lib.vm_gated_scan_backward(device.index, kind, batch, steps, channels, _sequence(x), _sequence(gate), states.data_ptr(), _pointer(lengths),
                                         _sequence(dy), _pointer(d_last), _sequence(dx), _sequence(d_gate), d_h0.data_ptr(), _pointer(workspace), size,
                                         _stream(device)))
    return dx, d_gate, d_h0


def _row_sequence(x):
    return C.byref(abi.vm_sequence(x.data_ptr(), x.stride(0), 0, x.stride(1)))


def gated_step(state, x, gate, index=None, out=None):
    """One step for every row of x [rows, channels]: advances row index[row] (int32; None: row) of state [slots, channels] float32 in place
    and returns the rows' new states in x's type. Rows whose index is outside the table, or already taken by an earlier row, give 0.
    out: where the result is written instead of a new tensor (it overlaps no other argument)."""
    kind = _type(x, "x", 2)
    rows, channels = x.shape
    device, lib = x.device, abi.load()
    _like(gate, "gate", x.shape, x.dtype, device)
    if not isinstance(state, torch.Tensor) or state.dim() != 2:
        _refuse("state must have 2 dimensions")
    slots = state.shape[0]
    _like(state, "state", (slots, channels), torch.float32, device)
    if channels > 1 and state.stride(1) != 1:
        _refuse("the channels of a state must lie side by side")
    if index is not None:
        _like(index, "index", (rows,), torch.int32, device, dense=True)
    y = torch.empty((rows, channels), dtype=x.dtype, device=device) if out is None else _like(out, "out", x.shape, x.dtype, device)
    size = lib.vm_gated_step_workspace(rows, slots) if index is not None else 0
    workspace = _workspace(size, device)
    abi.check(lib.vm_gated_step(device.index, kind, rows, slots, channels, state.data_ptr(), state.stride(0), _row_sequence(x), _row_sequence(gate),
                                _pointer(index), _row_sequence(y), _pointer(workspace), size, _stream(device)))
    return y
