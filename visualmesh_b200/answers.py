"""Operators on what a network answered, for torch tensors on the GPU: how sure it was of every row, and what a sequence of frames adds.

    got = scores(classifications, labels, top=2, probabilities=True)      # vm_scores
    dx = scores_backward(x, got, labels, d_log_prob=...)                  # vm_scores_backward
    got = gated_scan(x, gate, h0, keep=True)                              # vm_gated_scan
    dx, d_gate, d_h0 = gated_scan_backward(x, gate, got.states, dy)       # vm_gated_scan_backward
    y = gated_step(state, x, gate, index)                                 # vm_gated_step

What each computes, masks, lengths and special values included, is written beside its entry point in include/vmcuda.h. The calls
enqueue on torch's current stream of the tensors' device and return without waiting; they may be captured into a CUDA graph. Results and
workspaces are new tensors of every call. Tensors have float32, float16 or bfloat16 elements with any strides that are not negative,
where nothing else is said. Autograd does not see these calls: the gradients are functions of their own, a tensor that requires a
gradient is refused where gradients are recorded, and so is one with a tangent of forward differentiation. What gated_step writes in place
counts as written. Refused calls raise VisualMeshError.
"""
from typing import NamedTuple, Optional

import torch

from . import abi
from .abi import VisualMeshError  # noqa: F401  (re-export)

abi.load()
try:
    from . import _answers as _native
except ImportError as e:
    raise RuntimeError("visualmesh_b200._answers cannot be imported: build it with `python -m visualmesh_b200.build`") from e


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


def scores(x, labels=None, top=0, probabilities=False) -> Scores:
    """x: [rows, classes], logits or (probabilities) what a softmax wrote, the classes of a row side by side; labels: [rows] int32 or int64,
    -1 where a row has none; top: how many of the best classes."""
    return Scores(*_native.scores(x, labels, top, probabilities))


def scores_backward(x, scored: Scores, labels=None, d_log_prob=None, d_entropy=None, d_log_sum=None, probabilities=False):
    """The gradient of x from those of the scores that scores(x, labels, probabilities=probabilities) returned ([rows] float32, None: zero)."""
    return _native.scores_backward(x, scored.entropy, scored.log_sum, labels, d_log_prob, d_entropy, d_log_sum, probabilities)


def gated_scan(x, gate, h0=None, lengths=None, keep=False) -> Scanned:
    """x, gate: [batch, steps, channels]; h0: [batch, channels] float32; lengths: [batch] int32. A stride of 0 (expand) repeats x or gate.
    keep: also the states that gated_scan_backward needs."""
    return Scanned(*_native.gated_scan(x, gate, h0, lengths, keep))


def gated_scan_backward(x, gate, states, dy=None, d_last=None, lengths=None):
    """(dx, d_gate, d_h0) from the gradients of y and last (None: zero). x, gate and lengths as gated_scan had them, states as it kept them.
    An x or gate that expand repeats gets a gradient for every place it was used at: what belongs to the one value is their sum."""
    return _native.gated_scan_backward(x, gate, states, dy, d_last, lengths)


def gated_step(state, x, gate, index=None, out=None):
    """One step for every row of x [rows, channels]: advances row index[row] (int32; None: row) of state [slots, channels] float32 in place
    and returns the rows' new states in x's type. Rows whose index is outside the table, or already taken by an earlier row, give 0.
    out: where the result is written instead of a new tensor (it overlaps no other argument)."""
    return _native.gated_step(state, x, gate, index, out)
