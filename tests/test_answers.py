"""Calls of the operators on answers that are refused before any device is asked, and empty ones, which need none."""
import ctypes as C

import pytest
import torch

from visualmesh_b200 import abi, answers
from visualmesh_b200.engine import VisualMeshError

P = 4096  # an address that is never read: every call here ends before its launch
OK, REFUSED = abi.VM_OK, abi.VM_ERR_INVALID_ARGUMENT


def scores(x=P, type=abi.VM_F32, rows=3, classes=5, stride=5, flags=0, labels=P, top=0, log_prob=P, entropy=P, log_sum=P, top_log_prob=None, top_index=None):
    return abi.load().vm_scores(-1, x, type, rows, classes, stride, flags, labels, top, log_prob, entropy, log_sum, top_log_prob, top_index, None)


def scores_backward(x=P, type=abi.VM_F32, rows=3, classes=5, stride=5, flags=0, labels=P, entropy=P, log_sum=P, d_log_prob=P, d_entropy=P, d_log_sum=P, dx=P, dx_stride=5):
    return abi.load().vm_scores_backward(-1, x, type, rows, classes, stride, flags, labels, entropy, log_sum, d_log_prob, d_entropy, d_log_sum, dx, dx_stride, None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(x=P + 2), dict(type=3), dict(type=-1), dict(rows=-1), dict(rows=2**31), dict(classes=0), dict(classes=-4), dict(stride=-5), dict(stride=2**61),
    dict(flags=4), dict(labels=P + 2), dict(labels=P + 4, flags=abi.VM_LABELS_64), dict(labels=None), dict(top=-1), dict(top=6, top_log_prob=P, top_index=P),
    dict(top=33, classes=40, stride=40, top_log_prob=P, top_index=P), dict(top=2, top_log_prob=P), dict(top=2, top_index=P),
])
def test_scores_refuses(bad):
    assert scores(**bad) == REFUSED
    assert abi.load().vm_last_error()


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(x=P + 2), dict(type=3), dict(rows=-1), dict(rows=2**31), dict(classes=0), dict(stride=-5), dict(flags=8), dict(labels=None), dict(entropy=None),
    dict(log_sum=None), dict(dx=None), dict(dx=P + 1), dict(dx_stride=4), dict(dx_stride=2**61),
])
def test_scores_backward_refuses(bad):
    assert scores_backward(**bad) == REFUSED


def sequence(data=P, b=77, t=7, c=1):
    return C.byref(abi.vm_sequence(data, b, t, c))


def scan(type=abi.VM_F32, batch=2, steps=11, channels=7, x=(), gate=(), y=(), workspace=P, size=1 << 30):
    as_sequence = lambda v: v if v is None else sequence(*v)
    return abi.load().vm_gated_scan(-1, type, batch, steps, channels, as_sequence(x), as_sequence(gate), None, None, as_sequence(y), None, None, workspace, size, None)


def scan_backward(type=abi.VM_F32, batch=2, steps=11, channels=7, x=(), gate=(), states=P, dy=(), dx=(), d_gate=(), workspace=P, size=1 << 30):
    as_sequence = lambda v: v if v is None else sequence(*v)
    return abi.load().vm_gated_scan_backward(-1, type, batch, steps, channels, as_sequence(x), as_sequence(gate), states, None, as_sequence(dy), None, as_sequence(dx),
                                             as_sequence(d_gate), None, workspace, size, None)


def step(type=abi.VM_F32, rows=4, slots=9, channels=7, state=P, stride=7, x=(P, 7, 0, 1), gate=(P, 7, 0, 1), index=P, y=(P, 7, 0, 1), workspace=P, size=1 << 20):
    as_sequence = lambda v: v if v is None else sequence(*v)
    return abi.load().vm_gated_step(-1, type, rows, slots, channels, state, stride, as_sequence(x), as_sequence(gate), index, as_sequence(y), workspace, size, None)


SEQUENCES = [dict(x=None), dict(x=(None,)), dict(gate=None), dict(x=(P + 2,)), dict(gate=(P + 1,)), dict(x=(P, -1, 7, 1)), dict(gate=(P, 77, -7, 1)), dict(x=(P, 77, 7, -1)),
             dict(x=(P, 2**61, 7, 1)), dict(type=3), dict(batch=-1), dict(steps=-1), dict(channels=-1), dict(batch=2**31), dict(steps=2**31), dict(channels=2**31),
             dict(batch=2**30, channels=2**30)]


@pytest.mark.parametrize("bad", SEQUENCES + [dict(y=(P, 77, 0, 1)), dict(y=(P, 7, 7, 1)), dict(y=(P, 77, 7, 2)), dict(y=(P, 77, 6, 1)), dict(y=(P, 0, 7, 1)), dict(y=(P + 2,))])
def test_scan_refuses(bad):
    assert scan(**bad) == REFUSED


@pytest.mark.parametrize("bad", SEQUENCES + [dict(states=None), dict(dy=(P + 2,)), dict(dy=(P, 77, -1, 1)), dict(dx=(P, 77, 0, 1)), dict(d_gate=(P, 7, 7, 1)), dict(dx=(P + 3,))])
def test_scan_backward_refuses(bad):
    assert scan_backward(**bad) == REFUSED


@pytest.mark.parametrize("bad", [
    dict(type=3), dict(rows=-1), dict(slots=-1), dict(slots=2**31), dict(channels=-1), dict(state=None), dict(stride=6), dict(stride=2**61), dict(x=None), dict(gate=None),
    dict(x=(P + 2, 7, 0, 1)), dict(y=(P, 6, 0, 1)), dict(y=(P, 0, 0, 1)), dict(index=None, rows=10), dict(rows=4000, workspace=None), dict(rows=4000, workspace=P + 4), dict(rows=4000, size=8),
])
def test_step_refuses(bad):
    assert step(**bad) == REFUSED


def test_a_workspace_that_is_too_small_is_refused():
    """At sizes that need one."""
    lib = abi.load()
    needed = [(b, t, d) for b in (1, 3) for t in (1, 64, 4096, 100000) for d in (1, 64, 4096) if lib.vm_gated_workspace(b, t, d)]
    for b, t, d in needed:
        strides = (P, t * d, d, 1)
        assert scan(batch=b, steps=t, channels=d, x=strides, gate=strides, y=strides, size=lib.vm_gated_workspace(b, t, d) - 1) == REFUSED
        assert scan(batch=b, steps=t, channels=d, x=strides, gate=strides, y=strides, workspace=None) == REFUSED
        assert scan(batch=b, steps=t, channels=d, x=strides, gate=strides, y=strides, workspace=P + 8) == REFUSED
        assert scan_backward(batch=b, steps=t, channels=d, x=strides, gate=strides, dy=strides, dx=strides, d_gate=strides, size=0) == REFUSED


def test_empty_calls_need_no_device():
    assert scores(rows=0, x=None, labels=None, log_prob=None) == OK
    assert scores_backward(rows=0, x=None, dx=None) == OK
    assert scan(batch=0, x=None, gate=None) == OK
    assert scan_backward(channels=0, x=None, gate=None, states=None) == OK
    assert step(rows=0, x=None, gate=None) == OK
    assert abi.load().vm_gated_workspace(-1, 5, 5) == 0 and abi.load().vm_gated_step_workspace(0, 5) == 0


@pytest.mark.parametrize("call", [
    lambda x: answers.scores(x[0]),
    lambda x: answers.scores_backward(x[0], answers.Scores(None, x[0, :, 0], x[0, :, 0], None, None)),
    lambda x: answers.gated_scan(x, x),
    lambda x: answers.gated_scan_backward(x, x, x),
    lambda x: answers.gated_step(x[0], x[0], x[0]),
])
def test_tensors_of_the_host_are_refused(call):
    with pytest.raises(VisualMeshError):
        call(torch.zeros(2, 3, 4))
