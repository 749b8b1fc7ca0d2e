"""Pointers that no element of their type begins on are refused: a load or store there would be a fault of the GPU. Every call ends before its launch."""
import ctypes as C

import pytest

from visualmesh_b200 import abi

P = 4096


def sequence():
    return C.byref(abi.vm_sequence(P, 77, 7, 1))


def scores(log_prob=P, entropy=P, log_sum=P, top_log_prob=P, top_index=P):
    return abi.load().vm_scores(-1, P, abi.VM_F32, 3, 5, 5, 0, P, 2, log_prob, entropy, log_sum, top_log_prob, top_index, None)


def scores_backward(entropy=P, log_sum=P, d_log_prob=P, d_entropy=P, d_log_sum=P):
    return abi.load().vm_scores_backward(-1, P, abi.VM_F32, 3, 5, 5, 0, P, entropy, log_sum, d_log_prob, d_entropy, d_log_sum, P, 5, None)


def scan(h0=P, lengths=P, last=P, states=P):
    return abi.load().vm_gated_scan(-1, abi.VM_F32, 2, 11, 7, sequence(), sequence(), h0, lengths, sequence(), last, states, P, 1 << 30, None)


def scan_backward(states=P, lengths=P, d_last=P, d_h0=P):
    return abi.load().vm_gated_scan_backward(-1, abi.VM_F32, 2, 11, 7, sequence(), sequence(), states, lengths, sequence(), d_last, sequence(), sequence(), d_h0, P, 1 << 30, None)


def step(state=P, index=P):
    row = C.byref(abi.vm_sequence(P, 7, 0, 1))
    return abi.load().vm_gated_step(-1, abi.VM_F32, 4, 9, 7, state, 7, row, row, index, row, P, 1 << 20, None)


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("call,name", [(call, name) for call in (scores, scores_backward, scan, scan_backward, step)
                                       for name in call.__code__.co_varnames[:call.__code__.co_argcount]])
def test_pointers_beside_their_elements_are_refused(call, name, off):
    assert call(**{name: P + off}) == abi.VM_ERR_INVALID_ARGUMENT
    assert b"aligned" in abi.load().vm_last_error()
