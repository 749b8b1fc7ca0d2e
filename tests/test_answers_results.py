"""What can be said of a batch's results and their engine without a device."""
from visualmesh_b200 import abi


def test_waiting_without_an_engine_is_refused():
    assert abi.load().vm_wait_for(None, None) == abi.VM_ERR_INVALID_ARGUMENT
    assert abi.load().vm_last_error()
